"""Launcher CLIs of the distributed programs (one rank per GPU, torchrun).

The reference's MPI programs are started as `mpirun -np P ./gauss_*_input`
(OpenMP_and_MPI/README.txt); their equivalents here are

  python -m torch.distributed.run --nproc-per-node P --master-addr 127.0.0.1 \\
      -m gelim.cli.dist_gauss [-s N | FILE]
  python -m torch.distributed.run --nproc-per-node P --master-addr 127.0.0.1 \\
      -m gelim.cli.dist_matmul N

Single-GPU programs are native executables under bin/ (csrc/tools).
"""
from __future__ import annotations

import contextlib
import os
import sys


@contextlib.contextmanager
def library_reports_to_stderr():
    """What libraries print on descriptor 1 meanwhile goes to stderr.

    gloo reports its connections there, from C++ and in pieces that mix with
    the other ranks', which would break up the lines of these programs.  For a
    program that owns its process, while it has no other thread that prints;
    without an effect where stdout or stderr is closed or something else's."""
    try:
        own = sys.stdout.fileno() == 1 and sys.stderr.fileno() == 2
    except (AttributeError, OSError, ValueError):
        own = False
    if not own:
        yield
        return
    sys.stdout.flush()
    keep = os.dup(1)
    os.dup2(2, 1)
    try:
        yield
    finally:
        os.dup2(keep, 1)
        os.close(keep)
