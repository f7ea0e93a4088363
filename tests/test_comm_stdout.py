"""Joining a gloo job in programs whose standard output is closed, or written by another thread meanwhile."""
import os
import socket
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

JOIN = """
import os, sys
{before}
import torch
from gelim.parallel import destroy, init_from_env
comm = init_from_env(device="cpu", timeout_s=60)
t = torch.full((1,), float(comm.rank + 1))
comm.all_reduce(t)
{after}
print("sum", t.item(), file=sys.stderr, flush=True)
destroy()
"""


def port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def two_ranks(before, after="", **kw):
    env = dict(os.environ, WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port()), PYTHONPATH=str(ROOT),
               OMP_NUM_THREADS="1")
    ranks = [subprocess.Popen([sys.executable, "-c", JOIN.format(before=before, after=after)],
                              env=dict(env, RANK=str(r), LOCAL_RANK=str(r)), cwd=ROOT, stderr=subprocess.PIPE, text=True,
                              **kw) for r in range(2)]
    try:
        out = [p.communicate(timeout=120) for p in ranks]
    finally:
        for p in ranks:
            p.kill()
    for p, (_, err) in zip(ranks, out):
        assert p.returncode == 0 and "sum 3.0" in err, err
    return out


def test_closed_stdout():
    """As a daemon starts: file descriptor 1 closed, sys.stdout None."""
    two_ranks("assert sys.stdout is None", preexec_fn=lambda: os.close(1))


def test_descriptor_1_of_something_else():
    """A daemon's first file gets descriptor 1: what it writes while the ranks join stays in it."""
    two_ranks("""
import tempfile, threading
f = tempfile.TemporaryFile()
assert f.fileno() == 1
stop, n = threading.Event(), 0
def write():
    global n
    while not stop.is_set():
        n += os.write(1, b"\\1")
writer = threading.Thread(target=write, daemon=True)
writer.start()
""", """
stop.set()
writer.join()
f.seek(0)
assert f.read().count(b"\\1") == n, "bytes went elsewhere"
""", preexec_fn=lambda: os.close(1))


def test_other_threads_keep_their_stdout():
    """Lines of another thread, printed while the ranks join, reach standard output, all of them."""
    out = two_ranks("""
import threading
stop, n = threading.Event(), 0
def write():
    global n
    while not stop.wait(0.001):
        os.write(1, b"line\\n")
        n += 1
writer = threading.Thread(target=write, daemon=True)
writer.start()
""", """
stop.set()
writer.join()
os.write(1, b"written %d\\n" % n)
""", stdout=subprocess.PIPE)
    for text, _ in out:
        assert text.count("line\n") == int(text.rsplit("written ", 1)[1])


def test_launcher_with_stdout_closed():
    env = dict(os.environ, WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port()), PYTHONPATH=str(ROOT),
               OMP_NUM_THREADS="1")
    ranks = [subprocess.Popen([sys.executable, "-m", "gelim.cli.dist_gauss", "-s", "64", "--block", "16", "--device", "cpu"],
                              env=dict(env, RANK=str(r), LOCAL_RANK=str(r)), cwd=ROOT, stderr=subprocess.PIPE, text=True,
                              preexec_fn=lambda: os.close(1)) for r in range(2)]
    try:
        out = [p.communicate(timeout=120) for p in ranks]
    finally:
        for p in ranks:
            p.kill()
    for p, (_, err) in zip(ranks, out):
        assert p.returncode == 0, err
