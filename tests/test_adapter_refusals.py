"""What the adapter products and the clipping refuse without a GPU, and the native argument block's layout."""
import math

import pytest
import torch


def test_argument_block_matches_the_native_struct(gelim):
    from gelim import _native
    from gelim.ops import adapter

    lay = _native.lib().gelim_adapter_args_layout
    assert lay(0) == adapter._ARGS.size and lay(1) == 8 and lay(2) == 19 * 8 and lay(3) == 29 * 8
    assert lay(4) == -1


def test_cpu_tensors_and_types(gelim):
    X, W, A, B = torch.zeros(2, 8), torch.zeros(8, 8), torch.zeros(1, 8, 2), torch.zeros(1, 2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        gelim.ops.adapter_matmul(X, W, A, B)
    with pytest.raises(TypeError):
        gelim.ops.adapter_matmul(X.double(), W.double(), A.double(), B.double())
    with pytest.raises(ValueError, match="CUDA"):
        gelim.ops.adapter_matmul_grad(X, X, W, A, B)
    with pytest.raises(ValueError, match="CUDA"):
        gelim.ops.clip_global_norm([X], 1.0)
    with pytest.raises(ValueError):
        gelim.ops.clip_global_norm([], 1.0)
    with pytest.raises(ValueError):
        gelim.ops.clip_global_norm([X], math.nan)


@pytest.mark.parametrize("field, value", [("dtype", 3), ("dtype", -1), ("T", -1), ("T", 2 ** 30 + 1), ("K", 0), ("N", -4),
                                          ("r", 0), ("r", 257), ("n", 0), ("n", 65536), ("X", 0), ("W", 0), ("A", 0),
                                          ("B", 0), ("Y", 0), ("ws_bytes", 0)])
@pytest.mark.parametrize("grad", [False, True])
def test_native_entry_refuses(gelim, field, value, grad):
    """The native checks come before any GPU call, so they are reached without a GPU."""
    from gelim import _native
    from gelim.ops import adapter

    names = ("dtype T K N r n X ldx W ldw w_trans A a_stride lda a_trans B b_stride ldb b_trans index scale scale_value "
             "Y ldy dX lddx dA dB ws ws_bytes").split()
    vals = dict.fromkeys(names, 0)
    vals.update(dtype=1, T=100, K=64, N=64, r=8, n=2, X=4096, ldx=64, W=4096, ldw=64, A=4096, a_stride=512, lda=8, B=4096,
                b_stride=512, ldb=64, scale_value=1.0, Y=4096, ldy=64, ws=4096, ws_bytes=1 << 40)
    vals[field] = value
    lib = _native.lib()
    fn = lib.gelim_adapter_matmul_grad if grad else lib.gelim_adapter_matmul
    assert fn(adapter._ARGS.pack(*[vals[k] for k in names]), None) == _native.E_ARG
    assert "adapter" in _native.last_error()


@pytest.mark.parametrize("sizes", [dict(T=2 ** 30 - 64, K=8, N=8, n=1), dict(T=64, K=1, N=2 ** 30 - 64, n=1),
                                   dict(T=100, K=2 ** 19, N=64, n=65535)])
def test_sizes_beyond_one_launch(gelim, sizes):
    from gelim import _native
    from gelim.ops import adapter

    v = dict(r=16) | sizes
    grad = v["T"] == 100
    with pytest.raises(_native.GelimError, match="one launch"):
        adapter._workspace_bytes(grad, 1, v["T"], v["K"], v["N"], v["r"], v["n"], v["K"], v["N"], 0, v["r"], 0, v["N"], 0,
                                 v["N"], 0, 0, 0, True)
    # as many rows as one launch takes
    assert adapter._workspace_bytes(False, 1, 2 ** 26, 64, 64, 16, 1, 64, 64, 0, 16, 0, 64, 0, 64, 0, 0, 0, False) > 0
