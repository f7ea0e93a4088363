"""What the adapter calls ask for as workspace: no more than the call at hand uses.  Sizes only, no GPU."""
import pytest

MIB = 2 ** 20


def need(grad, T, K, N, r, n, dtype=1, indexed=True, x=0, w=0, y=0, wt=0):
    from gelim.ops import adapter

    return adapter._workspace_bytes(grad, dtype, T, K, N, r, n, K, K if wt else N, wt, r, 0, N, 0, N, x, w, y, indexed)


@pytest.mark.parametrize("T", [5, 128])
def test_no_parts_where_no_adapter_has_two_pieces(gelim, T):
    """Up to 128 rows the factor gradients are written without parts to add up: three layouts of the factors (two of B's
    and A's sums, one of A's columns) and what belongs to the rows is all there is: at most 16 parts of dX, as the
    large product's sum is cut into no more, and per row less than 1 KB of low-rank sums at this rank."""
    K, N, r, n = 4096, 4096, 16, 2000
    layouts = n * r * (2 * K + N) * 2
    assert need(True, T, K, N, r, n) <= layouts + 16 * T * K * 4 + T * 1024 + MIB


@pytest.mark.parametrize("T", [100, 1000])
def test_results_that_are_not_wanted_need_no_room(gelim, T):
    """Each of the three results alone: the copies and layouts that it reads.  X one element behind a multiple of 16 bytes
    is copied, 2 T K bytes and less than a page to fill rows up, for dA and dB only."""
    K, N, r, n = 4096, 2048, 16, 40
    layout = {"A as columns of S": n * r * K * 2, "B as columns of D": n * r * N * 2, "A as rows": n * r * K * 2}
    whole = need(True, T, K, N, r, n, x=2)
    dX, dA, dB = (need(tuple(k == j for j in range(3)), T, K, N, r, n, x=2) for k in range(3))
    copy = T * K * 2
    assert max(dX, dA, dB) < whole
    assert dX <= whole - copy - layout["A as columns of S"]
    assert dA <= whole - layout["A as columns of S"] - layout["A as rows"]
    assert dB <= whole - layout["B as columns of D"] - layout["A as rows"]
    assert need((False, True, True), T, K, N, r, n, x=2) - need((False, True, True), T, K, N, r, n) >= copy
    assert need((True, False, False), T, K, N, r, n, x=2) == need((True, False, False), T, K, N, r, n)
    assert need((False, False, False), T, K, N, r, n, x=2) == 0


@pytest.mark.parametrize("T", [130, 200, 3000])
def test_pieces_go_by_rows_not_by_resident_adapters(gelim, T):
    """Beyond as many adapters as rows another one costs its layouts and its entry of the order, no parts of gradients."""
    K, N, r = 1024, 2048, 64
    more = need(True, T, K, N, r, T + 300) - need(True, T, K, N, r, T)
    assert more <= 300 * (r * (2 * K + N) * 2 + 4) + 1024


@pytest.mark.parametrize("T", [128, 200])
def test_small_batch_beside_many_adapters(gelim, T):
    """What one piece a row would need, the most that rows can be cut into, for both gradients in fp32."""
    K, N, r, n = 8192, 8192, 64, 500
    layouts, parts = n * r * (2 * K + N) * 2, (T // 32 + T) * r * (K + N) * 4
    assert need(True, T, K, N, r, n) <= layouts + parts + 16 * T * K * 4 + T * 8192


def test_no_rows_need_the_same_with_and_without_an_index(gelim):
    """An index of no rows has no address, so the call cannot tell the two apart."""
    for grad in (False, True):
        assert need(grad, 0, 64, 48, 4, 2) == need(grad, 0, 64, 48, 4, 2, indexed=False)


@pytest.mark.parametrize("T", [65, 200, 3000, 8192])
def test_layouts_go_by_rows_not_by_resident_adapters(gelim, T):
    """Beyond as many adapters as rows another one costs its entry of the order."""
    for grad in (False, True):
        assert need(grad, T, 1024, 2048, 64, T + 300) - need(grad, T, 1024, 2048, 64, T) <= 300 * 4 + 1024


@pytest.mark.parametrize("T, r, padded", [(200, 64, 64), (1000, 8, 16), (4000, 33, 64)])
def test_parts_are_those_of_adapters_with_several_pieces(gelim, T, r, padded):
    """Rows in pieces of 32 at least: adapters of more than one piece have no more than twice T / 32 together.  Beside
    those the layouts with their ranks padded, dX's parts and per row the low-rank sums."""
    K, N, n = 8192, 4096, 500
    layouts, parts = min(n, T) * padded * (2 * K + N) * 2, 2 * (T // 32) * padded * (K + N) * 4
    assert need(True, T, K, N, r, n) <= layouts + parts + 16 * T * K * 4 + T * 8192
