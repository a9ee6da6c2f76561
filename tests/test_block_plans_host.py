"""How the linear layer's calls are planned, as their workspace queries show it: host
arithmetic, no GPU calls."""
import pytest


@pytest.fixture(scope="module")
def mx():
    from torch_vulkan import mx as m
    m.lib()
    return m


GIB = 1 << 30


def padded(v):
    return -(-v // 128) * 128


def planes(m, k, n, backward):
    """Bytes of the packed operands alone."""
    m, k, n = padded(m), padded(k), padded(n)
    return 4 * (m * k + n * k + (m * n if backward else 0))


@pytest.mark.parametrize("m,k,n", [(65536, 4096, 16384), (32768, 16384, 16384), (4096, 1024, 4096)])
def test_large_forwards_are_packed(mx, m, k, n):
    """Whose operands are far below the bound, and half as long in the other form."""
    got = mx.linear_workspace(m, k, n, mx.ACT_GELU)
    assert planes(m, k, n, False) <= got <= planes(m, k, n, False) * 1.1 + (64 << 20)


@pytest.mark.parametrize("m,k,n", [(32768, 4096, 16384), (4096, 1024, 4096), (65536, 1024, 4096)])
def test_large_backwards_are_packed(mx, m, k, n):
    got = mx.linear_workspace(m, k, n, mx.ACT_GELU, True)
    assert got >= planes(m, k, n, True) + 4 * m * n


@pytest.mark.parametrize("m,k,n", [(3300000, 129, 129), (2500000, 65, 257), (200000, 129, 129), (50000, 130, 130)])
def test_narrow_operands_are_not_padded_to_twice_their_size(mx, m, k, n):
    """dz, sums and a K split's partials alone."""
    assert mx.linear_workspace(m, k, n, mx.ACT_GELU, True) <= 4 * m * n + (160 << 20)


@pytest.mark.parametrize("m,k,n,backward", [(1 << 20, 4096, 4096, False), (1 << 18, 16384, 16384, False), (1 << 17, 8192, 8192, True),
                                            (3000000, 512, 768, True), (5000000, 300, 300, True), (1 << 16, 16384, 16384, True)])
def test_no_call_takes_more_than_the_bound(mx, m, k, n, backward):
    """8 GiB of packed operands and dz, and what little counts, sums and partials take."""
    got = mx.linear_workspace(m, k, n, mx.ACT_GELU, backward)
    assert got <= max(8 * GIB, 4 * m * n * backward) + 17 * 4 * (m + n + k) + (256 << 20)
    if planes(m, k, n, backward) + 4 * m * n * backward > 8 * GIB:
        assert got <= 4 * m * n * backward + (160 << 20), "in tiles"


# ------------------------------------------------ overlapping buffers of one call
def refused(mx, call, *args):
    with pytest.raises(mx.MXError) as e:
        mx.check(getattr(mx.lib(), call)(*args))
    return e.value


AT = 1 << 20   # addresses that no refused call reads
SIZE = 8 * 9 * 4


def matrices(mx, *rows):
    return (mx.MatrixPair * len(rows))(*[mx.MatrixPair(i, o, 8, 9) for i, o in rows]), len(rows)


@pytest.mark.parametrize("rows", [
    [(AT, 2 * AT), (3 * AT, 2 * AT)],                    # one output twice
    [(AT, 2 * AT), (3 * AT, 2 * AT + SIZE - 4)],         # the last element of one
    [(AT, 2 * AT), (2 * AT + 4, 3 * AT)],                # an output under another's input
    [(AT, AT + 4)],                                      # its own input, not whole
    [(AT, 2 * AT), (2 * AT - 4, 2 * AT - 4)],
    [(2 * AT, 2 * AT), (2 * AT, 4 * AT)],                # in place, and another's input
])
def test_orthogonalize_refuses_overlaps(mx, rows):
    import ctypes as C
    arr, count = matrices(mx, *rows)
    ns = mx.NewtonSchulz(5, 3.4445, -4.775, 2.0315, 1e-7)
    e = refused(mx, "mx_orthogonalize", arr, count, C.byref(ns), AT // 2, 1 << 30, None)
    assert e.status == mx.MX_ERR_INVALID and "overlaps" in str(e)


@pytest.mark.parametrize("rows", [
    [(AT, 2 * AT, 3 * AT), (AT, 4 * AT, 5 * AT)],             # a parameter twice
    [(AT, 2 * AT, 3 * AT), (4 * AT, 5 * AT, 3 * AT)],         # a momentum buffer twice
    [(AT, 2 * AT, AT)],                                       # its own parameter as its momentum
    [(AT, AT, 3 * AT)],                                       # as its gradient
    [(AT, 2 * AT, 3 * AT), (AT + SIZE - 4, 4 * AT, 5 * AT)],  # views of one storage
    [(AT, 2 * AT, 3 * AT), (4 * AT, 3 * AT + 40, 5 * AT)],    # a gradient over another's momentum
])
def test_muon_refuses_overlaps(mx, rows):
    import ctypes as C
    arr = (mx.MuonTensor * len(rows))(*[mx.MuonTensor(p, g, m, 8, 9) for p, g, m in rows])
    hp = mx.MuonHParams(0.02, 0.1, 0.95, 1, 0, mx.NewtonSchulz(5, 3.4445, -4.775, 2.0315, 1e-7))
    e = refused(mx, "mx_muon_step", arr, len(rows), C.byref(hp), AT // 2, 1 << 30, None)
    assert e.status == mx.MX_ERR_INVALID and "overlaps" in str(e)
