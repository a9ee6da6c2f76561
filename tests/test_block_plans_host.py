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
