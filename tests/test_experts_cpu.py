"""The routed feed-forward and 8-bit entries without a GPU: what they refuse,
before any device work, and the empty calls that they accept."""
import ctypes

from chelis_b200 import lib as L

OK, DOMAIN, UNSUPPORTED = 0, 1, 4


def test_router_and_row_entries_refuse():
    lib = L.load()
    one = ctypes.c_void_p(16)  # never read
    route = lib.chelis_cuda_expert_route
    assert route(L.DTYPE_F32, None, 0, 4, 2, 1, None, None) == OK
    assert route(L.DTYPE_F64, one, 1, 4, 2, 1, one, one) == UNSUPPORTED
    assert route(L.DTYPE_F32, one, 1, 4, 5, 1, one, one) == DOMAIN
    assert route(L.DTYPE_F32, one, 1, 4, 0, 1, one, one) == DOMAIN
    assert route(L.DTYPE_F32, one, -1, 4, 1, 1, one, one) == DOMAIN
    assert route(L.DTYPE_F32, one, 1, 2000, 1, 1, one, one) == UNSUPPORTED
    assert route(L.DTYPE_F32, one, 1, 40, 33, 1, one, one) == UNSUPPORTED
    assert route(L.DTYPE_F32, one, 1 << 30, 40, 4, 1, one, one) == UNSUPPORTED
    assert route(L.DTYPE_F32, None, 1, 4, 2, 1, one, one) == DOMAIN
    assert "expert_route" in L.last_error()
    assert lib.chelis_cuda_expert_route_bwd(L.DTYPE_F32, one, None, one, 1, 4, 2, 1, one) == DOMAIN
    sort = lib.chelis_cuda_expert_sort
    assert sort(one, 1, 33, 4, one, one, one) == UNSUPPORTED
    assert sort(one, 1, 1, 1025, one, one, one) == UNSUPPORTED
    assert sort(one, 1 << 31, 1, 4, one, one, one) == UNSUPPORTED
    assert sort(one, 1, 1, 4, None, one, one) == DOMAIN
    assert sort(None, 1, 1, 4, one, one, one) == DOMAIN
    assert lib.chelis_cuda_expert_spread(L.DTYPE_F32, None, one, one, 1, 1, 8, one) == DOMAIN
    assert lib.chelis_cuda_expert_spread(L.DTYPE_F32, None, None, None, 0, 1, 8, None) == OK
    assert lib.chelis_cuda_expert_spread(L.DTYPE_I32, one, one, one, 1, 1, 8, one) == UNSUPPORTED
    assert lib.chelis_cuda_expert_combine(L.DTYPE_F32, one, one, one, 1, 1, -8, one) == DOMAIN
    assert lib.chelis_cuda_expert_combine_bwd(L.DTYPE_BF16, one, one, None, one, one, 1, 1, 8, one, one) == DOMAIN


def test_8_bit_entries_refuse():
    lib = L.load()
    one, odd = ctypes.c_void_p(16), ctypes.c_void_p(8)
    quant = lib.chelis_cuda_quantize8
    assert quant(L.DTYPE_F64, 0, 0, one, 1, 4, 4, one, one) == UNSUPPORTED
    assert quant(L.DTYPE_F32, 2, 0, one, 1, 4, 4, one, one) == UNSUPPORTED
    assert quant(L.DTYPE_F32, 0, 2, one, 1, 4, 4, one, one) == DOMAIN
    assert quant(L.DTYPE_F32, 0, L.BLOCKS_ROWS, one, 2, 4, 4, one, one) == DOMAIN
    assert quant(L.DTYPE_F32, 0, 0, one, 1, -4, 4, one, one) == DOMAIN
    assert quant(L.DTYPE_F32, 0, 0, one, 1, 4, 4, odd, one) == DOMAIN
    assert quant(L.DTYPE_F32, 0, 0, None, 1, 0, 4, None, None) == OK
    places = lib.chelis_cuda_quantize8_places
    assert [places(0, 0), places(1, 0), places(128, 0), places(129, 0)] == [0, 128, 128, 256]
    assert [places(0, 3), places(300, 3)] == [384, 640]
    assert places(-1, 0) == -1
    turned = lib.chelis_cuda_quantize8_transposed
    assert turned(L.DTYPE_F32, 0, one, None, 3, 4, 4, one, one) == DOMAIN
    assert turned(L.DTYPE_F32, 0, one, one, 0, 4, 4, one, one) == DOMAIN
    assert turned(L.DTYPE_F32, 0, one, one, 1025, 4, 4, one, one) == UNSUPPORTED
    product = lib.chelis_cuda_matmul8
    assert product(0, 0, 1, 0, 4, 4, None, None, None, None, None, 1, 0, L.DTYPE_F32, None) == OK
    assert product(0, 2, 1, 4, 4, 4, one, one, one, one, None, 1, 0, L.DTYPE_F32, one) == UNSUPPORTED
    assert product(0, 0, 1, 4, 4, 4, one, one, one, one, None, 1, 0, L.DTYPE_F64, one) == UNSUPPORTED
    assert product(0, 0, 1, 4, 4, 4, one, one, one, one, None, 2, 0, L.DTYPE_F32, one) == DOMAIN
    assert product(0, 0, 1, 4, 4, 4, one, one, one, one, one, 1025, 0, L.DTYPE_F32, one) == UNSUPPORTED
    assert product(0, 0, 1, 4, 4, 4, odd, one, one, one, None, 1, 0, L.DTYPE_F32, one) == DOMAIN
    assert product(0, 0, 1, 4, -4, 4, one, one, one, one, None, 1, 0, L.DTYPE_F32, one) == DOMAIN
    assert product(0, 0, 1, 4, 1 << 31, 4, one, one, one, one, None, 1, 0, L.DTYPE_F32, one) == UNSUPPORTED
    wgrad = lib.chelis_cuda_matmul8_wgrad
    assert wgrad(0, 0, 4, 4, 100, one, one, one, one, None, 1, 0, L.DTYPE_F32, one) == DOMAIN
    assert "places" in L.last_error()
    assert wgrad(0, 0, 0, 4, 128, None, None, None, None, None, 1, 0, L.DTYPE_F32, None) == OK
