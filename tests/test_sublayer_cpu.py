"""The entries of the 16-bit feed-forward sublayer without a GPU: what they
refuse, before any device work, and the empty calls that they accept; the
reference functions that the GPU tests compare with, against differences."""
import ctypes

import numpy as np
import pytest

import _sublayer_ref as S
from chelis_b200 import lib as L
from chelis_b200 import ops

OK, DOMAIN, UNSUPPORTED = 0, 1, 4
BF, F32 = L.DTYPE_BF16, L.DTYPE_F32


def test_product_entries_refuse():
    lib = L.load()
    one = ctypes.c_void_p(16)  # never read

    def product(dtype=BF, m=4, n=4, k=4, a=one, b=one, bias=None, bias_dtype=0, act=0, residual=None, through=None,
                pre=None, out_dtype=BF, out=one):
        return lib.chelis_cuda_matmul16(dtype, 0, 0, m, n, k, a, b, bias, bias_dtype, act, residual, through, pre, out_dtype, out)

    assert product(m=0, a=None, b=None, out=None) == OK and product(n=0) == OK
    assert product(dtype=F32) == UNSUPPORTED
    assert product(act=4) == UNSUPPORTED and product(act=-1) == UNSUPPORTED
    assert product(out_dtype=L.DTYPE_F16) == UNSUPPORTED
    assert product(bias=one, bias_dtype=L.DTYPE_F16) == UNSUPPORTED
    assert product(m=-1) == DOMAIN and product(k=-1) == DOMAIN
    assert product(n=1 << 31) == UNSUPPORTED
    assert product(a=None) == DOMAIN and product(out=None) == DOMAIN
    assert product(through=one, pre=one) == DOMAIN and product(through=one, residual=one) == DOMAIN
    assert "through" in L.last_error()
    act = lib.chelis_cuda_activation16_bwd
    assert act(BF, 1, None, None, 0, None) == OK
    assert act(F32, 1, one, one, 4, one) == UNSUPPORTED and act(BF, 9, one, one, 4, one) == UNSUPPORTED
    assert act(BF, 1, one, one, -4, one) == DOMAIN and act(BF, 1, one, None, 4, one) == DOMAIN
    sums = lib.chelis_cuda_column_sums16
    assert sums(BF, None, 4, 0, None) == OK
    assert sums(F32, one, 4, 4, one) == UNSUPPORTED and sums(BF, one, -1, 4, one) == DOMAIN
    assert sums(BF, None, 4, 4, one) == DOMAIN and sums(BF, one, 4, 4, None) == DOMAIN


def test_norm_entries_refuse():
    lib = L.load()
    one = ctypes.c_void_p(16)

    def norm(dtype=F32, kind=0, rows=4, hidden=8, x=one, branch=one, pg=None, pb=None, gate=None, groups=1, scale=1.0,
             g2=None, b2=None, y=one, h=None):
        return lib.chelis_cuda_residual_norm(dtype, kind, rows, hidden, x, branch, pg, pb, gate, groups, scale, g2, b2, 1e-5, y, h)

    assert norm(rows=0) == OK and norm(hidden=0) == OK
    assert norm(dtype=L.DTYPE_F64) == UNSUPPORTED and norm(kind=2) == UNSUPPORTED and norm(hidden=8193) == UNSUPPORTED
    assert norm(rows=-1) == DOMAIN and norm(groups=3) == DOMAIN and norm(groups=0) == DOMAIN
    assert norm(pb=one) == DOMAIN and norm(b2=one) == DOMAIN and norm(y=None) == DOMAIN and norm(g2=one) == DOMAIN
    assert norm(branch=None, y=None, g2=one, h=one, scale=0.5) == DOMAIN
    assert norm(branch=None, y=None, gate=one, g2=one, h=one) == DOMAIN
    assert norm(branch=None, y=None) == DOMAIN

    def bwd(dtype=F32, rows=4, dy=one, dh=None, y=one, branch=one, pg=None, pb=None, gate=None, groups=1, g2=None, dx=one,
            dbranch=one, dpg=None, dpb=None, dgate=None, dg2=None, db2=None):
        return lib.chelis_cuda_residual_norm_bwd(dtype, 0, rows, 8, dy, dh, y, branch, pg, pb, gate, groups, 1.0, g2, 1e-5, dx,
                                                 dbranch, dpg, dpb, dgate, dg2, db2)

    assert bwd(rows=0) == OK
    assert bwd(dy=None) == DOMAIN and bwd(dx=None) == DOMAIN and bwd(dh=one) == DOMAIN and bwd(g2=one) == DOMAIN
    assert bwd(dpg=one) == DOMAIN and bwd(dgate=one) == DOMAIN and bwd(dg2=one) == DOMAIN
    assert bwd(pg=one, branch=None) == DOMAIN and bwd(gate=one, dbranch=None) == DOMAIN
    assert bwd(gate=one, groups=3) == DOMAIN


def test_balance_entries_refuse():
    lib = L.load()
    one = ctypes.c_void_p(16)
    f, b = lib.chelis_cuda_expert_balance, lib.chelis_cuda_expert_balance_bwd
    assert f(F32, one, one, None, 4, 8, 9, one, one) == DOMAIN and f(F32, one, one, None, -1, 8, 2, one, one) == DOMAIN
    assert f(F32, one, one, None, 4, 2000, 2, one, one) == UNSUPPORTED
    assert f(L.DTYPE_F64, one, one, None, 4, 8, 2, one, one) == UNSUPPORTED
    assert f(F32, None, one, None, 4, 8, 2, one, one) == DOMAIN and f(F32, one, one, None, 4, 8, 2, None, one) == DOMAIN
    assert b(F32, None, None, None, 0, 8, 2, 1.0, None, None, None) == OK
    assert b(F32, one, None, None, 4, 8, 2, 1.0, None, None, one) == DOMAIN
    assert b(F32, one, one, None, 4, 8, 0, 1.0, None, None, one) == DOMAIN


def _list(*tensors):
    """(n, data, counts, dtypes) of (address, count, dtype)."""
    n = len(tensors)
    return (n, (ctypes.c_void_p * n)(*[t[0] for t in tensors]), (ctypes.c_int64 * n)(*[t[1] for t in tensors]),
            (ctypes.c_int32 * n)(*[t[2] for t in tensors]))


def test_gradient_lists_refuse():
    lib = L.load()
    one = ctypes.c_void_p(16)
    norm = lib.chelis_cuda_grad_norm
    assert norm(-1, None, None, None, one) == DOMAIN and norm(1, None, None, None, one) == DOMAIN
    assert norm(*_list((64, 4, L.DTYPE_F64)), one) == UNSUPPORTED
    assert norm(*_list((64, -4, F32)), one) == DOMAIN and norm(*_list((None, 4, F32)), one) == DOMAIN
    assert norm(*_list((66, 4, F32)), one) == DOMAIN and norm(*_list((64, 4, F32)), None) == DOMAIN

    def clip(src, dst, bound=1.0):
        n, data, counts, dtypes = _list(*src)
        _, out, _, out_dtypes = _list(*dst)
        return lib.chelis_cuda_clip_grads(n, data, counts, dtypes, out, out_dtypes, bound, one)

    a, b = (1024, 64, F32), (2048, 64, F32)
    assert clip([a], [a], -1.0) == DOMAIN and clip([a], [a], float("nan")) == DOMAIN
    assert clip([a, a], [a, a]) == DOMAIN and "overlap" in L.last_error()
    assert clip([a, b], [b, a]) == DOMAIN and clip([a, (1024 + 252, 64, F32)], [a, (1024 + 252, 64, F32)]) == DOMAIN
    assert clip([a], [(1024, 64, BF)]) == DOMAIN and clip([a], [(1028, 64, F32)]) == DOMAIN
    assert clip([a], [(900, 64, BF)]) == DOMAIN  # [900, 1028)
    assert clip([a, b], [(4096, 64, F32), (4096 + 128, 64, F32)]) == DOMAIN
    assert clip([a], [(None, 64, F32)]) == DOMAIN and clip([a], [(4096, 64, L.DTYPE_F64)]) == UNSUPPORTED


def test_packed_entries_take_their_arguments_in_order():
    """Each entry packed refuses what it refuses called by its arguments, with the
    same message; the last argument is looked at too."""
    import struct
    lib = L.load()

    def same(entry, fmt, direct, *args):
        status = direct(*args)
        text = L.last_error()
        packed = struct.pack("=q" + fmt, 0, *[0 if a is None else a for a in args])
        assert lib.chelis_cuda_call_packed(entry, packed) == status != OK and L.last_error() == text

    P = 1 << 40  # never read
    f = lib.chelis_cuda_matmul16
    good = (BF, 0, 1, 4, 5, 6, P, P, P, BF, 2, P, None, P, BF, P)
    for i, bad in ((0, F32), (3, -1), (4, 1 << 31), (5, -1), (6, None), (7, None), (9, L.DTYPE_F16), (10, 9), (12, P), (14, L.DTYPE_F16),
                   (15, None)):
        same(L.PACKED_MATMUL16, "16q", f, *good[:i], bad, *good[i + 1:])
    same(L.PACKED_ACTIVATION16_BWD, "6q", lib.chelis_cuda_activation16_bwd, BF, 1, P, P, 4, None)
    same(L.PACKED_ACTIVATION16_BWD, "6q", lib.chelis_cuda_activation16_bwd, BF, 1, P, P, -4, P)
    same(L.PACKED_COLUMN_SUMS16, "5q", lib.chelis_cuda_column_sums16, BF, P, 4, 4, None)
    f = lib.chelis_cuda_residual_norm
    good = (F32, 1, 4, 8, P, P, P, P, P, 2, 0.5, P, P, 1e-5, P, P)
    for i, bad in ((0, 9), (1, 2), (2, -1), (3, 9000), (4, None), (5, None), (6, None), (9, 3), (11, None), (14, None), (15, None)):
        same(L.PACKED_RESIDUAL_NORM, "10qd2qd2q", f, *good[:i], bad, *good[i + 1:])
    same(L.PACKED_RESIDUAL_NORM, "10qd2qd2q", f, F32, 1, 4, 8, P, None, None, None, None, 1, 0.5, P, P, 1e-5, None, P)
    f = lib.chelis_cuda_residual_norm_bwd
    good = (F32, 1, 4, 8, P, P, P, P, P, P, P, 2, 0.5, P, 1e-5, P, P, P, P, P, P, P)
    for i, bad in ((0, 9), (2, -1), (5, None), (6, None), (7, None), (8, None), (10, None), (11, 3), (13, None), (15, None), (16, None)):
        same(L.PACKED_RESIDUAL_NORM_BWD, "12qdqd7q", f, *good[:i], bad, *good[i + 1:])
    f = lib.chelis_cuda_expert_balance
    good = (F32, P, P, None, 4, 8, 2, P, P)
    for i, bad in ((0, 9), (1, None), (2, None), (4, -1), (5, 2000), (6, 9), (7, None), (8, None)):
        same(L.PACKED_EXPERT_BALANCE, "9q", f, *good[:i], bad, *good[i + 1:])
    f = lib.chelis_cuda_expert_balance_bwd
    good = (F32, P, P, None, 4, 8, 2, 1.0, None, None, P)
    for i, bad in ((0, 9), (1, None), (2, None), (4, -1), (6, 0), (10, None)):
        same(L.PACKED_EXPERT_BALANCE_BWD, "7qd3q", f, *good[:i], bad, *good[i + 1:])
    n, data, counts, dtypes = _list((1024, 64, F32))
    at = [ctypes.addressof(v) for v in (data, counts, dtypes)]
    same(L.PACKED_GRAD_NORM, "5q", lib.chelis_cuda_grad_norm, n, *at, None)
    same(L.PACKED_GRAD_NORM, "5q", lib.chelis_cuda_grad_norm, -1, *at, P)
    same(L.PACKED_CLIP_GRADS, "6qdq", lib.chelis_cuda_clip_grads, n, *at, at[0], at[2], -1.0, P)
    same(L.PACKED_CLIP_GRADS, "6qdq", lib.chelis_cuda_clip_grads, n, *at, at[0], at[2], 1.0, None)
    assert lib.chelis_cuda_call_packed(99, struct.pack("=q", 0)) == UNSUPPORTED
    assert lib.chelis_cuda_call_packed(0, None) == DOMAIN


class _Fake:
    def __init__(self, device, contiguous=True):
        self.device_index, self.contiguous = device, contiguous

    def get_device(self):
        return self.device_index

    def is_contiguous(self):
        return self.contiguous


def test_tensors_lie_on_the_current_device(monkeypatch):
    monkeypatch.setattr(ops.torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops, "_initialised", {0, 1})
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    ops._begin("op", _Fake(0), None, _Fake(0))
    for tensors in ((_Fake(0), _Fake(1)), (_Fake(1),), (_Fake(-1),), (_Fake(0, False),)):
        with pytest.raises(ValueError):
            ops._begin("op", *tensors)


def test_host_tensors_are_refused():
    import torch
    a, x = torch.zeros(4, 4, dtype=torch.bfloat16), torch.zeros(4, 4)
    for bad in (lambda: ops.matmul16(a, a), lambda: ops.residual_norm(x, x), lambda: ops.grad_norm([x]),
                lambda: ops.expert_balance(x, x.int()), lambda: ops.clip_grads([x], 1.0), lambda: ops.column_sums16(a)):
        with pytest.raises(ValueError, match="CUDA tensors"):
            bad()


@pytest.mark.parametrize("name", ["relu", "gelu", "silu"])
def test_reference_slopes_against_differences(name):
    z = np.linspace(-6, 6, 241) + 0.003
    numeric = (S.act(z + 1e-6, name)[0] - S.act(z - 1e-6, name)[0]) / 2e-6
    assert np.abs(numeric - S.act(z, name)[1]).max() < 1e-8
    assert np.abs(S.act(z, name)[1]).max() <= S.STEEP[name]


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_reference_norm_gradients_against_differences(kind):
    rng = np.random.default_rng(0)
    rows, hidden = 6, 10
    p = dict(post_gamma=rng.standard_normal(hidden), post_beta=rng.standard_normal(hidden), gate=rng.standard_normal((3, hidden)),
             pre_gamma=rng.standard_normal(hidden), pre_beta=rng.standard_normal(hidden), scale=0.7, eps=1e-5, kind=kind)
    at = dict(p, x=rng.standard_normal((rows, hidden)), branch=rng.standard_normal((rows, hidden)))
    dy, dh = rng.standard_normal((2, rows, hidden))

    def loss(v):
        y, _, h, _ = S.join(v["x"], v["branch"], v)
        return float((dy * y + dh * h).sum())

    grads = S.join_bwd(dy, dh, S.join(at["x"], at["branch"], p)[0], at["branch"], p)
    for name in ("x", "branch", "post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta"):
        d = rng.standard_normal(at[name].shape)
        numeric = (loss(dict(at, **{name: at[name] + 1e-6 * d})) - loss(dict(at, **{name: at[name] - 1e-6 * d}))) / 2e-6
        assert abs(numeric - (grads["d" + name][0] * d).sum()) < 1e-6


def _kernel(file, name):
    """The source of a kernel, from its name to the brace that ends it."""
    import os
    from chelis_b200 import build
    text = open(os.path.join(build.CSRC, file)).read()
    return text[text.index(f"    {name}("):].split("\n}\n")[0]


def test_gradients_that_may_be_results_are_no_read_only_data():
    """activation16_bwd's dz may be dy: neither may be promised to the compiler as
    read alone, by __restrict__ or by __ldg."""
    text = _kernel("linear16.cu", "act_bwd_kernel")
    assert "const T *dy" in text and "T *dz" in text and "__ldg" not in text and "load_pack<T, VEC>(dy" not in text


def test_numbers_that_are_clipped_in_place_are_no_read_only_data():
    """One launch reads few numbers for their norm and scales them: by plain loads."""
    text = _kernel("clip.cu", "small_kernel")
    assert "squares_part<32, !SCALE>" in text and "__restrict__" not in text and "__ldg" not in text
