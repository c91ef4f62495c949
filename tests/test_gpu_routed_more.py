"""Paths of the routed feed-forward and 8-bit operators that small random
cases do not reach: kernels' second turns of their grid, special values in every
layout and type, unaligned bases, the block-scaled product's ways of storing,
part boundaries, side streams and captured graphs.

Comparisons are equality wherever the arithmetic is exact: quantising rounds
once, and products of small integers are exact.  Which product kernel a case
takes is asserted by its number of launches.
"""
import numpy as np
import pytest

import _experts_ref as R

pytestmark = pytest.mark.gpu

TYPES = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def _dtype(name):
    import torch
    return getattr(torch, TYPES[name])


@pytest.fixture(autouse=True)
def _seed():
    import torch
    torch.manual_seed(1)


def _same(got, ref):
    assert got.shape == ref.shape
    assert ((got == ref) | (np.isnan(got) & np.isnan(ref))).all()


def _values(data):
    return data.float().cpu().double().numpy()


# ------------------------------------------------------------- quantisers

def _special(shape, dtype, seed):
    """Random numbers with infinities, NaNs, the type's extremes and zeros in
    some blocks; whole blocks of zeros, of NaN and of infinities."""
    import torch
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    x *= torch.exp2(torch.randint(-8, 9, (*shape[:-1], 1), generator=gen).float())
    x = x.to(_dtype(dtype))
    info = torch.finfo(_dtype(dtype))
    odd = torch.tensor([float("inf"), float("-inf"), float("nan"), info.max, -info.max, info.tiny, -0.0,
                        info.smallest_normal / 4], dtype=torch.float64).to(_dtype(dtype))
    flat = x.reshape(-1)
    at = torch.randperm(flat.numel(), generator=gen)[:max(8, flat.numel() // 1500)]
    flat[at] = odd[torch.arange(at.numel()) % odd.numel()]
    rows = x.shape[-2]
    x[..., : min(rows, 3), :] = 0.0
    if rows > 140:
        x[..., 5, :] = float("nan")
        x[..., 6, :] = float("inf")
        x[..., 7, :] = info.tiny
    return x


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (40, 264), (150, 257), (300, 520)])
@pytest.mark.parametrize("blocks", ["rows", "tiles", "transposed"])
def test_special_values_in_every_layout(cuda, blocks, rows, cols, dtype, fmt):
    x = _special((rows, cols), dtype, rows + cols)
    xr = x.double().numpy()
    if blocks == "transposed":
        b = cuda.quantize8_transposed(x.cuda(), fmt)
        padded = np.zeros((-(-rows // 128) * 128, cols))
        padded[:rows] = xr
        q, s = R.quantize(np.ascontiguousarray(padded.T), fmt, 1)
        _same(_values(b.data), q)
        _same(b.scales.cpu().double().numpy(), s.T)
        return
    b = cuda.quantize8(x.cuda(), fmt, blocks)
    q, s = R.quantize(xr, fmt, 1 if blocks == "rows" else 128)
    _same(_values(b.data)[:, :cols], q)
    assert not _values(b.data)[:, cols:].any()
    _same(b.scales.cpu().double().numpy(), s.T if blocks == "rows" else s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("blocks", ["rows", "tiles", "transposed"])
def test_quantiser_at_an_odd_address(cuda, blocks, dtype):
    """A base that 16 bytes do not divide gives what an aligned one does."""
    import torch
    base = _special((1, 200 * 256 + 1), dtype, 3).cuda().reshape(-1)
    x = base[1:].view(200, 256)
    assert x.data_ptr() % 16
    for fmt in ("e4m3", "e5m2"):
        make = (lambda v: cuda.quantize8_transposed(v, fmt)) if blocks == "transposed" else \
            (lambda v: cuda.quantize8(v, fmt, blocks))
        got, want = make(x), make(x.clone())
        assert torch.equal(got.data.view(torch.uint8), want.data.view(torch.uint8))
        assert torch.equal(got.scales, want.scales)


def _plain(x, fmt, dim):
    """Data and scales of blocks of 128 along dim by elementary operations: frexp
    and a division by a power of two are exact, the cast rounds once."""
    import torch
    kind = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}[fmt]
    v = x.double().unflatten(dim, (-1, 128))
    top = v.abs().amax(dim + 1, keepdim=True)
    f, e = torch.frexp(top)
    e = e - (9 if fmt == "e4m3" else 16) + (f > 0.875).int()
    s = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e.clamp(min=-126)), torch.ones_like(top))
    return (v / s).float().to(kind).flatten(dim, dim + 1), s.squeeze(dim + 1).float()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_quantisers_second_turn_of_the_grid(cuda, dtype):
    """More tiles than resident blocks, so that each kernel's loop runs again
    over its shared memory."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((20480, 2048), generator=gen, device="cuda").to(_dtype(dtype))
    q, s = _plain(x, "e4m3", 1)
    b = cuda.quantize8(x)
    assert torch.equal(b.data.view(torch.uint8), q.view(torch.uint8)) and torch.equal(b.scales, s.t())
    q, s = _plain(x, "e5m2", 0)
    b = cuda.quantize8_transposed(x, "e5m2")
    assert torch.equal(b.data.view(torch.uint8), q.t().view(torch.uint8)) and torch.equal(b.scales, s)
    b = cuda.quantize8(x.view(4, 5120, 2048), "e4m3", "tiles")
    v = x.view(4, 40, 128, 16, 128).transpose(2, 3).reshape(4, 40, 16, 128 * 128)
    top = v.double().abs().amax(-1)
    f, e = torch.frexp(top)
    s = torch.ldexp(torch.ones_like(top), e - 9 + (f > 0.875).int())
    assert torch.equal(b.scales, s.float())
    want = (v.double() / s[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(b.data.view(torch.uint8).view(4, 40, 128, 16, 128).transpose(2, 3).reshape(want.shape), want)


@pytest.mark.parametrize("groups", [300, 1024])
def test_quantise_transposed_by_many_experts(cuda, groups):
    import torch
    rng = np.random.default_rng(groups)
    rows, cols = 3000, 40
    counts = rng.multinomial(rows - 7, rng.dirichlet(np.ones(groups)))
    off = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    x = torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32))
    b = cuda.quantize8_transposed(x.cuda(), "e5m2", off)
    padded = np.zeros(((rows // 128 + groups) * 128, cols))
    at = row = 0
    for c in counts:
        padded[at:at + c] = x[row:row + c].numpy()
        row += c
        at += -(-c // 128) * 128
    q, s = R.quantize(np.ascontiguousarray(padded.T), "e5m2", 1)
    _same(_values(b.data), q)
    _same(b.scales.cpu().double().numpy(), s.T)


def test_quantise_transposed_looks_its_rows_up_at_once(cuda):
    """1024 experts of 16 rows and one matrix of as many blocks of 128 take the
    same tiles, and the experts' read an eighth of the data: finding a tile's
    rows may not cost more than the tile itself."""
    import torch

    def us(rows, off):
        x = torch.randn((rows, 1024), device="cuda").bfloat16()
        cuda.quantize8_transposed(x, "e4m3", off)
        best = float("inf")
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                cuda.quantize8_transposed(x, "e4m3", off)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 100)
        return best
    off = (torch.arange(1025, device="cuda") * 16).int()
    assert us(16384, off) <= 2 * us((128 + 1024) * 128, None)


# --------------------------------------------------- rows there and back

@pytest.mark.parametrize("dtype,hidden", [("f32", 64), ("bf16", 65)])
def test_rows_second_turn_of_the_grid(cuda, dtype, hidden):
    """12000 tokens of 8 slots, integers: every sum is exact."""
    import torch
    rng = np.random.default_rng(hidden)
    t, k, experts = 12000, 8, 16
    ids = np.argsort(rng.random((t, experts)), 1)[:, :k].astype(np.int32)
    ids[rng.random(ids.shape) < 0.05] = -1
    order = cuda.expert_sort(torch.from_numpy(ids).cuda(), experts)
    position, source = order.position.long(), order.source.long()
    x = torch.randint(-4, 5, (t, hidden), device="cuda").to(_dtype(dtype))
    ys = torch.randint(-4, 5, (t * k, hidden), device="cuda").to(_dtype(dtype))
    w = torch.randint(-2, 3, (t, k), device="cuda").float()
    taken = (source >= 0)[:, None]
    rows = x[source.clamp(min=0) // k]
    assert torch.equal(cuda.expert_gather(x, order), torch.where(taken, rows, torch.zeros_like(rows)))
    there = (position >= 0)[..., None]
    back = torch.where(there, ys[position.clamp(min=0)].float(), torch.zeros(1, device="cuda"))
    assert torch.equal(cuda.expert_gather_bwd(ys, order), back.sum(1).to(ys.dtype))
    assert torch.equal(cuda.expert_combine(ys, w, order), (back * w[..., None]).sum(1).to(ys.dtype))
    dys, dw = cuda.expert_combine_bwd(x, ys, w, order)
    scaled = rows.float() * w.reshape(-1)[source.clamp(min=0)][:, None]
    assert torch.equal(dys, torch.where(taken, scaled, torch.zeros_like(scaled)).to(ys.dtype))
    assert torch.equal(dw, (back * x.float()[:, None]).sum(2))


# ---------------------------------------------------------------- products

def _integers(shape, low, high):
    import torch
    return torch.randint(low, high + 1, shape, device="cuda").float()


def _launches(cuda, call):
    before = cuda.launch_count()
    out = call()
    return out, cuda.launch_count() - before


BLOCK_SCALED, PARTS = 2, 3  # launches: packing and product; and the sums of the parts


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("rows,n,k,counts,dtype", [
    (4700, 2048, 2048, [2500, 0, 1, 2190], "bf16"),   # stored by TMA, ragged ends row by row
    (4700, 2055, 2048, [2500, 0, 1, 2190], "f16"),    # two-byte units
    (4700, 2054, 2048, [2500, 0, 1, 2190], "bf16"),   # four-byte units
    (4700, 2051, 2048, [2500, 0, 1, 2190], "f32"), (4700, 2056, 2040, [1000, 900, 1300, 1500], "f32"),
    (2400, 4099, 2200, None, "f16"), (2400, 4104, 2200, None, "bf16")])
def test_block_scaled_product_stores(cuda, rows, n, k, counts, dtype, trans_b):
    """Enough work for the block-scaled kernel, unsplit: every way in which it
    stores, of groups that end inside a tile.  Integers: sums below 2^24 are
    exact, and the result is rounded once."""
    import torch
    a = _integers((rows, k), -7, 7)
    shape = (n, k) if trans_b else (k, n)
    b = _integers(shape if counts is None else (len(counts), *shape), -3, 3)
    a8, b8 = cuda.quantize8(a), cuda.quantize8(b, "e5m2", "tiles")
    off = None if counts is None else torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    y, launches = _launches(cuda, lambda: cuda.matmul8(a8, b8, trans_b, off, _dtype(dtype)))
    assert launches == BLOCK_SCALED
    at = 0
    for e, c in enumerate([rows] if counts is None else counts):
        w = (b if counts is None else b[e]).double()
        want = a[at:at + c].double() @ (w.t() if trans_b else w)
        assert torch.equal(y[at:at + c], want.to(_dtype(dtype)))
        at += c
    assert not y[at:].any()
    cuda.device_status()


@pytest.mark.parametrize("counts,n,k,dtype,launches", [
    ([2600], 128, 256, "f32", 2), ([9001], 77, 263, "f32", 2), ([3000, 0, 130, 5000, 1], 100, 300, "f32", 2),
    ([60000], 520, 600, "f32", PARTS), ([40000, 0, 15000, 1], 301, 520, "f32", PARTS),
    ([40000, 0, 15000, 700], 520, 264, "bf16", PARTS), ([4300], 1500, 1300, "f32", PARTS),
    ([3000, 0, 130, 5000, 1], 1100, 1032, "bf16", BLOCK_SCALED)])
def test_weight_gradient_of_integers(cuda, counts, n, k, dtype, launches):
    """Whole and in parts, by one block and block-scaled: no block of 128 may be
    missing or counted twice."""
    import torch
    rows = sum(counts)
    dy, x = _integers((rows, n), -3, 3), _integers((rows, k), -3, 3)
    off = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda") if len(counts) > 1 else None
    a8, b8 = cuda.quantize8_transposed(dy, "e5m2", off), cuda.quantize8_transposed(x, "e4m3", off)
    got, n_launches = _launches(cuda, lambda: cuda.matmul8_wgrad(a8, b8, off, _dtype(dtype)))
    assert n_launches == launches
    at = 0
    for e, c in enumerate(counts):
        want = dy[at:at + c].double().t() @ x[at:at + c].double()
        assert torch.equal(got[e] if off is not None else got, want.to(_dtype(dtype)))
        at += c
    cuda.device_status()


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("rows,n,k,counts,launches", [
    (129, 40, 1400, None, 2), (70, 517, 4000, None, 2), (195, 129, 2100, [50, 0, 140], 2),
    (300, 1000, 19200, None, PARTS), (287, 1001, 9500, [100, 0, 180], PARTS)])
def test_products_of_integers_in_parts(cuda, rows, n, k, counts, launches, trans_b):
    import torch
    a = _integers((rows, k), -3, 3)
    shape = (n, k) if trans_b else (k, n)
    b = _integers(shape if counts is None else (len(counts), *shape), -3, 3)
    a8, b8 = cuda.quantize8(a), cuda.quantize8(b, "e5m2", "tiles")
    off = None if counts is None else torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    y, n_launches = _launches(cuda, lambda: cuda.matmul8(a8, b8, trans_b, off, torch.float32))
    assert n_launches == launches
    at = 0
    for e, c in enumerate([rows] if counts is None else counts):
        w = (b if counts is None else b[e]).double()
        assert torch.equal(y[at:at + c].double(), a[at:at + c].double() @ (w.t() if trans_b else w))
        at += c
    assert not y[at:].any()
    cuda.device_status()


SHAPES = [(5, 256, 512), (300, 256, 512), (100, 300, 2600), (2400, 4104, 2200), (300, 1000, 19200)]


@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_products_on_a_side_stream(cuda, rows, n, k):
    """Scratch, packing and product follow the stream that is current, with
    other products queued on the first one meanwhile."""
    import torch
    a, b = _integers((rows, k), -3, 3), _integers((n, k), -3, 3)
    a8, b8 = cuda.quantize8(a), cuda.quantize8(b, "e4m3", "tiles")
    want = a.double() @ b.double().t()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = []
    for _ in range(4):
        with torch.cuda.stream(side):
            outs.append(cuda.matmul8(a8, b8, dtype=torch.float32))
        outs.append(cuda.matmul8(a8, b8, dtype=torch.float32))
    torch.cuda.synchronize()
    for y in outs:
        assert torch.equal(y.double(), want)
    cuda.device_status()


@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_products_in_a_captured_graph(cuda, rows, n, k):
    """A replay computes from what the operands hold then."""
    import torch
    a8 = cuda.quantize8(_integers((rows, k), -3, 3))
    b8 = cuda.quantize8(_integers((n, k), -3, 3), "e4m3", "tiles")
    cuda.matmul8(a8, b8, dtype=torch.float32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cuda.matmul8(a8, b8, dtype=torch.float32)
    for _ in range(3):
        a, b = _integers((rows, k), -3, 3), _integers((n, k), -3, 3)
        for to, v in ((a8, cuda.quantize8(a)), (b8, cuda.quantize8(b, "e4m3", "tiles"))):
            to.data.copy_(v.data)
            to.scales.copy_(v.scales)
        graph.replay()
        assert torch.equal(y.double(), a.double() @ b.double().t())
    cuda.device_status()


def test_sort_in_a_captured_graph(cuda):
    """Two and three kernels, overlapped, on new ids at each replay."""
    import torch
    for t, k, experts in ((4000, 4, 16), (20000, 8, 64)):
        ids = torch.randint(0, experts, (t, k), dtype=torch.int32, device="cuda")
        cuda.expert_sort(ids, experts)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            order = cuda.expert_sort(ids, experts)
        for _ in range(5):
            ids.copy_(torch.randint(-1, experts, (t, k), dtype=torch.int32, device="cuda"))
            graph.replay()
            flat = ids.reshape(-1).long()
            key = torch.where(flat < 0, torch.full_like(flat, experts), flat)
            sort = torch.sort(key, stable=True)
            routed = int((flat >= 0).sum())
            assert torch.equal(order.source[:routed].long(), sort.indices[:routed])
            assert (order.source[routed:] == -1).all()
            assert torch.equal(order.offsets.long(), torch.searchsorted(sort.values, torch.arange(experts + 1, device="cuda")))
            place = torch.full_like(flat, -1)
            place[sort.indices[:routed]] = torch.arange(routed, device="cuda")
            assert torch.equal(order.position.reshape(-1).long(), place)
    cuda.device_status()
