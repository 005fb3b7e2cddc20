"""Rotary positions, the paged key-value cache and paged attention on the GPU against plain 64-bit forms
(tests/decode_reference.py, where the bounds are derived).  Cached values are compared bit for bit."""
import math

import numpy as np
import pytest
import torch

from tests import decode_reference as ref
from torch_engine_b200 import lib as L
from torch_engine_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def within(got, want, bound, what=""):
    got = got.detach().cpu().double()
    off = (got - want).abs() - bound
    assert not torch.isnan(got).any(), what
    assert float(off.max()) <= 0.0, (what, float((got - want).abs().max()), float(off.max()))


# ------------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,H,T,d,rot", [(1, 1, 1, 64, 64), (3, 5, 7, 64, 32), (2, 3, 33, 80, 80), (2, 2, 5, 96, 24), (2, 3, 4, 7, 6), (1, 4, 3, 130, 128),
                                         (2, 40, 1, 128, 128), (1, 6, 300, 64, 64), (2, 2, 3, 16, 0), (1, 2, 2, 1024, 1024), (5, 1, 2, 66, 66)])
def test_rotary(backend, B, H, T, d, rot, interleaved):
    x = normal(B * 1000 + d, B, H, T, d)
    f = torch.tensor(L.rotary_inv_freq(rot), dtype=torch.float64)
    positions = torch.randint(0, 1 << 20, (B, T), generator=torch.Generator().manual_seed(T))
    positions[0, 0] = -17
    for inverse, call in ((False, backend.rotary), (True, backend.rotary_backward)):
        y = call(x.cuda(), positions.cuda(), f.cuda(), interleaved=interleaved, scale=1.25)
        want = ref.rotary(x, positions, f, interleaved, 1.25, inverse)
        within(y, want, ref.rotary_bound(x, f, interleaved, 1.25))
        assert torch.equal(y[..., rot:].cpu(), x[..., rot:])
    backend.check_device_status()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_views_and_in_place(backend, interleaved):
    """q and k blocks of a projections' buffer as one view of 2H heads, turned in place, the v block untouched; positions
    shared by the batch; a view that is not 16-byte aligned gives the same numbers."""
    B, T, H, d = 3, 9, 2, 64
    f = torch.tensor(L.rotary_inv_freq(d), dtype=torch.float64)
    buffer = normal(5, B, T, 3 * H * d)
    positions = torch.arange(T) * 1000 + 3
    qk = lambda b: b[:, :, :2 * H * d].view(B, T, 2 * H, d).transpose(1, 2)
    want = ref.rotary(qk(buffer), positions.expand(B, T), f, interleaved)
    on = buffer.cuda()
    out = backend.rotary(qk(on), positions.cuda(), f.cuda(), interleaved=interleaved, out=qk(on))
    assert out.data_ptr() == on.data_ptr()
    within(qk(on), want, ref.rotary_bound(qk(buffer), f, interleaved))
    assert torch.equal(on[:, :, 2 * H * d:].cpu(), buffer[:, :, 2 * H * d:])
    odd = torch.empty(B * T * 3 * H * d + 1, device="cuda")[1:].view(B, T, 3 * H * d)
    odd.copy_(buffer)
    assert torch.equal(backend.rotary(qk(odd), positions.cuda(), f.cuda(), interleaved=interleaved), qk(on))
    # [B,T,H,d] order of the result, and a broadcast input
    place = torch.empty(B, T, 2 * H, d, device="cuda").transpose(1, 2)
    backend.rotary(qk(odd), positions.cuda(), f.cuda(), interleaved=interleaved, out=place)
    assert torch.equal(place, qk(on))
    one = normal(6, 1, 1, 1, d).cuda().expand(2, 3, T, d)
    want = ref.rotary(one.cpu(), positions.expand(2, T), f, interleaved)
    within(backend.rotary(one, positions.cuda(), f.cuda(), interleaved=interleaved), want, ref.rotary_bound(one.cpu(), f, interleaved))


def test_rotary_backward_is_the_gradient(backend):
    """<rotary(x + h) - rotary(x), g> = <h, rotary_backward(g)>: rotary is linear, so a difference of any width is exact but
    for rounding, which the elementwise bounds, taken as independent, add up to."""
    B, H, T, d, rot = 2, 3, 11, 64, 48
    f = torch.tensor(L.rotary_inv_freq(rot), dtype=torch.float64)
    x, h, g = (normal(s, B, H, T, d) for s in (1, 2, 3))
    positions = torch.arange(B * T).view(B, T) * 37
    call = lambda fn, t: fn(t.cuda(), positions.cuda(), f.cuda(), scale=0.75).cpu().double()
    left = ((call(backend.rotary, x + h) - call(backend.rotary, x)) * g.double()).sum()
    right = (((x + h).double() - x.double()) * call(backend.rotary_backward, g)).sum()
    # 12 * 2^-24 * 0.75 * (|x0| + |x1|) * |g| per element of three calls, ~ normal: 4 sigma over B*H*T*d elements
    tol = 4 * 3 * 12 * 2.0 ** -24 * 0.75 * 2 * 2 * math.sqrt(B * H * T * d)
    assert abs(float(left - right)) <= tol


def test_rotary_empty_and_refusals(backend):
    f = torch.ones(4, dtype=torch.float64, device="cuda")
    pos = torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    assert backend.rotary(torch.zeros(2, 3, 0, 8, device="cuda"), pos, f).shape == (2, 3, 0, 8)
    x, pos = torch.zeros(2, 3, 4, 8, device="cuda"), torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    for bad in (lambda: backend.rotary(x.double(), pos, f), lambda: backend.rotary(x, pos.int(), f), lambda: backend.rotary(x, pos, f.float()),
                lambda: backend.rotary(x.cpu(), pos, f), lambda: backend.rotary(x[0], pos, f), lambda: backend.rotary(x, pos[:, :3], f),
                lambda: backend.rotary(x.transpose(2, 3), torch.zeros(2, 8, dtype=torch.int64, device="cuda"), f[:2]),
                lambda: backend.rotary(x, pos, torch.ones(5, dtype=torch.float64, device="cuda")), lambda: backend.rotary(x, pos, f, out=x[:1])):
        with pytest.raises(L.BackendError):
            bad()


# -------------------------------------------------------------------------------------------------------------- cache
def make_cache(dtype, pages, heads, page, d, order="phsd", fill=None):
    """A cache whose memory runs in the given order of p(ages), h(eads), s(lots), d, every byte set to `fill` first."""
    extent = dict(p=pages, h=heads, s=page, d=d)
    size = {"f32": 4, "bf16": 2, "e4m3": 1}[dtype]

    def tensor():
        raw = torch.full([extent[c] for c in order[:-1]] + [d * size], 0x7f if fill is None else fill, dtype=torch.uint8, device="cuda").view(DTYPES[dtype])
        return raw.permute([order.index(c) for c in "phsd"])
    k, v = tensor(), tensor()
    if dtype != "e4m3":
        return ops.KvCache(k, v)
    scales = [torch.full((pages, heads, page), float("nan"), device="cuda") for _ in range(2)]
    return ops.KvCache(k, v, *scales)


def scattered(lengths, page, pages, seed=0):
    """A page table for these lengths over distinct pages in scattered order, -1 where a row needs none."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(1, max(-(-n // page) for n in lengths))
    table = torch.full((len(lengths), width), -1, dtype=torch.int64)
    for b, n in enumerate(lengths):
        for i in range(-(-n // page)):
            table[b, i] = order.pop()
    return table


def stored(x, dtype):
    """What the cache stands for after a row of float32 went in, in double."""
    if dtype == "e4m3":
        return torch.from_numpy(np.stack([ref.e4m3_row(r)[0] for r in x.reshape(-1, x.shape[-1]).numpy()])).view(x.shape)
    return x.to(DTYPES[dtype]).double()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("B,H,T,d,page,order", [(1, 1, 1, 16, 16, "phsd"), (3, 2, 21, 48, 13, "phsd"), (2, 3, 40, 64, 16, "pshd"), (2, 2, 9, 80, 1, "phsd"),
                                                (2, 5, 70, 128, 64, "hpsd"), (1, 2, 17, 192, 8, "pshd"), (2, 1, 12, 256, 300, "phsd")])
def test_append_and_read(backend, dtype, B, H, T, d, page, order):
    lengths = [max(0, T - 5 * b) for b in range(B)]
    pages = sum(-(-n // page) for n in lengths) + 3
    table = scattered(lengths, page, pages)
    positions = torch.full((B, T), -1, dtype=torch.int64)
    for b, n in enumerate(lengths):
        positions[b, :n] = torch.randperm(n, generator=torch.Generator().manual_seed(b))      # any order of tokens
    k, v = normal(1, B, H, T, d) * 3, normal(2, B, H, T, d)
    v[:, :, 0] = 0.0
    cache = make_cache(dtype, pages, H, page, d, order)
    before = cache.k.clone().view(torch.uint8)
    backend.kv_append(cache, k.cuda(), v.cuda(), table.cuda(), positions.cuda())
    got_k, got_v = backend.kv_read(cache, table.cuda(), positions.cuda())
    there = (positions >= 0)[:, None, :, None]
    for got, x in ((got_k, k), (got_v, v)):
        want = torch.where(there, stored(x, dtype), torch.zeros((), dtype=torch.float64))
        assert torch.equal(got.cpu().double(), want)
    # bytes of places no token went to are as they were
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(B):
        for t in range(T):
            if positions[b, t] >= 0:
                p, s = ref.place(table, b, int(positions[b, t]), page)
                touched[p, s] = True
                if dtype == "e4m3":
                    assert float(cache.k_scale[p, 0, s]) == ref.e4m3_row(k[b, 0, t].numpy())[1]
    after = cache.k.view(torch.uint8)
    same = (after == before).all(dim=-1).cpu()
    assert bool((same | touched[:, None, :]).all())
    backend.check_device_status()


def test_append_from_views(backend):
    """k and v blocks of a projections' buffer, one that is not 16-byte aligned, and one head broadcast over the batch."""
    B, T, H, d, page = 2, 6, 3, 32, 4
    table, positions = scattered([T] * B, page, 8).cuda(), torch.arange(T).repeat(B, 1).cuda()
    raw = normal(3, B * T * 3 * H * d + 1)
    for skip in (0, 1):
        buffer = raw.cuda()[skip:skip + B * T * 3 * H * d].view(B, T, 3, H, d)
        k, v = buffer[:, :, 1].transpose(1, 2), buffer[:, :, 2].transpose(1, 2)
        cache = make_cache("f32", 8, H, page, d)
        backend.kv_append(cache, k, v, table, positions)
        got = backend.kv_read(cache, table, positions)
        assert torch.equal(got[0], k) and torch.equal(got[1], v)
    one = normal(4, 1, 1, 1, d).cuda().expand(B, H, T, d)
    backend.kv_append(cache, one, one, table, positions)
    assert torch.equal(backend.kv_read(cache, table, positions)[0], one)


def test_eight_bit_rows_at_the_borders(backend):
    """Largest magnitudes at and next to 448 * 2^e, ties, subnormal rows, zeros, and values that are not finite."""
    d = 16
    rows = np.zeros((12, d), dtype=np.float32)
    rows[0, 0] = 448.0
    rows[1, 0] = np.nextafter(np.float32(448.0), np.float32(1e9))
    rows[2, 0] = -np.nextafter(np.float32(448.0), np.float32(0.0))
    rows[3, :6] = [256.0, 17.0, 19.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10]
    rows[4] = np.linspace(-1e-38, 1e-38, d)
    rows[5, 3] = np.float32(1e-45)
    rows[6] = np.linspace(-3.4e38, 3.4e38, d)
    rows[7, :4] = [np.inf, 1.0, -np.inf, 2.0]
    rows[8, :3] = [np.nan, -5.0, 0.3]
    rows[9] = np.nan
    rows[10] = np.float32(448.0) * np.float32(2.0) ** np.arange(-8, 8)
    x = torch.from_numpy(rows).view(1, 1, 12, d)
    cache = make_cache("e4m3", 3, 1, 4, d)
    table, positions = torch.tensor([[2, 0, 1]]).cuda(), torch.arange(12).unsqueeze(0).cuda()
    backend.kv_append(cache, x.cuda(), x.cuda(), table, positions)
    got = backend.kv_read(cache, table, positions)[1].cpu().double()
    want = stored(x, "e4m3").float().double()        # as float32: the smallest subnormals are held by it too
    assert torch.equal(torch.nan_to_num(got, nan=-12345.0), torch.nan_to_num(want, nan=-12345.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
def test_bad_places_are_skipped_and_reported(backend, dtype):
    H, d, page = 2, 32, 4
    cache = make_cache(dtype, 3, H, page, d, fill=0)
    if dtype == "e4m3":
        cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0)
    k = normal(1, 1, H, 4, d).cuda() + 10.0
    sound = torch.tensor([[0, 5, -1, -1]]).cuda()
    for table, positions in (([[2, 3]], [[0, 5, 1, 2]]), ([[2, -1]], [[0, 5, 1, 2]]), ([[2, 1]], [[0, 8, 1, 2]]), ([[2, 1]], [[0, 1 << 40, 1, 2]])):
        table, positions = torch.tensor(table).cuda(), torch.tensor(positions).cuda()
        cache.k.view(torch.uint8).zero_()
        backend.kv_append(cache, k, k, table, positions)
        with pytest.raises(L.BackendError) as e:
            backend.check_device_status()
        assert "KV cache" in str(e.value)
        assert bool((cache.k[2, :, :3].float() != 0).all()) and bool((cache.k[0].float() == 0).all()) and bool((cache.k[1].float() == 0).all())
        got, _ = backend.kv_read(cache, table, positions)
        with pytest.raises(L.BackendError):
            backend.check_device_status()
        assert bool((got[:, :, 1] == 0).all()) and bool((got[:, :, 0] != 0).all())
    backend.check_device_status()
    backend.kv_read(cache, torch.tensor([[2, 1]]).cuda(), sound)
    backend.check_device_status()


def test_cache_refusals(backend):
    cache = backend.kv_cache(4, 2, 8, 32, "bf16")
    k, table, pos = torch.zeros(1, 2, 3, 32, device="cuda"), torch.zeros(1, 2, dtype=torch.int64, device="cuda"), torch.zeros(1, 3, dtype=torch.int64, device="cuda")
    for bad in (lambda: backend.kv_append(cache, k.bfloat16(), k, table, pos), lambda: backend.kv_append(cache, k[:, :1], k, table, pos),
                lambda: backend.kv_append(cache, k, k, table.int(), pos), lambda: backend.kv_append(cache, k, k, table, pos[:, :2]),
                lambda: backend.kv_append(cache, k, k, table.t().expand(2, 2).t(), pos), lambda: backend.kv_read(cache, table[0], pos),
                lambda: backend.kv_append(cache, k.cpu(), k, table, pos), lambda: backend.kv_cache(4, 2, 8, 24) and backend.kv_read(backend.kv_cache(4, 2, 8, 24), table, pos),
                lambda: ops.KvCache(cache.k, cache.v, cache.k, cache.v), lambda: ops.KvCache(cache.k, cache.v.float()), lambda: ops.KvCache(cache.k.half(), cache.v.half()),
                lambda: ops.KvCache(torch.zeros(2, 2, 8, 32, device="cuda").to(torch.float8_e4m3fn), torch.zeros(2, 2, 8, 32, device="cuda").to(torch.float8_e4m3fn)),
                lambda: ops.KvCache(cache.k.cpu(), cache.v.cpu()), lambda: ops.KvCache(cache.k[0], cache.v[0])):
        with pytest.raises(L.BackendError):
            bad()
    with pytest.raises(ValueError):
        backend.kv_cache(4, 2, 8, 32, "int8")
    empty = torch.zeros(1, 2, 0, 32, device="cuda")
    backend.kv_append(cache, empty, empty, table, pos[:, :0])


# ---------------------------------------------------------------------------------------------------------- attention
class Scene:
    """Rows of the given lengths in a cache whose unused places hold NaN, and the exact answers."""

    def __init__(self, dtype, lengths, hq, hk, d, page, seed=0, order="phsd", spread=1.0, value_order=None):
        self.dtype, self.lengths, self.hq, self.hk, self.d, self.page = dtype, lengths, hq, hk, d, page
        self.pages = sum(-(-n // page) for n in lengths) + 3
        self.table = scattered(lengths, page, self.pages, seed)
        longest = max(1, max(lengths))
        self.cache = make_cache(dtype, self.pages, hk, page, d, order, fill=0xff)      # all bits set: NaN in every type
        if value_order:
            other = make_cache(dtype, self.pages, hk, page, d, value_order, fill=0xff)
            self.cache = ops.KvCache(self.cache.k, other.v, self.cache.k_scale, self.cache.v_scale)
        k, v = normal(seed + 1, len(lengths), hk, longest, d) * spread, normal(seed + 2, len(lengths), hk, longest, d)
        self.q = normal(seed + 3, len(lengths), hq, d) * 1.5
        at = torch.arange(longest).expand(len(lengths), -1)
        self.positions = torch.where(at < torch.tensor(lengths).unsqueeze(1), at, torch.full_like(at, -1))
        self.k, self.v = self.as_stored(k), self.as_stored(v)
        self.source = (k, v)

    def as_stored(self, x):
        if self.dtype != "e4m3":
            return x.to(DTYPES[self.dtype]).double()
        amax = x.abs().amax(dim=-1, keepdim=True).double()
        unit = torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
        y = x.double() / unit
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(y / step) * step * unit

    def fill(self, backend):
        backend.kv_append(self.cache, self.source[0].cuda(), self.source[1].cuda(), self.table.cuda(), self.positions.cuda())
        return self

    def check(self, o, lse, lens=None, window=0, scale=None, rows=None):
        scale = self.d ** -0.5 if scale is None else scale
        group = self.hq // self.hk
        for r in range(len(self.lengths)) if rows is None else rows:
            n = min(self.lengths[r], int(lens[r])) if lens is not None else self.lengths[r]
            first = max(0, n - window) if window else 0
            if n <= 0:
                assert bool((o[r] == 0).all()) and bool((lse[r] == -math.inf).all()), r
                continue
            for h in range(self.hk):
                heads = slice(h * group, (h + 1) * group)
                want, want_lse, absolute, top, reach = ref.attention(self.q[r, heads].double(), self.k[r, h, first:n], self.v[r, h, first:n], scale)
                bound, bound_lse = ref.attention_bound(self.d, n - first, absolute, top, reach)
                within(o[r, heads], want, bound, (r, h))
                within(lse[r, heads], want_lse, bound_lse, (r, h, "lse"))

    def run(self, backend, lens=None, **kw):
        lens = torch.tensor(self.lengths if lens is None else lens).cuda()
        return backend.paged_attention(self.q.cuda(), self.cache, self.table.cuda(), lens, want_lse=True, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("lengths,hq,hk,d,page,order", [
    ([1], 1, 1, 64, 16, "phsd"), ([0, 1, 2, 15, 16, 17, 31, 32, 33], 6, 6, 64, 16, "phsd"), ([63, 64, 65, 127, 128, 129, 0], 8, 2, 128, 16, "phsd"),
    ([200, 3], 7, 1, 128, 13, "phsd"), ([100, 90], 32, 2, 64, 1, "pshd"), ([300], 40, 2, 128, 64, "pshd"), ([257, 77, 0, 5], 3, 3, 16, 7, "phsd"),
    ([130, 260], 6, 2, 48, 16, "hpsd"), ([95], 10, 5, 80, 32, "phsd"), ([96, 1], 4, 4, 96, 5, "phsd"), ([70], 9, 1, 112, 16, "phsd"),
    ([150, 33], 5, 1, 192, 16, "pshd"), ([300, 40], 16, 2, 256, 16, "phsd"), ([66], 2, 2, 256, 100, "phsd"), ([1000, 1], 4, 1, 32, 16, "phsd"),
    ([0, 0], 4, 2, 64, 16, "phsd"), ([5000], 2, 1, 64, 16, "phsd"), ([3001, 2999], 12, 2, 128, 32, "phsd")])
def test_attention(backend, dtype, lengths, hq, hk, d, page, order):
    scene = Scene(dtype, lengths, hq, hk, d, page, order=order).fill(backend)
    o, lse = scene.run(backend)
    scene.check(o, lse)
    o2, lse2 = scene.run(backend)
    assert torch.equal(o, o2) and torch.equal(lse, lse2), "two runs differ"
    backend.check_device_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("d,page", [(64, 16), (80, 16), (128, 7)])
def test_attention_with_keys_and_values_in_different_orders(backend, dtype, d, page):
    scene = Scene(dtype, [90, 33, 0, 200], 6, 2, d, page, order="phsd", value_order="pshd").fill(backend)
    scene.check(*scene.run(backend))
    scene = Scene(dtype, [90, 33, 0, 200], 6, 2, d, page, order="hpsd", value_order="phsd").fill(backend)
    scene.check(*scene.run(backend))
    backend.check_device_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
def test_attention_of_many_rows(backend, dtype):
    """More rows than a block has threads, some empty, one long among short ones; a sample of the rows is checked."""
    lengths = [(37 * r) % 90 for r in range(300)]
    lengths[123], lengths[299] = 2600, 0
    scene = Scene(dtype, lengths, 4, 2, 64, 16).fill(backend)
    o, lse = scene.run(backend)
    scene.check(o, lse, rows=[0, 1, 2, 90, 122, 123, 124, 127, 128, 129, 180, 255, 256, 298, 299])
    o2, _ = scene.run(backend)
    assert torch.equal(o, o2)
    # each row alone gives the same within the bounds: no row reads another's share
    assert bool(torch.isfinite(o).all())
    backend.check_device_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("window", [1, 16, 50, 64, 129, 100000])
def test_attention_window(backend, dtype, window):
    scene = Scene(dtype, [0, 1, 49, 50, 51, 300, 129], 6, 2, 64, 13).fill(backend)
    o, lse = scene.run(backend, window=window)
    scene.check(o, lse, window=window)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
def test_attention_with_peaked_and_shifted_scores(backend, dtype):
    """Scores of magnitude 60 and more, where one token takes nearly all, and a scale of either sign and of zero."""
    scene = Scene(dtype, [400, 37], 8, 2, 128, 16, spread=8.0).fill(backend)
    for scale in (None, 0.5, -0.25, 0.0):
        o, lse = scene.run(backend, scale=scale)
        scene.check(o, lse, scale=scale)


def test_attention_rows_that_share_pages(backend):
    """A short prompt as rows of one sequence: every row of the table the same memory, lengths growing by one."""
    scene = Scene("bf16", [41], 8, 2, 64, 16).fill(backend)
    q = normal(9, 41, 8, 64)
    lens = torch.arange(1, 42)
    o, lse = backend.paged_attention(q.cuda(), scene.cache, scene.table.cuda().expand(41, -1), lens.cuda(), want_lse=True)
    for r in range(41):
        for h in range(2):
            heads = slice(4 * h, 4 * h + 4)
            want, want_lse, absolute, top, reach = ref.attention(q[r, heads].double(), scene.k[0, h, :r + 1], scene.v[0, h, :r + 1], 64 ** -0.5)
            bound, bound_lse = ref.attention_bound(64, r + 1, absolute, top, reach)
            within(o[r, heads], want, bound, (r, h))
            within(lse[r, heads], want_lse, bound_lse, (r, h))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
def test_attention_over_parts_joins_to_the_whole(backend, dtype):
    """The log-sum-exp joins attention over the last 100 tokens with attention over those before."""
    scene = Scene(dtype, [350], 4, 2, 64, 16).fill(backend)
    whole, whole_lse = scene.run(backend)
    late, late_lse = scene.run(backend, window=100)
    early, early_lse = scene.run(backend, lens=[250])
    lse = torch.logaddexp(late_lse.double(), early_lse.double())
    o = late.double() * torch.exp(late_lse.double() - lse).unsqueeze(-1) + early.double() * torch.exp(early_lse.double() - lse).unsqueeze(-1)
    scene.check(o, lse)
    scene.check(whole, whole_lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
def test_attention_views(backend, dtype):
    """q inside a projections' buffer, also at an odd offset, the result in a wider buffer, no log-sum-exp."""
    rows, hq, hk, d = 3, 8, 2, 64
    scene = Scene(dtype, [40, 0, 77], hq, hk, d, 16).fill(backend)
    plain, lse = scene.run(backend)
    for skip in (0, 1, 3):
        raw = torch.full((rows * (hq + 2 * hk) * d + skip,), float("nan"), device="cuda")[skip:].view(rows, hq + 2 * hk, d)
        raw[:, :hq].copy_(scene.q)
        wide = torch.full((rows, hq + 1, d + 4), 7.0, device="cuda")
        out = backend.paged_attention(raw[:, :hq], scene.cache, scene.table.cuda(), torch.tensor(scene.lengths).cuda(), out=wide[:, 1:, 4:])
        assert torch.equal(out, plain)
        assert bool((wide[:, 0] == 7).all()) and bool((wide[:, :, :4] == 7).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
def test_attention_reports_bad_pages_and_lengths(backend, dtype):
    """A length beyond the table is cut to it; a page outside the cache counts as masked; both are reported."""
    scene = Scene(dtype, [40, 64, 48], 4, 2, 64, 16).fill(backend)
    o, lse = scene.run(backend, lens=[40, 1 << 40, 48])
    with pytest.raises(L.BackendError) as e:
        backend.check_device_status()
    assert "KV cache" in str(e.value)
    scene.check(o, lse)
    good = scene.table.clone()
    for wrong in (-1, scene.pages, 1 << 40):
        scene.table = good.clone()
        scene.table[0, 2] = wrong           # tokens 32 .. 39 of row 0
        scene.table[2, :] = wrong           # all of row 2
        o, lse = scene.run(backend)
        with pytest.raises(L.BackendError):
            backend.check_device_status()
        scene.check(o, lse, lens=[32, 64, 0])
    backend.check_device_status()


def test_attention_without_pages(backend):
    """Caches and tables of no extent."""
    cache = backend.kv_cache(0, 2, 16, 64, "bf16")
    q, lens = torch.ones(2, 4, 64, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    table = torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    o, lse = backend.paged_attention(q, cache, table, lens, want_lse=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    assert backend.paged_attention(q[:0], cache, table[:0], lens[:0]).shape == (0, 4, 64)
    backend.check_device_status()
    # lengths and page numbers where there are no pages: masked and reported
    o, lse = backend.paged_attention(q, cache, torch.zeros(2, 3, dtype=torch.int64, device="cuda"), lens + 5, want_lse=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    with pytest.raises(L.BackendError):
        backend.check_device_status()


def test_attention_beyond_32_bit_offsets(backend):
    """Pages whose elements lie past 2^31 (and 2^32 bytes) from the base; page numbers written only at the far end."""
    hk, d, page = 8, 256, 64
    pages = (1 << 31) // (hk * d * page) + 40
    k, v = (torch.empty((pages, hk, page, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = ops.KvCache(k, v)
    n = 200
    table = torch.tensor([[pages - 1, pages - 7, 0, pages - 2]])
    x, y = normal(1, 1, hk, n, d), normal(2, 1, hk, n, d)
    backend.kv_append(cache, x.cuda(), y.cuda(), table.cuda(), torch.arange(n).unsqueeze(0).cuda())
    q = normal(3, 1, hk, d)
    o, lse = backend.paged_attention(q.cuda(), cache, table.cuda(), torch.tensor([n]).cuda(), want_lse=True)
    back = backend.kv_read(cache, table.cuda(), torch.arange(n).unsqueeze(0).cuda())
    x, y = x.bfloat16().double(), y.bfloat16().double()
    assert torch.equal(back[0].cpu().double(), x) and torch.equal(back[1].cpu().double(), y)
    for h in range(hk):
        want, want_lse, absolute, top, reach = ref.attention(q[0, h:h + 1].double(), x[0, h], y[0, h], d ** -0.5)
        bound, bound_lse = ref.attention_bound(d, n, absolute, top, reach)
        within(o[0, h:h + 1], want, bound)
        within(lse[0, h:h + 1], want_lse, bound_lse)


def test_attention_needs_its_workspace(backend):
    small = ops.Backend(0, workspace_bytes=4096)
    cache = small.kv_cache(4, 2, 8, 32, "f32")
    q, table, lens = torch.zeros(1, 4, 32, device="cuda"), torch.zeros(1, 2, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(L.BackendError) as e:
        small.paged_attention(q, cache, table, lens)
    assert e.value.status == L.TE_ERR_WORKSPACE
    small.close()


def test_attention_refusals(backend):
    cache = backend.kv_cache(4, 2, 8, 32, "f32")
    q, table, lens = torch.zeros(1, 4, 32, device="cuda"), torch.zeros(1, 2, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    for bad in (lambda: backend.paged_attention(q.half(), cache, table, lens), lambda: backend.paged_attention(q[:, :3], cache, table, lens),
                lambda: backend.paged_attention(q[..., :16], cache, table, lens), lambda: backend.paged_attention(q, cache, table.int(), lens),
                lambda: backend.paged_attention(q, cache, table, lens.int()), lambda: backend.paged_attention(q, cache, table, lens.expand(2)),
                lambda: backend.paged_attention(q.cpu(), cache, table, lens), lambda: backend.paged_attention(q, cache, table, lens, window=-1),
                lambda: backend.paged_attention(q, cache, table, lens, out=q[:, :2]), lambda: backend.paged_attention(q, cache, table, lens, scale=float("nan"))):
        with pytest.raises(L.BackendError):
            bad()


# ----------------------------------------------------------------------------------------------------------- together
def decode_step(backend, qkv, hq, hk, d, cache, table, lens, inv_freq):
    """One new token of each row: qkv [rows, (hq + 2 hk) d] from the projections, turned in place, kept, attended to."""
    rows = qkv.shape[0]
    heads = qkv.view(rows, 1, hq + 2 * hk, d).transpose(1, 2)
    positions = (lens - 1).unsqueeze(1)
    backend.rotary(heads[:, :hq + hk], positions, inv_freq, out=heads[:, :hq + hk])
    backend.kv_append(cache, heads[:, hq:hq + hk], heads[:, hq + hk:], table, positions)
    return backend.paged_attention(heads[:, :hq, 0], cache, table, lens)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
def test_tokens_one_by_one_as_a_whole_sequence(backend, dtype):
    """Projections, rotary positions, cache and attention token by token, against causal attention of the whole sequence in
    64 bits.  f32: within the derived bounds widened by what turning q and k in FP32 moves a score (12 * 2^-24 of |x0| + |x1|
    on either side: 4 * 12 * 2^-24 of sum |q||k|).  8- and 16-bit caches: k and v are off by half a step, 2^-9 resp. 2^-4 of
    the value plus 2^-10 of the row's scale, so that scores and values move by no more than that of their absolute sums."""
    B, T, hq, hk, d, page = 2, 37, 4, 2, 64, 16
    E = 96
    inv_freq = backend.rotary_inv_freq(d, scaling="parts", factor=4.0, trained_length=16)
    x, w = normal(1, B, T, E), normal(2, (hq + 2 * hk) * d, E) / math.sqrt(E)
    cache = backend.kv_cache(B * 3 + 1, hk, page, d, dtype)
    table = scattered([T] * B, page, B * 3 + 1).cuda()
    outs, projected = [], []
    for t in range(T):
        qkv = backend.linear_forward(x[:, t].contiguous().cuda(), w.cuda(), precision="3xtf32")
        projected.append(qkv.cpu().clone())
        outs.append(decode_step(backend, qkv, hq, hk, d, cache, table, torch.full((B,), t + 1, device="cuda"), inv_freq).cpu())
    backend.check_device_status()
    got = torch.stack(outs, 2)                                                    # [B, hq, T, d]
    heads = torch.stack(projected, 1).view(B, T, hq + 2 * hk, d).transpose(1, 2)
    positions = torch.arange(T).expand(B, T)
    turned = ref.rotary(heads[:, :hq + hk], positions, inv_freq.cpu())
    q, k, v = turned[:, :hq], turned[:, hq:], heads[:, hq + hk:].double()
    step = {"f32": 0.0, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4 + 2.0 ** -9}[dtype]
    for b in range(B):
        for h in range(hq):
            kh, vh = k[b, h // 2], v[b, h // 2]
            for t in range(T):
                want, _, absolute, top, reach = ref.attention(q[b, h, t:t + 1], kh[:t + 1], vh[:t + 1], d ** -0.5)
                bound, _ = ref.attention_bound(d, t + 1, absolute, top, reach)
                largest = vh[:t + 1].abs().max()
                moved = (48 * 2.0 ** -24 + step) * reach                          # of every score
                bound = bound + 2 * torch.expm1(2 * moved) * absolute + step * (absolute + largest)
                within(got[b, h, t:t + 1], want, bound, (b, h, t))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "e4m3"])
def test_captured_steps_replay_with_new_contents(backend, dtype):
    """A decode step captured into a graph and replayed as the sequences grow gives what eager calls give."""
    rows, hq, hk, d, page = 3, 8, 2, 64, 16
    inv_freq = backend.rotary_inv_freq(d)
    table = scattered([90] * rows, page, 20).cuda()
    caches = [backend.kv_cache(20, hk, page, d, dtype) for _ in range(2)]
    prompt = normal(1, rows, hk, 70, d).cuda()
    at = torch.arange(70, device="cuda").expand(rows, -1)
    for c in caches:
        backend.kv_append(c, prompt, prompt.flip(2), table, at)
    qkv, lens = torch.zeros(rows, (hq + 2 * hk) * d, device="cuda"), torch.full((rows,), 70, device="cuda")
    twin = qkv.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode_step(backend, qkv, hq, hk, d, caches[0], table, lens, inv_freq)
    torch.cuda.current_stream().wait_stream(side)
    decode_step(backend, twin, hq, hk, d, caches[1], table, lens, inv_freq)      # what the warm-up wrote, in the other cache too
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = decode_step(backend, qkv, hq, hk, d, caches[0], table, lens, inv_freq)
    for step in range(20):
        new = normal(100 + step, rows, (hq + 2 * hk) * d).cuda()
        lens.copy_(torch.tensor([71 + step, 71, 71 + step // 2]))
        qkv.copy_(new)
        graph.replay()
        want = decode_step(backend, new.clone(), hq, hk, d, caches[1], table, lens, inv_freq)
        assert torch.equal(out, want), step
    for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):
        assert torch.equal(a.view(torch.uint8)[table[:, :5]], b.view(torch.uint8)[table[:, :5]])
    backend.check_device_status()


def test_two_captured_graphs_share_the_workspace_one_after_the_other(backend):
    """Graphs of two scenes captured from one backend (one joins inside, one by the second kernel), replayed in turn with eager calls
    between them."""
    scenes = [Scene("bf16", [700, 0, 1500, 33], 8, 2, 64, 16).fill(backend), Scene("f32", [6000], 1, 1, 64, 16, seed=9).fill(backend)]
    want = [s.run(backend) for s in scenes]
    graphs, outs = [], []
    for s in scenes:
        q, table, lens = s.q.cuda(), s.table.cuda(), torch.tensor(s.lengths).cuda()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(backend.paged_attention(q, s.cache, table, lens, want_lse=True))
        graphs.append((graph, q, table, lens))
    for turn in range(6):
        for i in (0, 1, 1, 0):
            for t in outs[i]:
                t.zero_()
            graphs[i][0].replay()
            again = scenes[1 - i].run(backend)
            assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1]), (turn, i)
            assert torch.equal(again[0], want[1 - i][0])
    backend.check_device_status()


def test_captured_before_any_other_call():
    """A context's first calls may be captured ones: a process of its own, whose first use of these kernels is in a capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from torch_engine_b200 import ops
be = ops.Backend(0, workspace_bytes=64 << 20)
x = torch.ones(2, 3, 1, 64, device="cuda")
table, pos, lens = torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.ones(2, dtype=torch.int64, device="cuda")
table[1] = 1
cache, f = be.kv_cache(2, 1, 16, 64, "bf16"), be.rotary_inv_freq(64)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = be.rotary(x, pos, f)
    be.kv_append(cache, y[:, 1:2], y[:, 2:], table, pos)
    o = be.paged_attention(y[:, :1, 0], cache, table, lens)
g.replay()
be.check_device_status()
assert torch.equal(o, torch.ones(2, 1, 64, device="cuda")), o
print("captured first")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


def test_on_another_stream_and_a_context_of_its_own(backend):
    """Two backends on two streams at once: each has its own workspace."""
    other = ops.Backend(0, workspace_bytes=64 << 20)
    scenes = [Scene("bf16", [3000, 10, 1500], 8, 2, 128, 16, seed=s).fill(backend) for s in (0, 50)]
    want = [s.run(backend) for s in scenes]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for be, scene, stream in zip((backend, other), scenes, streams):
            with torch.cuda.stream(stream):
                got.append(scene.run(be))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(got, want):
            assert torch.equal(a, c) and torch.equal(b, d)
    other.check_device_status()
    other.close()
