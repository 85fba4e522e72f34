"""The 4-bit paged cache (scratchtape_b200/kv4.py) against plain statements in 64 bits.

The statements below take a cache apart by the documented address of each code and evaluate rotation, quantiser and
attention in float64.  Bounds, from the arithmetic:

append   a stored value lies within half a step of its key or value; zero and scale are rounded to f16, which moves
         it by at most 2^-11 |zero| + 15 * 2^-11 scale more; f32 rotation adds 2^-22 (|a| + |b|)
read     f32: exact (a 4-bit code times an 11-bit scale, one rounding of the sum: 2^-24); f16 / bf16: one rounding
attend   f32: scores within about 2^-20 of their own size (below 32 here) and weights held to 22 bits: 3e-5 max|v|;
         16-bit types: the result's own rounding (2^-11 / 2^-8 of it), weights rounded to f16 (2^-11 max|v|) and,
         where keys are rounded to f16, scores off by at most 2^-11 (2^-10 max|v|): together 2^-9 max|v| more
lse      f32: 3e-5 absolute; 16-bit types 2^-9
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}
DEV = "cuda"


def kv4():
    from scratchtape_b200 import kv4 as m
    return m


def values64(data, d, group):
    """[slots, heads, d] keys and values of a whole cache in float64."""
    pages, heads, tiles, nb = data.shape
    t = data.permute(0, 2, 1, 3).reshape(-1, heads, nb)
    tok, c = torch.arange(16, device=DEV)[:, None], torch.arange(d, device=DEV)[None]
    ng, out = d // group, []
    for at, meta in (((c // group) * 8 * group + tok * (group // 2) + (c % group) // 2, 16 * d),
                     (8 * d + (c // 2) * 16 + 4 * ((tok & 7) >> 1) + 2 * (tok & 1) + (tok >> 3), 16 * d + 64 * ng)):
        code = (t[:, :, at] >> ((c & 1) * 4).expand_as(at).to(torch.uint8)) & 15
        m = t[:, :, meta:meta + 64 * ng].contiguous().view(F16).view(-1, heads, ng, 16, 2).double()
        m = m.transpose(2, 3).repeat_interleave(group, 3)
        out.append((code.double() * m[..., 0] + m[..., 1]).transpose(1, 2).reshape(-1, heads, d))
    return out


def rotate64(x, cos, sin, positions, interleaved):
    x = x.double().clone()
    if cos is None:
        return x
    r = 2 * cos.shape[1]
    i = torch.arange(r // 2, device=DEV)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    c, s = cos.double()[positions.long()][:, None], sin.double()[positions.long()][:, None]
    xa, xb = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
    return x


def check_held(got, x, group):
    """got: what the cache stands for; x: what was put in (float64, finite)."""
    g = x.clamp(-65504, 65504).unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = (hi - lo) / 15
    bound = 0.5 * step + 2.0 ** -11 * lo.abs() + 16 * 2.0 ** -11 * step + 2.0 ** -21 * g.abs().amax(-1, keepdim=True) \
        + 2.0 ** -24
    assert ((got.unflatten(-1, (-1, group)) - g).abs() <= bound).all()


def table(lens, page, spare=2, seed=0):
    need = [-(-n // page) for n in lens]
    perm = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    out = torch.full((len(lens), max(1, max(need))), 1 << 30, dtype=torch.int32)  # never to be read
    at = 0
    for b, n in enumerate(need):
        out[b, :n] = perm[at:at + n]
        at += n
    return sum(need) + spare, out.to(DEV)


def slots_of(pages, b, lo, hi, page):
    i = torch.arange(lo, hi, device=DEV)
    return pages[b].long()[i // page] * page + i % page


def filled(lens, kv_heads, d, group, page, seed):
    """A cache whose slots past each length hold all ones (NaN scales), and its table."""
    n, pages = table(lens, page, seed=seed)
    data = torch.full((n, kv_heads, page // 16, kv4().tile_bytes(d, group)), 255, dtype=torch.uint8, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for b, m in enumerate(lens):
        k = torch.randn((m, kv_heads, d), generator=g, device=DEV) + 0.5
        v = torch.randn((m, kv_heads, d), generator=g, device=DEV)
        kv4().append(data, k, v, slots_of(pages, b, 0, m, page), group)
    return data, pages


def attend64(q, data, pages, lens, counts, scale, group, causal, window, one):
    d, page = q.shape[2], data.shape[2] * 16
    k_all, v_all = values64(data, d, group)
    share = q.shape[1] // data.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:2], 0.0 if one else -math.inf, dtype=torch.float64, device=DEV)
    at, vmax = 0, 1e-30
    for b, (m, n) in enumerate(zip(lens, counts)):
        if m and n:
            sl = slots_of(pages, b, 0, m, page)
            k, v = k_all[sl].repeat_interleave(share, 1), v_all[sl].repeat_interleave(share, 1)
            vmax = max(vmax, v.abs().max().item())
            x = torch.einsum("ihd,jhd->hij", q[at:at + n].double(), k) * scale
            pos, key = torch.arange(m - n, m, device=DEV)[:, None], torch.arange(m, device=DEV)[None]
            seen = torch.ones((n, m), dtype=torch.bool, device=DEV)
            if causal:
                seen &= key <= pos
            if window:
                seen &= key > pos - window
            x = torch.where(seen, x, -math.inf)
            if one:
                x = torch.cat([x, torch.zeros(x.shape[:2] + (1,), dtype=x.dtype, device=DEV)], -1)
            s = torch.logsumexp(x, -1)
            p = torch.exp(x - torch.where(s > -math.inf, s, 0.0)[..., None])[..., :m]
            o[at:at + n] = torch.einsum("hij,jhd->ihd", p, v)
            lse[at:at + n] = s.T
        at += n
    return o, lse, vmax


def close(o, want, vmax, dtype):
    err = (o.double() - want).abs()
    tol = ROUND[dtype] * want.abs() + (3e-5 if dtype == F32 else 2.0 ** -9) * vmax
    assert torch.isfinite(o).all() and (err <= tol).all(), "off by %.3g of %.3g" % (err.max(), vmax)


def close_lse(lse, want, dtype):
    none = want == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert ((lse.double() - want)[~none].abs() <= (3e-5 if dtype == F32 else 2.0 ** -9)).all()


ATTEND = [
    # lens, rows of each, heads, kv_heads, d, group, page, type, causal, window, one
    ([1], [1], 1, 1, 64, 64, 16, F32, True, 0, False),
    ([0, 5, 16, 17, 33], None, 4, 4, 64, 64, 16, F32, True, 0, True),
    ([0, 5, 16, 17, 33], None, 4, 4, 64, 32, 32, F16, True, 0, False),
    ([128, 77, 1, 300], None, 8, 2, 128, 64, 64, BF16, True, 0, False),
    ([1000, 31], None, 7, 1, 128, 128, 16, F16, True, 0, False),
    ([1000, 31], None, 6, 2, 128, 32, 128, F32, True, 0, False),
    ([700, 5000, 3], None, 16, 2, 128, 64, 128, BF16, True, 0, False),
    ([9000], None, 32, 8, 128, 64, 64, F16, True, 0, True),
    ([9000], None, 3, 1, 64, 64, 48, F32, True, 0, False),
    ([40, 3, 0, 200], [4, 5, 2, 3], 8, 2, 128, 64, 16, BF16, True, 0, False),  # more rows than keys
    ([40, 3, 0, 200], [4, 0, 2, 3], 8, 2, 128, 64, 16, F32, False, 0, False),
    ([300, 64, 65], [7, 1, 8], 10, 2, 64, 32, 32, F16, True, 20, False),
    ([300, 64, 65], [7, 1, 8], 5, 1, 128, 64, 32, BF16, False, 17, True),
    ([257, 90], [40, 90], 4, 1, 128, 64, 64, BF16, True, 0, False),
    ([257, 90], [40, 90], 8, 8, 64, 64, 16, F32, True, 33, False),
    ([700, 513, 130], [300, 513, 129], 8, 2, 128, 64, 64, F16, True, 0, False),
    ([700, 513, 130], [300, 513, 129], 6, 2, 64, 32, 16, BF16, True, 100, True),
    ([700, 20], [300, 50], 4, 2, 128, 128, 64, BF16, False, 0, False),
    ([1500], [700], 16, 1, 128, 32, 32, F16, True, 0, False),
    ([600, 30], [140, 30], 9, 3, 64, 64, 64, F32, True, 0, False),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend(dev, case):
    lens, counts, heads, kv_heads, d, group, page, dtype, causal, window, one = ATTEND[case]
    data, pages = filled(lens, kv_heads, d, group, page, case)
    rows = sum(counts) if counts else len(lens)
    g = torch.Generator(device=DEV).manual_seed(100 + case)
    q = (torch.randn((rows, heads, d), generator=g, device=DEV) * 2).to(dtype)
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=DEV) \
        if counts else None
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    args = dict(q_start=start, max_q=max(counts) if counts else None, causal=causal, one=one, window=window,
                return_lse=True)
    o, lse = kv4().attend(q, data, pages, kv_len, d ** -0.5, group, **args)
    want, want_lse, vmax = attend64(q, data, pages, lens, counts or [1] * len(lens), d ** -0.5, group, causal, window,
                                    one)
    close(o, want, vmax, dtype)
    close_lse(lse, want_lse, dtype)
    again, lse2 = kv4().attend(q, data, pages, kv_len, d ** -0.5, group, **args)
    assert torch.equal(o, again) and torch.equal(lse, lse2)
    assert dev.last_kernel.startswith("k_kv4_")
    alone = kv4().attend(q, data, pages, kv_len, d ** -0.5, group, **dict(args, return_lse=False))
    close(alone, want, vmax, dtype)  # bf16 goes another way without a log-sum-exp
    dev.sync()


TILED = [
    # lens, rows of each, heads, kv_heads, d, group, page, causal, window, one: many rows of bf16
    ([900], [900], 8, 2, 128, 64, 64, True, 0, False),
    ([513, 700], [513, 128], 16, 4, 128, 128, 16, True, 0, True),
    ([640, 1000, 65, 0, 300], [300, 257, 65, 40, 310], 8, 1, 128, 32, 48, True, 70, False),
    ([700, 20, 511], [500, 450, 1], 12, 2, 64, 64, 32, True, 0, False),
    ([333, 900], [333, 640], 7, 1, 64, 32, 128, False, 0, True),
    ([1200], [600], 5, 5, 128, 64, 16, False, 200, False),
    ([300, 290, 280, 310, 150], [300, 290, 280, 310, 150], 12, 3, 64, 32, 16, True, 0, False),
]


@pytest.mark.parametrize("case", range(len(TILED)))
@pytest.mark.parametrize("aligned", [True, False])
def test_attend_by_tiles(dev, case, aligned):
    """Many rows of bf16, queries in rows of a wider tensor, on 16-byte boundaries or not."""
    lens, counts, heads, kv_heads, d, group, page, causal, window, one = TILED[case]
    data, pages = filled(lens, kv_heads, d, group, page, 50 + case)
    g = torch.Generator(device=DEV).manual_seed(case)
    off = 8 if aligned else 3
    wide = torch.randn((sum(counts), heads * d + 2 * off), generator=g, device=DEV).to(BF16) * 2
    q = wide[:, off:off + heads * d].unflatten(1, (heads, d))
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    args = dict(q_start=start, max_q=max(counts), causal=causal, one=one, window=window)
    o = kv4().attend(q, data, pages, kv_len, d ** -0.5, group, **args)
    assert dev.last_kernel == "k_kv4_attn_tiles" or case in (4, 5)  # few heads and keys: either kernel
    want, _, vmax = attend64(q, data, pages, lens, counts, d ** -0.5, group, causal, window, one)
    close(o, want, vmax, BF16)
    assert torch.equal(o, kv4().attend(q, data, pages, kv_len, d ** -0.5, group, **args))
    dev.sync()


@pytest.mark.parametrize("case", [2, 5])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attend_by_tiles_from_a_cold_cache(dev, case, dtype):
    """Two or three blocks of keys a tile, far from the chip: values come late, and the last product later than scores."""
    lens, counts, heads, kv_heads, d, group, page, causal, window, one = TILED[case]
    data, pages = filled(lens, kv_heads, d, group, page, 80 + case)
    g = torch.Generator(device=DEV).manual_seed(case)
    q = (torch.randn((sum(counts), heads, d), generator=g, device=DEV) * 2).to(dtype)
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    args = dict(q_start=start, max_q=max(counts), causal=causal, one=one, window=window)
    flush, outs = torch.empty(1 << 28, dtype=torch.uint8, device=DEV), []
    for i in range(40):
        flush.fill_(i)
        outs.append(kv4().attend(q, data, pages, kv_len, d ** -0.5, group, **args))
    want, _, vmax = attend64(q, data, pages, lens, counts, d ** -0.5, group, causal, window, one)
    close(outs[0], want, vmax, dtype)
    assert all(torch.equal(o, outs[0]) for o in outs)
    dev.sync()


@pytest.mark.parametrize("case", [0, 1, 2, 3, 6])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attend_by_tiles_with_lse(dev, case, dtype):
    lens, counts, heads, kv_heads, d, group, page, causal, window, one = TILED[case]
    data, pages = filled(lens, kv_heads, d, group, page, 70 + case)
    g = torch.Generator(device=DEV).manual_seed(case)
    q = (torch.randn((sum(counts), heads, d), generator=g, device=DEV) * 2).to(dtype)
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o, lse = kv4().attend(q, data, pages, kv_len, d ** -0.5, group, q_start=start, max_q=max(counts), causal=causal,
                          one=one, window=window, return_lse=True)
    assert dev.last_kernel == "k_kv4_attn_tiles"
    want, want_lse, vmax = attend64(q, data, pages, lens, counts, d ** -0.5, group, causal, window, one)
    close(o, want, vmax, dtype)
    close_lse(lse, want_lse, dtype)
    dev.sync()


def test_tiles_and_a_page_outside_the_cache(dev):
    """Keys of a page number out of range are left out and reported, by either kernel; a score far above those
    before it, and rows whose first keys are hidden, rescale what was summed."""
    import scratchtape_b200._native as N
    d, group, page, n = 128, 64, 32, 640
    data, pages = filled([n], 2, d, group, page, 9)
    k = torch.randn((n, 2, d), device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
    k[300] *= 30.0
    k[500] *= 90.0
    v = torch.randn((n, 2, d), device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    kv4().append(data, k, v, slots_of(pages, 0, 0, n, page), group)
    q = torch.randn((n, 8, d), device=DEV, generator=torch.Generator(device=DEV).manual_seed(6)).to(BF16)
    start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    kv_len = torch.tensor([n], dtype=torch.int32, device=DEV)
    call = lambda p, **a: kv4().attend(q, data, p, kv_len, 0.1, group, q_start=start, **a)  # noqa: E731
    o = call(pages)
    assert dev.last_kernel == "k_kv4_attn_tiles"
    want, _, vmax = attend64(q, data, pages, [n], [n], 0.1, group, True, 0, False)
    close(o, want, vmax, BF16)
    dev.sync()
    wrong = pages.clone()
    wrong[0, 3], wrong[0, 7] = data.shape[0], -1
    for a in ({}, {"return_lse": True}):
        got = call(wrong, **a)
        with pytest.raises(N.StError, match="INVALID_ARG"):
            dev.sync()
        dev.sync()
        got = got[0] if a else got
        assert torch.isfinite(got).all()
        close(got[:96], want[:96], vmax, BF16)  # rows that do not see them
        hidden = [j for j in range(n) if j // page not in (3, 7)]
        kk, vv = (x[slots_of(pages, 0, 0, n, page)][hidden].repeat_interleave(4, 1) for x in values64(data, d, group))
        x = torch.einsum("hd,jhd->hj", q[n - 1].double(), kk) * 0.1
        close(got[n - 1], torch.einsum("hj,jhd->hd", torch.softmax(x, -1), vv), vmax, BF16)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attend_extremes(dev, dtype):
    """Queries and keys of large and tiny size, one score far above the rest, equal scores, equal values."""
    d, group, page, lens = 128, 64, 32, [200, 200, 200, 200]
    data, pages = filled(lens, 2, d, group, page, 5)
    k = torch.randn((200, 2, d), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    k[:, 0] = 0.0                     # every score 0
    k[50, 1] = 40.0                   # one key far above the rest
    v = torch.full((200, 2, d), 0.75, device=DEV)
    kv4().append(data, k, v, slots_of(pages, 0, 0, 200, page), group)
    kv4().append(data, k * 3e-6, v * 1e-6, slots_of(pages, 1, 0, 200, page), group)
    kv4().append(data, k * 100, torch.randn_like(v) * 3000, slots_of(pages, 2, 0, 200, page), group)
    q = torch.randn((4, 4, d), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    q[0] *= 30.0
    q[1] *= 2000.0
    q[2] *= 1e-2
    q[3, 0] = 0.0
    q[3, 1] *= 1e-3
    q = q.to(dtype)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o, lse = kv4().attend(q, data, pages, kv_len, 0.05, group, return_lse=True)
    want, want_lse, _ = attend64(q, data, pages, lens, [1] * 4, 0.05, group, True, 0, False)
    vals = values64(data, d, group)[1]
    for b in range(4):
        close(o[b], want[b], vals[slots_of(pages, b, 0, 200, page)].abs().max().item(), dtype)
    big = want_lse.abs().clamp(min=1.0)
    assert ((lse.double() - want_lse).abs() <= (3e-6 if dtype == F32 else 2.0 ** -9) * big + 3e-5).all()
    dev.sync()


def test_attend_strided_queries_and_stream(dev):
    """Queries inside a fused projection's rows; the call on a stream of its own."""
    lens, heads, kv_heads, d, group, page = [100, 300, 7], 8, 2, 64, 64, 16
    data, pages = filled(lens, kv_heads, d, group, page, 3)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for off, dtype in ((1, BF16), (8, F16), (3, F32)):  # 2-byte, 16-byte and 4-byte aligned rows
        wide = torch.randn((3, heads * d + 24 + off), device=DEV).to(dtype)
        q = wide[:, off:off + heads * d].unflatten(1, (heads, d))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            o = kv4().attend(q, data, pages, kv_len, 0.125, group)
        s.synchronize()
        want, _, vmax = attend64(q, data, pages, lens, [1] * 3, 0.125, group, True, 0, False)
        close(o, want, vmax, dtype)
    turned = torch.randn((d, heads, 3), device=DEV).permute(2, 1, 0)  # rows of d not contiguous
    want, _, vmax = attend64(turned, data, pages, lens, [1] * 3, 0.125, group, True, 0, False)
    close(kv4().attend(turned, data, pages, kv_len, 0.125, group), want, vmax, F32)


def test_attend_replayed_in_a_graph(dev):
    """A captured step attends over the lengths that the device holds at each replay."""
    heads, kv_heads, d, group, page = 8, 2, 128, 64, 32
    data, pages = filled([900, 400], kv_heads, d, group, page, 4)
    q = torch.randn((2, heads, d), device=DEV).to(BF16)
    kv_len = torch.tensor([10, 10], dtype=torch.int32, device=DEV)
    kv4().attend(q, data, pages, kv_len, 0.1, group)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = kv4().attend(q, data, pages, kv_len, 0.1, group)
    for lens in ([900, 1], [16, 400]):
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        want, _, vmax = attend64(q, data, pages, lens, [1, 1], 0.1, group, True, 0, False)
        close(o, want, vmax, BF16)


def test_a_cache_past_2_to_the_32(dev):
    """Slots whose bytes lie past 2^32 (4.7 GB): append, read, attend."""
    d, group, page, kv_heads = 128, 64, 128, 2
    nb = kv4().tile_bytes(d, group)
    n = (1 << 32) // (kv_heads * page // 16 * nb) + 2000
    data = torch.empty((n, kv_heads, page // 16, nb), dtype=torch.uint8, device=DEV)
    pages = torch.tensor([[n - 1, n - 700, 0]], dtype=torch.int32, device=DEV)
    k, v = torch.randn((300, kv_heads, d), device=DEV), torch.randn((300, kv_heads, d), device=DEV)
    slots = slots_of(pages, 0, 0, 300, page)
    kv4().append(data, k, v, slots, group)
    rk, rv = kv4().read(data, slots, d, group)
    check_held(rk.double(), k.double(), group)
    check_held(rv.double(), v.double(), group)
    q = torch.randn((1, 4, d), device=DEV)
    o = kv4().attend(q, data, pages, torch.tensor([300], dtype=torch.int32, device=DEV), 0.1, group)
    rk, rv = (x.double().repeat_interleave(2, 1) for x in (rk, rv))
    p = torch.softmax(torch.einsum("ihd,jhd->ihj", q.double(), rk) * 0.1, -1)
    close(o, torch.einsum("ihj,jhd->ihd", p, rv), rv.abs().max().item(), F32)
    dev.sync()


APPEND = [
    # n, first slot of the run, heads, kv_heads, d, group, page, type, rotary, interleaved
    (1, 0, 1, 1, 64, 64, 16, F32, 0, False),
    (5, 13, 3, 1, 64, 32, 16, F16, 64, False),
    (16, 16, 4, 4, 128, 64, 32, BF16, 128, False),
    (37, 3, 8, 2, 128, 128, 16, F32, 128, True),
    (200, 0, 4, 2, 128, 32, 64, BF16, 64, True),
    (333, 7, 5, 5, 64, 64, 48, F16, 22, False),
    (333, 32, 6, 3, 128, 64, 128, BF16, 6, True),
    (1500, 5, 2, 1, 128, 64, 64, F32, 64, False),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append_and_read(dev, case):
    n, first, heads, kv_heads, d, group, page, dtype, rotary, interleaved = APPEND[case]
    total, pages = table([first + n], page, seed=case)
    g = torch.Generator(device=DEV).manual_seed(case)
    data = torch.randint(0, 256, (total, kv_heads, page // 16, kv4().tile_bytes(d, group)), generator=g, device=DEV,
                         dtype=torch.uint8)
    before = data.clone()
    wide = torch.randn((n, heads + 2 * kv_heads, d + 5), generator=g, device=DEV).to(dtype)
    q, k, v = (wide[:, a:b, 3:3 + d] for a, b in ((0, heads), (heads, heads + kv_heads),
                                                  (heads + kv_heads, heads + 2 * kv_heads)))
    slots = slots_of(pages, 0, first, first + n, page)
    left = torch.arange(n, device=DEV) % 11 == 10
    slots = torch.where(left, -1 - torch.arange(n, device=DEV), slots)
    if case % 2:  # not only runs in order
        slots = torch.cat([slots[:n // 2], slots[n // 2:].flip(0)])
    cos = sin = positions = None
    if rotary:
        positions = torch.randint(0, 500, (n,), generator=g, device=DEV, dtype=torch.int32)
        angle = torch.rand((500, rotary // 2), generator=g, device=DEV) * 6.3
        cos, sin = angle.cos(), angle.sin()
    out = kv4().append(data, k, v, slots, group, q=q if rotary else None, cos=cos, sin=sin, positions=positions,
                       interleaved=interleaved)
    dev.sync()
    keep = slots >= 0
    held_k, held_v = values64(data, d, group)
    k64, v64 = rotate64(k, cos, sin, positions, interleaved), v.double()
    check_held(held_k[slots[keep]], k64[keep], group)
    check_held(held_v[slots[keep]], v64[keep], group)
    other = torch.ones(total * page, dtype=torch.bool, device=DEV)
    other[slots[keep]] = False  # all other slots keep their bytes
    was_k, was_v = values64(before, d, group)
    same = lambda a, b: torch.equal(a[other].nan_to_num(7.5), b[other].nan_to_num(7.5))  # noqa: E731
    assert same(held_k, was_k) and same(held_v, was_v)
    if rotary:
        want = rotate64(q, cos, sin, positions, interleaved)
        bound = ROUND[dtype] * want.abs() + 2.0 ** -22 * q.double().abs().amax() * 2
        assert ((out.double() - want).abs() <= bound).all()
    for rtype in (F32, F16, BF16):
        rk, rv = kv4().read(data, slots, d, group, rtype)
        for got, held in ((rk, held_k), (rv, held_v)):
            want = torch.where(keep[:, None, None], held[slots.clamp(min=0)], 0.0)
            err = (got.double() - want).abs()
            assert (err <= max(ROUND[rtype], 2.0 ** -24) * want.abs() + 2.0 ** -25).all()
    dev.sync()


def test_append_of_non_finite_and_equal_values(dev):
    d, group = 64, 32
    data = kv4().empty(1, 16, 1, d, group)
    k = torch.randn((4, 1, d), device=DEV)
    k[0, 0, 3], k[0, 0, 40], k[1, 0, 7] = math.nan, math.inf, -math.inf
    k[2], k[3, 0, :32] = 1.25, 1e30
    v = torch.zeros((4, 1, d), device=DEV)
    v[1] = -3.0
    kv4().append(data, k, v, torch.arange(4, device=DEV), group)
    rk, rv = kv4().read(data, torch.arange(4, device=DEV), d, group)
    assert torch.isfinite(rk).all() and torch.equal(rv, v)
    check_held(rk.double(), torch.nan_to_num(k.double(), nan=0.0, posinf=65504.0, neginf=-65504.0), group)
    assert torch.equal(rk[2], k[2]) and (rk[3, 0, :32] == 65504).all()


def test_empty_calls(dev):
    data = kv4().empty(2, 16, 2, 64)
    e = lambda *s, t=F32: torch.empty(s, dtype=t, device=DEV)  # noqa: E731
    kv4().append(data, e(0, 2, 64), e(0, 2, 64), e(0, t=torch.int64))
    assert kv4().read(data, e(0, t=torch.int64), 64)[0].shape == (0, 2, 64)
    assert kv4().attend(e(0, 4, 64), data, e(0, 1, t=torch.int32), e(0, t=torch.int32), 1.0).shape == (0, 4, 64)
    o = kv4().attend(torch.ones((2, 4, 64), device=DEV), data, e(2, 0, t=torch.int32),
                     torch.zeros(2, dtype=torch.int32, device=DEV), 1.0)
    assert (o == 0).all()


def test_refusals(dev):
    import scratchtape_b200._native as N
    m = kv4()
    data = m.empty(2, 16, 2, 64)
    k = torch.randn((3, 2, 64), device=DEV)
    slots = torch.arange(3, device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    cos = torch.ones((4, 32), device=DEV)
    for bad in (lambda: m.append(data, k[:, :1], k, slots),
                lambda: m.append(data, k.half(), k, slots),
                lambda: m.append(data, k.double(), k.double(), slots),
                lambda: m.append(data, k, k, slots.int()),
                lambda: m.append(data, k, k, slots[:2]),
                lambda: m.append(data, k, k, slots, 32),
                lambda: m.append(data, k, k, slots, q=k),
                lambda: m.append(data, k, k, slots, cos=cos, sin=cos[:, :3], positions=i32(0, 1, 2)),
                lambda: m.append(data[:, :, :, :-1], k, k, slots),
                lambda: m.read(data, slots, 128),
                lambda: m.read(data, slots, 64, dtype=torch.int32),
                lambda: m.attend(k, data, i32(0, 1), i32(3), 1.0),
                lambda: m.attend(k[:, :1], data, i32(0, 1).view(1, 2), i32(3), 1.0, q_start=i32(0, 3)),
                lambda: m.attend(k, data, i32(0, 1).view(1, 2), i32(3), 1.0, q_start=i32(0, 3), window=-1),
                lambda: m.empty(2, 20, 2, 64)):
        with pytest.raises(ValueError):
            bad()
    bad_shape = torch.zeros((2, 2, 1, m.tile_bytes(96, 32)), dtype=torch.uint8, device=DEV)
    with pytest.raises(N.StError, match="UNSUPPORTED"):
        m.read(bad_shape, slots, 96, 32)
    with pytest.raises(N.StError, match="UNSUPPORTED"):
        m.read(torch.zeros((2, 2, 65, m.tile_bytes(64, 64)), dtype=torch.uint8, device=DEV), slots, 64)
    odd = torch.zeros(2 * 2 * m.tile_bytes(64, 64) + 8, dtype=torch.uint8, device=DEV)[8:]
    with pytest.raises(N.StError, match="aligned"):
        m.read(odd.view(2, 2, 1, -1), slots, 64)


def test_what_only_the_device_sees(dev):
    """Slots, positions, pages and lengths out of range: left out, and reported at the next sync."""
    import scratchtape_b200._native as N
    m = kv4()
    data = m.empty(2, 16, 2, 64)
    k = torch.randn((3, 2, 64), device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    cos = torch.ones((4, 32), device=DEV)

    def told(f):
        r = f()
        with pytest.raises(N.StError, match="INVALID_ARG"):
            dev.sync()
        dev.sync()
        return r

    told(lambda: m.append(data, k, k, torch.tensor([0, 32, 1], device=DEV)))
    assert (m.read(data, torch.tensor([0, 1], device=DEV), 64)[0] != 0).any(-1).all()
    told(lambda: m.append(data, k, k, torch.arange(3, device=DEV), cos=cos, sin=cos, positions=i32(0, 4, -1)))
    rk, _ = told(lambda: m.read(data, torch.tensor([1 << 40, 0], device=DEV), 64))
    assert (rk[0] == 0).all() and (rk[1] != 0).any()
    q = torch.randn((1, 2, 64), device=DEV)
    m.append(data, k, k, torch.arange(3, device=DEV))
    want = m.attend(q, data, i32(0).view(1, 1), i32(3), 0.1)
    dev.sync()
    assert torch.isfinite(told(lambda: m.attend(q, data, i32(0).view(1, 1), i32(17), 0.1))).all()
    assert torch.equal(told(lambda: m.attend(q, data, i32(0).view(1, 1), i32(-3), 0.1)), torch.zeros_like(q))
    assert torch.equal(told(lambda: m.attend(q, data, i32(2).view(1, 1), i32(3), 0.1)), torch.zeros_like(q))
    assert torch.equal(told(lambda: m.attend(q, data, i32(-1).view(1, 1), i32(3), 0.1)), torch.zeros_like(q))
    told(lambda: m.attend(k, data, i32(0).view(1, 1), i32(3), 0.1, q_start=i32(0, 3), max_q=2))
    assert torch.equal(m.attend(q, data, i32(0).view(1, 1), i32(3), 0.1), want)
    dev.sync()
