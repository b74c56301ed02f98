"""The paged key / value cache and the attention of one new token that reads it (csrc/paged.hip), against the definition in 64 bits.
Bounds (U = 2^-24, e = torch.finfo(cache type).eps / 2, half a step of a value near one): a score, a sum of head_dim products taken in
fp32, is off by at most S = (head_dim + 8) U scale sum |q||k|, which moves every weight by 2 S of itself; the weights and the
result are each rounded once to the cache's type, so the result is off by e (sum p |v| + |out|) + 4 (S + (L / 64 + 32) U) sum p |v|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cache(P, Hkv, page, dh, dtype, seed):
    g = _gen(seed)
    return (torch.randn(P, Hkv, page, dh, generator=g).to(dtype).cuda(), torch.randn(P, Hkv, page, dh, generator=g).to(dtype).cuda())


def _tables(lens, page, seed, width=None, spare=3):
    """Block tables of a shuffled pool, and its number of pages; places behind a sequence's own pages hold entries outside the pool."""
    per = [-(-max(n, 0) // page) for n in lens]
    P = sum(per) + spare
    order = torch.randperm(P, generator=_gen(seed)).tolist()
    width = max(1, max(per)) if width is None else width
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    at = 0
    for m, c in enumerate(per):
        table[m, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    return table, P, order[at:]


def _ref(q, kp, vp, table, lens, scale):
    M, H, dh = q.shape
    P, Hkv, page, _ = kp.shape
    group = H // Hkv
    q, kp, vp = q.double().cpu(), kp.double().cpu(), vp.double().cpu()
    out, mag = torch.zeros(M, H, dh, dtype=torch.float64), torch.zeros(M, H, dh, dtype=torch.float64)
    lse, S = torch.full((M, H), -math.inf, dtype=torch.float64), torch.zeros(M, H, dtype=torch.float64)
    for m in range(M):
        n = min(int(lens[m]), table.shape[1] * page)
        keep = [j for j in range(max(n, 0)) if 0 <= int(table[m, j // page]) < P]
        if not keep:
            continue
        rows = [(int(table[m, j // page]), j % page) for j in keep]
        pi, oi = torch.tensor([r[0] for r in rows]), torch.tensor([r[1] for r in rows])
        for h in range(H):
            k, v = kp[pi, h // group, oi], vp[pi, h // group, oi]
            z = (k @ q[m, h]) * scale
            w = torch.softmax(z, dim=0)
            out[m, h], mag[m, h], lse[m, h] = w @ v, w @ v.abs(), torch.logsumexp(z, dim=0)
            S[m, h] = ((k.abs() @ q[m, h].abs()) * abs(scale)).max() * (dh + 8) * U
    return out, mag, lse, S


def _check(got, lse, ref, lens, dtype, what=""):
    out, mag, rl, S = ref
    e = torch.finfo(dtype).eps / 2
    L = max(1, int(max(lens)))
    r = (L / 64 + 32) * U
    bound = e * (mag + out.abs()) * (1 + 4 * e) + 4 * (S + r)[..., None] * mag + torch.finfo(dtype).tiny
    off = (got.double().cpu() - out).abs() - bound
    assert not torch.isnan(got).any(), what
    assert off.max().item() <= 0, "%s over its bound by %.3g" % (what, off.max().item())
    fine = torch.isfinite(rl)
    assert torch.equal(lse.cpu()[~fine].double(), rl[~fine]), what
    off = (lse.double().cpu() - rl).abs()[fine] - (2 * S + r + 4 * U * rl.abs().nan_to_num(posinf=0.0))[fine]
    assert off.numel() == 0 or off.max().item() <= 0, "%s lse over its bound by %.3g" % (what, off.max().item())


def _poison(kp, vp, table, lens, page, free):
    """NaN where no sequence has a key: the rest of the last pages, and pages that nobody holds."""
    for m, n in enumerate(lens):
        if n > 0 and n % page:
            pg = int(table[m, n // page])
            kp[pg, :, n % page:] = math.nan
            vp[pg, :, n % page:] = math.nan
    for pg in free:
        kp[pg] = math.nan
        vp[pg] = math.nan


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dh", [32, 64, 128])
@pytest.mark.parametrize("Hkv,group", [(8, 1), (1, 1), (2, 2), (3, 3), (2, 8), (1, 16), (1, 20), (2, 40)])
@pytest.mark.parametrize("page,lens", [(16, [1, 0, 17, 333]), (64, [64, 5, 700]), (32, [31, 32, 33, 1, 100, 65])])
def test_attn_paged_decode(dtype, dh, Hkv, group, page, lens):
    from ttts_amd import ops
    table, P, free = _tables(lens, page, dh + group)
    kp, vp = _cache(P, Hkv, page, dh, dtype, dh * page)
    _poison(kp, vp, table, lens, page, free)
    M, H = len(lens), Hkv * group
    q = (torch.randn(M, H, dh, generator=_gen(3)) * 1.5).to(dtype).cuda()
    out, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), dh ** -0.5)
    _check(out, lse, _ref(q, kp, vp, table, lens, dh ** -0.5), lens, dtype)
    assert out.dtype == dtype and not out[torch.tensor(lens) == 0].any()


@pytest.mark.parametrize("dtype,dh,Hkv,group,page,lens", [
    (torch.bfloat16, 64, 8, 1, 16, [2404]), (torch.float16, 128, 2, 8, 64, [9001, 1]), (torch.bfloat16, 64, 1, 4, 128, [20011]),
    (torch.bfloat16, 32, 1, 1, 1024, [5000, 12345, 0]), (torch.float16, 64, 4, 2, 32, list(range(1, 200, 7)))])
def test_attn_paged_decode_long_and_ragged(dtype, dh, Hkv, group, page, lens):
    from ttts_amd import ops
    table, P, free = _tables(lens, page, 1)
    kp, vp = _cache(P, Hkv, page, dh, dtype, 2)
    _poison(kp, vp, table, lens, page, free)
    q = (torch.randn(len(lens), Hkv * group, dh, generator=_gen(4)) * 2).to(dtype).cuda()
    out, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), dh ** -0.5)
    _check(out, lse, _ref(q, kp, vp, table, lens, dh ** -0.5), lens, dtype)


@pytest.mark.parametrize("dtype,dh,M,Hkv,group,page,longest", [
    (torch.bfloat16, 64, 70, 8, 1, 16, 300), (torch.float16, 128, 33, 16, 2, 32, 200), (torch.bfloat16, 32, 520, 1, 5, 16, 90),
    (torch.bfloat16, 64, 512, 1, 1, 16, 100), (torch.float16, 32, 257, 2, 3, 16, 60),
    (torch.bfloat16, 64, 70, 8, 1, 16, 5001)])
def test_many_sequences(dtype, dh, M, Hkv, group, page, longest):
    """As many sequences and heads as fill the card: no split up to 4096 keys, chunks beyond."""
    from ttts_amd import ops
    g = _gen(M)
    lens = torch.randint(0, min(longest, 130), (M,), generator=g).tolist()
    lens[3], lens[M - 1] = longest, 1
    table, P, free = _tables(lens, page, 1)
    kp, vp = _cache(P, Hkv, page, dh, dtype, 2)
    _poison(kp, vp, table, lens, page, free)
    q = (torch.randn(M, Hkv * group, dh, generator=_gen(4)) * 2).to(dtype).cuda()
    out, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), dh ** -0.5)
    some = sorted({0, 3, 4, 5, M // 2, M - 2, M - 1})
    pick = torch.tensor(some)
    ref = _ref(q[pick.cuda()], kp, vp, table[pick], [lens[i] for i in some], dh ** -0.5)
    _check(out[pick.cuda()], lse[pick.cuda()], ref, lens, dtype)
    assert torch.isfinite(out).all() and torch.equal(torch.isinf(lse).all(dim=1).cpu(), torch.tensor(lens) == 0)


def test_lengths_and_tables_out_of_range():
    """A negative length, one beyond the table, table entries outside the cache in the middle and over a whole sequence."""
    from ttts_amd import ops
    page, dh, Hkv, dtype = 16, 64, 2, torch.bfloat16
    lens = [200, 200, 200, 200, 40]
    table, P, _ = _tables(lens, page, 5)
    table[0, 3], table[0, 4], table[0, 12] = -1, P, 2 ** 31 - 1
    table[1, :] = -2 ** 31
    kp, vp = _cache(P, Hkv, page, dh, dtype, 6)
    q = torch.randn(5, 4, dh, generator=_gen(7)).to(dtype).cuda()
    said = [200, 200, -3, 10 ** 9, 40]
    out, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor(said, dtype=torch.int32).cuda(), 0.125)
    _check(out, lse, _ref(q, kp, vp, table, said, 0.125), [208], dtype)
    assert not out[1].any() and not out[2].any() and (lse[1:3] == -math.inf).all()


def test_large_scores_and_infinite_keys():
    """Scores of thousands (the maximum is taken off first), a negative scale, and a key of -inf scores beside others."""
    from ttts_amd import ops
    page, dh, dtype, lens = 16, 64, torch.float16, [300, 77]
    table, P, _ = _tables(lens, page, 5)
    kp, vp = _cache(P, 2, page, dh, dtype, 6)
    q = (torch.randn(2, 4, dh, generator=_gen(7)) * 40).to(dtype).cuda()
    for scale in (3.0, -0.5):
        out, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale)
        _check(out, lse, _ref(q, kp, vp, table, lens, scale), lens, dtype, "scale %g" % scale)
    pos = q.abs() + 0.5
    kp[int(table[0, 2]), :, 5] = -math.inf
    kp[int(table[0, 9]), :, 0] = -math.inf
    out, lse = ops.attn_paged_decode(pos, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), 0.125)
    ref = _ref(pos, kp, vp, table, lens, 0.125)
    finite_k = kp.nan_to_num(neginf=0.0)                   # for the size of the scores' error only
    ref = (ref[0], ref[1], ref[2], _ref(pos, finite_k, vp, table, lens, 0.125)[3])
    _check(out, lse, ref, lens, dtype, "infinite keys")


def test_views_and_sliced_tables():
    """Queries as a part of a packed projection, an output inside a wider buffer (the rest stays), a table cut to its first pages."""
    from ttts_amd import ops
    page, dh, Hkv, H, dtype = 16, 64, 2, 6, torch.bfloat16
    lens = [90, 33, 64]
    table, P, _ = _tables(lens, page, 5, width=9)
    kp, vp = _cache(P, Hkv, page, dh, dtype, 8)
    packed = torch.randn(3, (H + 2 * Hkv) * dh, generator=_gen(1)).to(dtype).cuda()
    q = packed[:, :H * dh].view(3, H, dh)
    wide = torch.full((3, 2 * H, dh), 7.0, dtype=dtype, device="cuda")
    L = torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), L, 0.1, out=wide[:, 1::2])
    _check(out, lse, _ref(q, kp, vp, table, lens, 0.1), lens, dtype)
    assert (wide[:, ::2] == 7.0).all()
    one = torch.randn(1, (H + 2 * Hkv) * dh + 4, generator=_gen(2)).to(dtype).cuda()[:, :(H + 2 * Hkv) * dh]   # one row: its pitch says nothing
    ops.kv_page_write(one[:, H * dh:(H + Hkv) * dh].view(1, Hkv, dh), one[:, (H + Hkv) * dh:].view(1, Hkv, dh), kp, vp,
                      torch.tensor([int(table[2, 3]) * page + 15]).cuda())
    assert torch.equal(kp[int(table[2, 3]), :, 15], one[0, H * dh:(H + Hkv) * dh].view(Hkv, dh))
    cut = table.cuda()[:, :3]
    out, lse = ops.attn_paged_decode(q, kp, vp, cut, L, 0.1)
    _check(out, lse, _ref(q, kp, vp, table[:, :3], lens, 0.1), lens, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,H,dh,page", [(1, 8, 64, 16), (7, 1, 32, 32), (300, 3, 128, 16), (5000, 2, 64, 1024), (65, 17, 128, 16), (40, 64, 64, 32)])
def test_kv_page_write(dtype, N, H, dh, page):
    from ttts_amd import ops
    P = -(-N // page) + 2
    kp, vp = _cache(P, H, page, dh, dtype, N)
    k0, v0 = kp.clone(), vp.clone()
    packed = torch.randn(N, 3 * H, dh, generator=_gen(2)).to(dtype).cuda()
    k, v = packed[:, H:2 * H], packed[:, 2 * H:]
    slots = torch.randperm(P * page, generator=_gen(3))[:N]
    if N > 4:
        slots[0], slots[1], slots[2], slots[3] = -1, P * page, 2 ** 62, -2 ** 63
    ops.kv_page_write(k, v, kp, vp, slots.cuda())
    for n in range(N):
        s = int(slots[n])
        if 0 <= s < P * page:
            k0[s // page, :, s % page] = k[n]
            v0[s // page, :, s % page] = v[n]
    assert torch.equal(kp.view(torch.int16), k0.view(torch.int16)) and torch.equal(vp.view(torch.int16), v0.view(torch.int16))


def test_nothing_to_do():
    from ttts_amd import ops
    kp, vp = _cache(2, 1, 16, 32, torch.bfloat16, 1)
    e = torch.empty(0, 1, 32, dtype=torch.bfloat16, device="cuda")
    ops.kv_page_write(e, e, kp, vp, torch.empty(0, dtype=torch.int64, device="cuda"))
    out, lse = ops.attn_paged_decode(e, kp, vp, torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), 1.0)
    assert out.shape == (0, 1, 32) and lse.shape == (0, 1)


def test_cache_past_32_bits():
    """Pages whose elements lie past 2^31 (a cache of 2 x 4.8 GB)."""
    from ttts_amd import ops
    page, Hkv, dh, dtype = 1024, 8, 128, torch.bfloat16
    P = 2300                                               # 2300 x 8 x 1024 x 128 = 2.4e9 elements
    kp = torch.zeros(P, Hkv, page, dh, dtype=dtype, device="cuda")
    vp = torch.zeros_like(kp)
    N = 50
    k, v = (torch.randn(N, Hkv, dh, generator=_gen(s)).to(dtype).cuda() for s in (1, 2))
    slots = torch.arange(N) + (P - 1) * page
    ops.kv_page_write(k, v, kp, vp, slots.cuda())
    assert torch.equal(kp[P - 1, :, :N], k.transpose(0, 1)) and torch.equal(vp[P - 1, :, :N], v.transpose(0, 1))
    q = torch.randn(1, Hkv, dh, generator=_gen(3)).to(dtype).cuda()
    out, lse = ops.attn_paged_decode(q, kp, vp, torch.tensor([[P - 1]], dtype=torch.int32).cuda(), torch.tensor([N], dtype=torch.int32).cuda(), dh ** -0.5)
    _check(out, lse, _ref(q, kp[P - 1:], vp[P - 1:], torch.zeros(1, 1, dtype=torch.int32), [N], dh ** -0.5), [N], dtype)


def test_streams_and_graphs():
    """On a side stream, and two captured graphs alive at once: every replay gives what the eager calls give."""
    from ttts_amd import ops
    page, dh, Hkv, H, dtype = 16, 64, 2, 4, torch.bfloat16
    lens = [3000, 1, 517]                                  # long enough to be split
    table, P, _ = _tables(lens, page, 5)
    table = table.cuda()
    kp, vp = _cache(P, Hkv, page, dh, dtype, 8)
    qs = [torch.randn(3, H, dh, generator=_gen(s)).to(dtype).cuda() for s in range(3)]
    Ls = [torch.tensor([n - d for n in lens], dtype=torch.int32).cuda() for d in (0, 1, 30)]
    step = lambda q, L: ops.attn_paged_decode(q, kp, vp, table, L, 0.125)  # noqa: E731
    want = [step(q, L) for q, L in zip(qs, Ls)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(qs[1], Ls[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    static = [(qs[0].clone(), Ls[0].clone()) for _ in range(2)]
    graphs, outs = [], []
    for q, L in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(q, L))
        graphs.append(g)
    for n in range(4):
        for j in (0, 1):
            static[j][0].copy_(qs[(n + j) % 3]); static[j][1].copy_(Ls[(n + j) % 3])
        graphs[0].replay(); graphs[1].replay()
        step(qs[2], Ls[2])
        torch.cuda.synchronize()
        for j in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[j], want[(n + j) % 3])), (n, j)


def test_refusals_on_the_gpu():
    from ttts_amd import ops
    from ttts_amd.lib import TttsError
    bf = torch.bfloat16
    kp, vp = _cache(3, 2, 16, 64, bf, 1)
    q = torch.zeros(2, 4, 64, dtype=bf, device="cuda")
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    k, slots = torch.zeros(2, 2, 64, dtype=bf, device="cuda"), torch.arange(2, device="cuda")
    off = torch.zeros(2 * 4 * 64 + 1, dtype=bf, device="cuda")[1:].view(2, 4, 64)
    att = ops.attn_paged_decode
    bad = [lambda: att(q.half(), kp, vp, table, lens, 1.0), lambda: att(q[:, :3], kp, vp, table, lens, 1.0), lambda: att(q, kp, vp, table.long(), lens, 1.0),
           lambda: att(q, kp, vp, table[:1], lens, 1.0), lambda: att(q, kp, vp, table, lens[:1], 1.0), lambda: att(q, kp, vp, table, lens.long(), 1.0),
           lambda: att(q, kp, vp, table, lens, math.inf), lambda: att(q, kp.float(), vp.float(), table, lens, 1.0), lambda: att(off, kp, vp, table, lens, 1.0),
           lambda: att(q, kp[:, :, :8].contiguous(), vp[:, :, :8].contiguous(), table, lens, 1.0), lambda: att(q, kp.transpose(1, 2), vp.transpose(1, 2), table, lens, 1.0),
           lambda: att(q[..., :48], kp[..., :48].contiguous(), vp[..., :48].contiguous(), table, lens, 1.0), lambda: att(q, kp, vp[:2], table, lens, 1.0),
           lambda: att(q, kp, vp, table, lens.cpu(), 1.0), lambda: att(q, kp, vp, table[:, :0], lens, 1.0),
           lambda: att(q, kp, vp, table, lens, 1.0, out=torch.zeros(2, 4, 32, dtype=bf, device="cuda")),
           lambda: ops.kv_page_write(k, k.half(), kp, vp, slots), lambda: ops.kv_page_write(k, k, kp, vp, slots.int()), lambda: ops.kv_page_write(k, k, kp, vp, slots[:1]),
           lambda: ops.kv_page_write(k.transpose(1, 2), k, kp, vp, slots), lambda: ops.kv_page_write(k, k, kp.cpu(), vp, slots),
           lambda: ops.kv_page_write(k, k, kp, vp, slots[None])]
    for n, f in enumerate(bad):
        with pytest.raises(TttsError):
            f()
            pytest.fail("refusal %d did not come" % n)


def _one_far(n, far, dtype, dh=32, page=64, big=1024.0):
    """One sequence of n keys: the first scores 0 (bits) with value 0, the others `far` bits below with value `big`."""
    table, P, _ = _tables([n], page, 4)
    kp, vp = torch.zeros(P, 1, page, dh, dtype=dtype), torch.zeros(P, 1, page, dh, dtype=dtype)
    for pg in table[0].tolist():
        kp[pg, :, :, 0], vp[pg] = 1.0, big
    kp[int(table[0, 0]), :, 0], vp[int(table[0, 0]), :, 0] = 0.0, 0.0
    q = torch.zeros(1, 1, dh, dtype=dtype)
    q[0, 0, 0] = -far
    return q.cuda(), kp.cuda(), vp.cuda(), table


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,far", [(4096, 25.5), (500, 20.0), (30000, 28.0)])
def test_attn_paged_decode_small_weights_add_up(dtype, n, far):
    """Weights of 2^-20 .. 2^-28 of the largest, thousands of them: less than fp16's own steps, and all there is of the result."""
    from ttts_amd import ops
    q, kp, vp, table = _one_far(n, far, dtype)
    out, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), math.log(2.0))
    ref, _, rl, S = _ref(q, kp, vp, table, [n], math.log(2.0))
    e = torch.finfo(dtype).eps / 2                       # the weights once, the result once
    r = (n / 64 + 32) * U
    assert ((out.double().cpu() - ref).abs() <= ref.abs() * (2.1 * e + 4 * (S[..., None] + r))).all(), (out[0, 0, 0].item(), ref[0, 0, 0].item())
    assert ((lse.double().cpu() - rl).abs() <= 2 * S + r).all()


@pytest.mark.parametrize("n", [1, 40, 1500])
def test_attn_paged_decode_scores_at_the_end_of_the_range(n):
    """Scores (in bits) between -3.0e38 and the lowest fp32 number are scores: equal ones share the values."""
    from ttts_amd import ops
    table, P, _ = _tables([n], 64, 5)
    kp, vp = _cache(P, 1, 64, 32, torch.bfloat16, 6)
    kp.zero_()
    kp[..., 0] = -(2.0 ** 64)
    q = torch.zeros(1, 1, 32, dtype=torch.bfloat16).cuda()
    q[0, 0, 0] = 1.7265625 * 2.0 ** 63                   # product -2.93e38; times 0.75 log2 e: -3.18e38
    out, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), 0.75)
    ref, mag, rl, _ = _ref(q, kp, vp, table, [n], 0.75)
    e = torch.finfo(torch.bfloat16).eps / 2
    assert ((out.double().cpu() - ref).abs() <= e * (mag + ref.abs()) * 1.1 + (n / 64 + 32) * U * mag).all()
    assert ((lse.double().cpu() - rl).abs() <= 8 * U * rl.abs()).all()


def test_attn_paged_decode_out_must_not_overlap():
    from ttts_amd import ops
    from ttts_amd.lib import TttsError
    table, P, _ = _tables([5, 6], 16, 7)
    kp, vp = _cache(P, 2, 16, 32, torch.bfloat16, 8)
    q = torch.randn(2, 4, 32, generator=_gen(9)).to(torch.bfloat16).cuda()
    args = (q, kp, vp, table.cuda(), torch.tensor([5, 6], dtype=torch.int32).cuda(), 0.2)
    want, _ = ops.attn_paged_decode(*args)
    one = torch.zeros(1, 1, 32, dtype=torch.bfloat16).cuda()
    for out in (one.expand(2, 4, 32), torch.zeros(2, 1, 32, dtype=torch.bfloat16).cuda().expand(2, 4, 32),
                torch.zeros(512, dtype=torch.bfloat16).cuda().as_strided((2, 4, 32), (32, 32, 1))):
        with pytest.raises(TttsError, match="overlap"):
            ops.attn_paged_decode(*args, out=out)
    across = torch.zeros(4, 2, 40, dtype=torch.bfloat16).cuda()[..., :32].transpose(0, 1)   # heads first in memory, with a pitch
    got, _ = ops.attn_paged_decode(*args, out=across)
    assert got is across and torch.equal(across, want)


def _vectorised(q, kp, vp, table, lens, scale):
    """(out, sum p |v|, lse, size of the scores' error) in 64 bits on the GPU, one sequence and cached head at a time."""
    M, H, dh = q.shape
    Hkv, page = kp.shape[1], kp.shape[2]
    group = H // Hkv
    out, mag = torch.zeros(2, M, H, dh, dtype=torch.float64, device="cuda")
    S = torch.zeros(M, H, dtype=torch.float64, device="cuda")
    for m, n in enumerate(lens):
        ids = table[m, :-(-n // page)].long().cuda()
        for h in range(Hkv if n else 0):
            k, v = (t[ids, h].reshape(-1, dh)[:n].double() for t in (kp, vp))
            heads = slice(h * group, (h + 1) * group)
            qs = q[m, heads].double()
            w = torch.softmax(qs @ k.t() * scale, dim=1)
            out[m, heads], mag[m, heads] = w @ v, w @ v.abs()
            S[m, heads] = (qs.abs() @ k.abs().t()).amax(dim=1) * abs(scale) * (dh + 8) * U
    return out, mag, S


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dh,Hkv,group,page,lens", [
    (64, 8, 1, 16, [613]), (64, 2, 3, 16, [2404, 0, 17, 900, 1]), (128, 2, 8, 64, [9001, 300]), (32, 1, 20, 32, [1500, 31]),
    (64, 4, 4, 16, list(range(2, 34))),
    (128, 8, 5, 32, [40 + 29 * i for i in range(70)])])
def test_attn_paged_decode_weights_are_not_rounded_to_the_cache_type(dtype, dh, Hkv, group, page, lens):
    """A weight enters the product with V in two parts of the cache's type, so the result has one rounding to that type, its own.  The first
    part is at most three half steps below the weight (3 e of it), the second off by e of that: 3 e^2 of the weight, doubled here."""
    from ttts_amd import ops
    table, P, _ = _tables(lens, page, 11)
    kp, vp = _cache(P, Hkv, page, dh, dtype, 12)
    q = (torch.randn(len(lens), Hkv * group, dh, generator=_gen(13)) * 1.5).to(dtype).cuda()
    scale = dh ** -0.5
    got, _ = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale)
    out, mag, S = _vectorised(q, kp, vp, table, lens, scale)
    e = torch.finfo(dtype).eps / 2
    r = (max(lens) / 64 + 32) * U
    inner = (6 * e * e + 4 * (S[..., None] + r)) * mag + torch.finfo(dtype).tiny
    off = (got.double() - out).abs() - e * (out.abs() + inner) - inner
    assert off.max().item() <= 0, off.max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attn_paged_decode_infinite_values(dtype):
    """A value of +inf among the keys of a sequence makes its column inf, as the definition does; the other columns stay."""
    from ttts_amd import ops
    lens = [1, 40, 900]
    table, P, _ = _tables(lens, 16, 14)
    kp, vp = _cache(P, 1, 16, 64, dtype, 15)
    for m in range(3):
        vp[int(table[m, 0]), 0, 0, 5 + m] = math.inf
    q = torch.randn(3, 2, 64, generator=_gen(16)).to(dtype).cuda() * 0.5
    got, _ = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), 0.125)
    for m in range(3):
        assert (got[m, :, 5 + m] == math.inf).all(), m
    others = torch.ones(3, 64, dtype=torch.bool)
    others[torch.arange(3), torch.arange(3) + 5] = False
    assert torch.isfinite(got.cpu()[others[:, None].expand(3, 2, 64)]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hkv", [1, 7])
def test_attn_paged_decode_longest_sequences(dtype, Hkv):
    """More than 2048 * 4096 keys, by a table that repeats a few pages: about 2000 parts, as many as there may be.  The last page
    is its own, and two keys of it hold a good part of the first queries' weight."""
    from ttts_amd import ops
    page, dh, pool = 1024, 32, 24
    width = 2048 * 4096 // page + 300
    g = _gen(Hkv)
    kp, vp = _cache(pool + 1, Hkv, page, dh, dtype, 21)
    table = torch.randint(0, pool, (1, width), generator=g, dtype=torch.int32)
    n = width * page - 100
    table[0, -1] = pool
    q = torch.randn(1, 2 * Hkv, dh, generator=g).to(dtype).cuda()
    scale = dh ** -0.5
    times = torch.bincount(table[0, :-1].long(), minlength=pool).double().cuda()
    vp[pool, :, :page - 100] = 3.0
    for key in (0, page - 101):
        kp[pool, :, key] = 0.0
        for h in range(Hkv):       # a key along each head's first query: its score is log(keys) and a little
            a = q[0, 2 * h].float()
            kp[pool, h, key] = (a * (15.6 / scale / (a @ a))).to(dtype)
    got, lse = ops.attn_paged_decode(q, kp, vp, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), scale)
    e = torch.finfo(dtype).eps / 2
    r = (32 * 8 + 2048 / 8 + 32) * U          # a lane's share of a part, a thread's share of the parts, and the rest
    for h in range(2 * Hkv):
        k, v = kp[:, h // 2].double(), vp[:, h // 2].double()
        z = k @ q[0, h].double() * scale
        z[pool, page - 100:] = -math.inf
        w = torch.exp(z - z.max()) * torch.cat([times, times.new_ones(1)])[:, None]
        L = w.sum()
        ref, mag = ((w / L)[..., None] * v).sum(dim=(0, 1)), ((w / L)[..., None] * v.abs()).sum(dim=(0, 1))
        S = (k.abs() @ q[0, h].double().abs()).max() * scale * (dh + 8) * U
        bound = e * ref.abs() + (1 + e) * (6 * e * e + 4 * (S + r)) * mag + torch.finfo(dtype).tiny
        assert ((got[0, h].double() - ref).abs() <= bound).all(), h
        want = z.max() + L.log()
        assert (lse[0, h].double() - want).abs() <= 2 * S + r + 4 * U * want.abs(), h
        if h % 2 == 0:
            assert 0.1 < (w[pool].sum() / L).item()
