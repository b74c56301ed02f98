"""Token log-probabilities with entropy and alternatives, and distillation on a teacher's alternatives (csrc/scoring.hip), against
their definitions in 64 bits.  Tolerances are error bounds of fp32 arithmetic (U = 2^-24, half a step of a value near one):
 * a row's log Z: its terms are each off by a few U (the exponential is good to one step), and a sum of C of them, taken in
   parts of at most C / 64 by one lane, by at most (C / 64 + 32) U of itself;
 * log p = (x - m) / T - log Z: two more roundings of the size of |log p|, and of |(x - m) / T| <= |log p|.
Outputs of 16 bits add half a step of their type, torch.finfo(t).eps / 2 of the value (and of its smallest step near zero)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LOWEST = {torch.float32: -3.4e38, torch.bfloat16: -3.3e38, torch.float16: -65504.0}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _logits(R, C, pitch, dtype, seed, offset=0, std=3.0):
    """[R, pitch] rows on the GPU, `offset` elements into their allocation; the columns from C on hold NaN."""
    buf = torch.full((offset + R * pitch,), math.nan, dtype=dtype, device="cuda")
    x = buf[offset:].view(R, pitch)
    x[:, :C] = (torch.randn(R, C, generator=_gen(seed)) * std).to(dtype).cuda()
    return x


def _inside(got, ref, bound, what):
    got, ref = got.double().cpu(), ref.cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), what
    fine = torch.isfinite(ref)
    off = (got - ref).abs()[fine] - bound[fine]
    assert off.numel() == 0 or off.max().item() <= 0, "%s: over its bound by %.3g" % (what, off.max().item())


def _half_step(ref, dtype):
    f = torch.finfo(dtype)
    return f.eps / 2 * ref.abs() + f.tiny * f.eps


def _ref_logprobs(x, tokens, C, top_k, T):
    """logp, entropy, top_logp, top_idx, y in 64 bits (rows with a distribution)."""
    x = x[:, :C].double().cpu()
    tokens = tokens.cpu()
    y = torch.log_softmax(x / T, dim=1)
    given = (tokens >= 0) & (tokens < C)
    logp = torch.where(given, y.gather(1, tokens.clamp(0, C - 1)[:, None])[:, 0], 0.0)
    ent = torch.special.entr(y.exp()).sum(dim=1)
    k = min(top_k, C)
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    v, i = v[:, :k], i[:, :k]
    tl = torch.where(v > -math.inf, y.gather(1, i), -math.inf)
    ti = torch.where(v > -math.inf, i, -1)
    pad = top_k - k
    return logp, ent, torch.nn.functional.pad(tl, (0, pad), value=-math.inf), torch.nn.functional.pad(ti, (0, pad), value=-1), y, given


def _r(C):
    return (C / 64 + 32) * U


SHAPES = [(1, 1, 1, 0), (3, 2, 2, 0), (5, 9, 16, 0), (8, 1026, 1088, 0), (130, 1026, 1026, 0), (7, 515, 515, 1), (33, 2048, 2048, 0),
          (9, 2049, 2056, 0), (6, 8194, 8256, 0), (4, 8195, 8195, 3), (3, 32768, 32768, 0), (2, 32801, 32808, 0), (2, 100003, 100003, 1),
          (1, 300007, 300008, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C,pitch,offset", SHAPES)
@pytest.mark.parametrize("top_k,T", [(0, 1.0), (5, 0.7), (64, 2.0)])
def test_token_logprobs(R, C, pitch, offset, dtype, top_k, T):
    from ttts_amd import ops
    x = _logits(R, C, pitch, dtype, R + C, offset)
    tokens = torch.randint(0, C, (R,), generator=_gen(C)).cuda()
    tokens[R // 2] = -1 if R % 2 else C
    r = ops.token_logprobs_fwd(x, tokens, C=C, top_k=top_k, temperature=T)
    logp, ent, tl, ti, y, given = _ref_logprobs(x, tokens, C, top_k, T)
    _inside(r.logp, logp, _r(C) + 4 * U * logp.abs(), "logp")
    # entropy = log Z - sum e t / Z: a second sum of that kind, of terms whose sum is entropy - log Z
    span = (ent.abs() + (y.max(dim=1).values).abs() + 1)
    _inside(r.entropy, ent, 3 * _r(C) * span, "entropy")
    if top_k:
        assert torch.equal(r.top_idx.cpu(), ti)
        _inside(r.top_logp, tl, _r(C) + 4 * U * tl.abs().nan_to_num(posinf=0.0), "top_logp")
    else:
        assert r.top_idx is None and r.top_logp is None
    lse = torch.logsumexp(x[:, :C].double().cpu() / T, dim=1)
    s = r.stats.double().cpu()
    _inside(s[:, 0] / T + s[:, 1], lse, _r(C) + 4 * U * s[:, 1].abs(), "log-sum-exp")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C,pitch,offset", [s for s in SHAPES if s[1] < 200000])
@pytest.mark.parametrize("T,with_entropy", [(1.0, True), (0.7, False), (2.0, True)])
def test_token_logprobs_gradient(R, C, pitch, offset, dtype, T, with_entropy):
    from ttts_amd import ops
    x = _logits(R, C, pitch, dtype, 7 * R + C, offset)
    tokens = torch.randint(0, C, (R,), generator=_gen(C + 1)).cuda()
    tokens[R // 2] = -5 if R % 2 else C + 3
    g_l, g_h = torch.randn(R, generator=_gen(5)), torch.randn(R, generator=_gen(6))
    r = ops.token_logprobs_fwd(x, tokens, C=C, temperature=T)
    d = ops.token_logprobs_bwd(x, tokens, r.stats, r.entropy, g_l.cuda(), g_h.cuda() if with_entropy else None, C=C, temperature=T)
    leaf = x[:, :C].double().cpu().requires_grad_(True)
    y = torch.log_softmax(leaf / T, dim=1)
    tok = tokens.cpu()
    given = (tok >= 0) & (tok < C)
    total = (y.gather(1, tok.clamp(0, C - 1)[:, None])[:, 0] * g_l.double() * given).sum()
    if with_entropy:
        total = total - ((y.exp() * y).sum(dim=1) * g_h.double()).sum()
    ref, = torch.autograd.grad(total, leaf)
    y = y.detach()
    p = y.exp()
    ent = torch.special.entr(p).sum(dim=1)
    gl, gh = (g_l.double().abs() * given)[:, None], (g_h.double().abs() * with_entropy)[:, None]
    # p is off by (_r(C) + 4 U |y|) of itself, y + H by that and three steps of the larger
    size = (gl * p + gh * p * (y.abs() + ent[:, None] + 1)) / T
    bound = size * (4 * _r(C) + 8 * U * (y.abs() + 1)) + 4 * U * gl / T + _half_step(ref, dtype) + 1e-37
    _inside(d[:, :C], ref, bound, "dlogits")
    assert d.dtype == dtype and d.shape == x.shape and not d[:, C:].any()
    # in the logits' own place
    x2 = x.clone() if offset == 0 else x
    d2 = ops.token_logprobs_bwd(x2, tokens, r.stats, r.entropy, g_l.cuda(), g_h.cuda() if with_entropy else None, C=C, temperature=T, dlogits=x2)
    assert d2 is x2 and torch.equal(d2, d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C", [70, 1026, 8195, 40000])
def test_token_logprobs_special_rows(dtype, C):
    """Rows whose mask leaves nothing or little, the type's lowest value, infinities, NaN, constant rows, zeros of both signs."""
    from ttts_amd import ops
    x = _logits(12, C, C, dtype, 3)
    x[0] = -math.inf                                       # nothing left
    x[1] = LOWEST[dtype]                                   # a mask of the lowest value on everything: uniform
    x[2] = -math.inf; x[2, C // 2] = 1.5                   # one class left
    x[3] = -math.inf; x[3, 1::2] = x[4, 1::2]              # half the classes
    x[5, C // 3] = math.nan
    x[6, C // 3] = math.inf
    x[7] = 0.25                                            # constant: alternatives in the order of the classes
    x[8] = -0.0; x[8, 5::3] = 0.0                          # zeros of both signs are equal
    x[9] = LOWEST[dtype]; x[9, 3] = 2.0; x[9, C - 1] = 2.0 # the lowest value beside ordinary ones
    x[10, : C // 2] = x[10, 0]                             # one value in half of the row
    x[11] = -math.inf; x[11, 0] = math.nan
    tokens = torch.arange(12).remainder(C).cuda()
    tokens[2] = C // 2; tokens[9] = C - 1; tokens[1] = C - 1
    k = 20
    r = ops.token_logprobs_fwd(x, tokens, top_k=k)
    keep = torch.tensor([i for i in range(12) if i not in (0, 5, 6, 11)])
    logp, ent, tl, ti, y, _ = _ref_logprobs(x[keep.cuda()], tokens[keep.cuda()], C, k, 1.0)
    span = ent.abs() + y.max(dim=1).values.abs() + 1
    _inside(r.logp.cpu()[keep], logp, _r(C) + 4 * U * logp.abs().nan_to_num(posinf=0.0), "logp")
    _inside(r.entropy.cpu()[keep], ent, 3 * _r(C) * span, "entropy")
    assert torch.equal(r.top_idx.cpu()[keep], ti)
    _inside(r.top_logp.cpu()[keep], tl, _r(C) + 4 * U * tl.abs().nan_to_num(posinf=0.0), "top_logp")
    assert r.logp[0].item() == -math.inf and r.entropy[0].item() == 0.0 and (r.top_idx[0] == -1).all() and (r.top_logp[0] == -math.inf).all()
    for i in (5, 6, 11):
        assert torch.isnan(r.logp[i]) and torch.isnan(r.entropy[i]) and torch.isnan(r.top_logp[i]).all() and (r.top_idx[i] == -1).all(), i
    ones = torch.ones(12, device="cuda")
    d = ops.token_logprobs_bwd(x, tokens, r.stats, r.entropy, ones, ones)
    assert not d[0].any() and torch.isnan(d[5]).any() and torch.isnan(d[6]).any()
    leaf = x[keep.cuda()].double().cpu()
    p = y.exp()
    ref = -p - torch.where(p > 0, p * (y.clamp(min=-1e4) + ent[:, None]), 0.0)
    ref[torch.arange(len(keep)), tokens.cpu()[keep]] += 1.0
    size = p * (y.abs().nan_to_num(posinf=0.0).clamp(max=1e4) + ent[:, None] + 2)
    assert torch.isfinite(leaf.exp()).any()
    _inside(d.cpu()[keep], ref, size * (4 * _r(C) + 8 * U * 100) + 4 * U + _half_step(ref, dtype), "dlogits")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C", [65, 100, 2048, 2049, 2561, 5000, 8194, 16384, 16385, 40000, 131072, 131081, 600001])
@pytest.mark.parametrize("top_k", [1, 33, 64])
def test_alternatives_where_values_repeat_or_crowd(dtype, C, top_k):
    """Rows whose largest values sit in few of a wave's lanes, sorted rows, rows of one, two and few values, few classes left: the
    alternatives are the stable order's, whatever the search for them runs into."""
    from ttts_amd import ops
    g = _gen(C + top_k)
    base = torch.randn(C, generator=g)
    at = torch.arange(C)
    rows = [base + 30.0 * ((at // 8) % 64 == 5),                        # one lane's columns
            base + 30.0 * ((at // 8) % 64 == 5) * (at % 8 == 3) + 20.0 * (at % 8 == 0),
            base.sort().values, base.sort(descending=True).values,
            torch.full((C,), -2.5), torch.where(torch.rand(C, generator=g) < 0.5, 1.0, 0.0), torch.where(at == C - 1, 1.0, 0.0),
            torch.randint(-3, 1, (C,), generator=g).float(),            # values below zero, repeated
            torch.where(at % 97 == 64, base, torch.tensor(-math.inf)),
            4096.0 + (at % 7).float() * 2.0 ** -11 if dtype == torch.float32 else base.round(),
            torch.where(at < C // 2, torch.tensor(LOWEST[dtype]), torch.tensor(-math.inf)),
            -base.abs() - 3.0]
    x = torch.stack(rows).to(dtype).cuda()
    r = ops.token_logprobs_fwd(x, torch.zeros(len(rows), dtype=torch.int64, device="cuda"), top_k=top_k)
    _, _, tl, ti, _, _ = _ref_logprobs(x, torch.zeros(len(rows), dtype=torch.int64), C, top_k, 1.0)
    assert torch.equal(r.top_idx.cpu(), ti)
    _inside(r.top_logp, tl, _r(C) + 4 * U * tl.abs().nan_to_num(posinf=0.0), "top_logp")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C,every,top_k", [(40000, 4, 64), (40000, 4, 9), (100003, 4, 33), (300000, 16, 64), (20000, 10, 20)])
def test_alternatives_crowd_into_few_parts_of_a_row(dtype, C, every, top_k):
    """The largest classes all in every `every`-th stretch of 2048, or all in one: few waves hold them, the others' bounds say little."""
    from ttts_amd import ops
    R = 5
    x = torch.randn(R, C, generator=torch.Generator().manual_seed(C + every))
    part = torch.arange(C) // 2048
    x[:3, part % every == 1] += 30.0
    x[3, part == every - 1] += 30.0
    x[4] = -x[4].abs() - 1.0                              # below zero throughout
    x = x.to(dtype).cuda()
    r = ops.token_logprobs_fwd(x, torch.zeros(R, dtype=torch.int64).cuda(), top_k=top_k)
    want = torch.sort(x.float().cpu(), dim=1, descending=True, stable=True).indices[:, :top_k]
    assert torch.equal(r.top_idx.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C,offset", [(600, 1), (1088, 3), (1089, 0), (2112, 1), (2113, 0), (2200, 5), (4600, 0), (16448, 1), (16449, 0), (32832, 0),
                                      (32833, 2), (131136, 0), (131137, 1)])
def test_alternatives_where_the_layout_of_a_row_changes(dtype, C, offset):
    """Widths around one wave's columns, the narrow rest, units of three steps, and the kernels' limits: the best classes are put
    at the first and last columns and around every multiple of 512 and of 2048."""
    from ttts_amd import ops
    R = 3
    g = torch.Generator().manual_seed(C)
    x = torch.randn(R, C + offset, generator=g)
    marks = sorted({c for m in (0, C) for c in range(m - 3, m + 3)} | {m + d for m in range(512, C, 512 if C < 6000 else 2048) for d in (-1, 0)})
    marks = [c for c in marks if 0 <= c < C]
    pick = torch.tensor(marks)[torch.randperm(len(marks), generator=g)[:40]]
    x[:, pick + offset] += 20.0
    x = x.to(dtype).cuda()[:, offset:]
    tok = pick[:R].clone().cuda()
    r = ops.token_logprobs_fwd(x, tok, top_k=64)
    y = x.float().cpu()
    assert torch.equal(r.top_idx.cpu(), torch.sort(y, dim=1, descending=True, stable=True).indices[:, :64])
    lp = torch.log_softmax(y.double(), dim=1)
    bound = _r(C) + 4 * U * y.abs().max().item()
    assert (r.logp.cpu().double() - lp.gather(1, tok.cpu()[:, None])[:, 0]).abs().max().item() <= bound
    # log Z - s / z: the one as above, the other's sums off by r of themselves each, |s / z| = log Z - H <= log C
    assert (r.entropy.cpu().double() + (lp.exp() * lp).sum(dim=1)).abs().max().item() <= bound * (1 + 2 * math.log(C))


def test_logits_far_from_zero():
    """The statistics hand the maximum and log Z on apart: rows around 4096 lose nothing of their gradient."""
    from ttts_amd import ops
    x = _logits(16, 1000, 1000, torch.float32, 1)
    far = x + 4096.0                                      # rounds x: the reference takes the rounded one
    tokens = torch.arange(16, device="cuda")
    one = torch.ones(16, device="cuda")
    r = ops.token_logprobs_fwd(far, tokens, top_k=3)
    d = ops.token_logprobs_bwd(far, tokens, r.stats, r.entropy, one)
    y = torch.log_softmax(far.double().cpu(), dim=1)
    ref = -y.exp()
    ref[torch.arange(16), torch.arange(16)] += 1
    _inside(d, ref, y.exp() * (4 * _r(1000) + 8 * U * (y.abs() + 1)) + 4 * U, "dlogits")


def _ref_distill(x, idx, t, C, T, tail):
    """(row_loss, p, listed, left, q_rest, y) in 64 bits; x leaf of [R, C] doubles."""
    y = torch.log_softmax(x / T, dim=1)
    there = (idx >= 0) & (idx < C)
    at = idx.clamp(0, C - 1)
    t = t.double()
    if tail:
        lp = t
        p = torch.where(there, t.exp(), 0.0)
    else:
        lp = torch.log_softmax((t / T).masked_fill(~there, -math.inf), dim=1).nan_to_num(nan=-math.inf)
        p = lp.exp()
    term = torch.where(p > 0, p * (torch.where(p > 0, lp, 0.0) - y.gather(1, at)), 0.0)
    loss = term.sum(dim=1)
    listed = torch.zeros(x.shape, dtype=torch.float64).scatter_add_(1, at, there.double()) > 0
    left = (1 - p.sum(dim=1)).clamp(min=0) if tail else torch.zeros(len(x), dtype=torch.float64)
    some = ((~listed) & (x.detach() > -math.inf)).any(dim=1)
    rest = torch.logsumexp(y.masked_fill(listed, -math.inf), dim=1)
    held = some & (left > 0)
    safe = torch.where(held, left, 1.0)
    loss = loss + torch.where(held, left * (safe.log() - torch.where(held, rest, 0.0)), 0.0)
    return loss, p, listed, torch.where(held, left, 0.0), rest, y


def _teacher(R, C, K, T, tail, seed, empty=0.1, repeat=False):
    g = _gen(seed)
    idx = torch.stack([torch.randperm(C, generator=g)[:K] if K <= C else torch.randint(0, C, (K,), generator=g) for _ in range(R)])
    t = torch.randn(R, K, generator=g) * 2
    if tail:
        t = torch.log_softmax(torch.cat([t, torch.full((R, 1), 1.0)], dim=1), dim=1)[:, :K].contiguous()
    gone = torch.rand(R, K, generator=g) < empty
    idx = torch.where(gone, torch.where(torch.rand(R, K, generator=g) < 0.5, -1, C + 2), idx)
    t = torch.where(gone, math.nan, t)                    # the value of an empty entry is not looked at
    if repeat and K >= 4:
        idx[:, K // 2] = idx[:, 0]; idx[:, K - 1] = idx[:, 0]
        for c in (K // 2, K - 1):
            t[:, c] = torch.where(idx[:, 0] == idx[:, c], torch.where(torch.isnan(t[:, 0]), t[:, 0], t[:, 0] - 1.0), t[:, c])
    return idx, t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C,pitch,offset", [s for s in SHAPES if s[1] < 200000])
@pytest.mark.parametrize("K,T,tail,repeat", [(1, 1.0, False, False), (20, 2.0, False, True), (64, 1.0, True, False), (128, 0.7, True, True)])
def test_distill(R, C, pitch, offset, dtype, K, T, tail, repeat):
    from ttts_amd import ops
    x = _logits(R, C, pitch, dtype, 11 * R + C, offset)
    repeat = repeat or K > C
    idx, t = _teacher(R, C, K, T, tail, C + K, repeat=repeat)
    g = torch.randn(R, generator=_gen(9))
    loss, stats = ops.distill_fwd(x, idx.cuda(), t.cuda(), C=C, temperature=T, tail=tail)
    d = ops.distill_bwd(x, idx.cuda(), t.cuda(), stats, g.cuda(), C=C, temperature=T, tail=tail)
    leaf = x[:, :C].double().cpu().requires_grad_(True)
    tz = torch.where((idx >= 0) & (idx < C), t, 0.0)
    ref, p, listed, left, rest, y = _ref_distill(leaf, idx, tz, C, T, tail)
    grad, = torch.autograd.grad((ref * g.double()).sum(), leaf)
    ref, y, rest = ref.detach(), y.detach(), rest.detach()
    q = y.exp()
    at = idx.clamp(0, C - 1)
    mass = p.sum(dim=1)
    # every p is off by a few U of itself and of its exponent, log q as log p above; what is left of the mass by K / 2 + 4 steps of the sum
    logs = torch.where(p > 0, p * (torch.where(p > 0, p, 1.0).log().abs() + y.gather(1, at).abs()), 0.0).sum(dim=1)
    l_off = (K / 2 + 8) * U * (1 + mass)
    r_log = torch.where(left > 0, torch.where(left > 0, left, 1.0).log().abs() + rest.nan_to_num(neginf=0.0).abs() + 1, 0.0)
    # the relative error of q_rest / q_listed is that of two sums
    bound = (_r(C) + 16 * U) * (mass + logs + left * (1 + rest.nan_to_num(neginf=0.0).abs())) + (K + 8) * U * logs + l_off * r_log * tail + 8 * U
    _inside(loss, ref, bound, "row_loss")
    target = torch.zeros(R, C, dtype=torch.float64).scatter_add_(1, at, p)
    r = torch.where(listed, 0.0, (y - rest[:, None]).exp().nan_to_num(nan=0.0, posinf=0.0))
    size = q * (mass + left)[:, None] + target + left[:, None] * r
    l_err = (l_off * tail)[:, None] * (q + r) * (left > 0)[:, None]
    gb = g.double().abs()[:, None] / T
    bound = gb * (size * (4 * _r(C) + (K + 16) * U + 8 * U * (y.abs() + 1)) + 2 * l_err + 4 * U * size) + _half_step(grad, dtype) + 1e-37
    _inside(d[:, :C], grad, bound, "dlogits")
    assert not d[:, C:].any()
    # added to what is there, in one rounding; the columns from C on stay
    base = torch.randn(x.shape, generator=_gen(4)).to(dtype).cuda()
    acc = ops.distill_bwd(x, idx.cuda(), t.cuda(), stats, g.cuda(), C=C, temperature=T, tail=tail, dlogits=base.clone(), accumulate=True)
    want = base[:, :C].double().cpu() + grad
    _inside(acc[:, :C], want, bound + _half_step(want, dtype) + 2 * U * want.abs(), "accumulated dlogits")
    assert torch.equal(acc[:, C:], base[:, C:])


@pytest.mark.parametrize("C", [40, 1026, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_special_rows(C, dtype):
    from ttts_amd import ops
    K = 16
    x = _logits(9, C, C, dtype, 2)
    idx, t = _teacher(9, C, K, 1.0, True, 1, empty=0.0)
    x[0] = -math.inf                                       # the student's mask leaves nothing
    x[1] = LOWEST[dtype]                                   # uniform
    idx[2] = -1                                            # no entries: tail mode compares the whole mass with the whole
    x[3] = -math.inf; x[3].scatter_(0, idx[3].cuda(), torch.linspace(-1, 1, K).to(dtype).cuda())   # every class left is named
    x[4, idx[4, 3]] = -math.inf                            # the teacher wants a class that the student forbids
    t[5] = -math.inf; t[5, 2] = 0.0                        # all mass on one class
    x[6, 3] = math.nan
    t[7, 4] = -math.inf
    for tail in (False, True):
        loss, stats = ops.distill_fwd(x, idx.cuda(), t.cuda(), tail=tail)
        d = ops.distill_bwd(x, idx.cuda(), t.cuda(), stats, torch.ones(9, device="cuda"), tail=tail)
        keep = torch.tensor([1, 2, 3, 5, 7, 8])
        leaf = x[keep.cuda()].double().cpu().requires_grad_(True)
        ref, p, listed, left, rest, y = _ref_distill(leaf, idx[keep], t[keep], C, 1.0, tail)
        _inside(loss.cpu()[keep], ref.detach(), 1e-5 * (1 + ref.detach().abs()), "row_loss")   # 1e-5 = 168 U: C / 64 of 40000 is 625 parts, most of them empty lanes' 20
        q = y.detach().exp()
        target = torch.zeros(len(keep), C, dtype=torch.float64).scatter_add_(1, idx[keep].clamp(min=0), p)
        r = torch.where(listed, 0.0, (y.detach() - rest.detach()[:, None]).exp().nan_to_num(0.0))
        grad = q * (p.sum(dim=1) + left)[:, None] - target - left[:, None] * r
        size = q + target + left[:, None] * r
        _inside(d.cpu()[keep], grad, size * 4e-5 + 40 * U + _half_step(grad, dtype), "dlogits")
        assert loss[0].item() == 0.0 and not d[0].any()
        assert loss[4].item() == math.inf and torch.isfinite(d[4]).all()
        assert torch.isnan(loss[6]) and torch.isnan(d[6]).any()
        if not tail:
            assert loss[2].item() == 0.0 and not d[2].any()


def test_gradients_agree_with_differences():
    """(f(x + h v) - f(x - h v)) / 2h of the kernels' own forward against <gradient, v>, |v| <= 1 per class: the cubic term is at most
    h^2 / 6 times a third cumulant (<= 8 / 6^(3/2) < 1) and the sums are good to 2 B / 2h with B the forward's bound."""
    from ttts_amd import ops
    R, C, h, K = 6, 1500, 2.0 ** -5, 24
    x = _logits(R, C, C, torch.float32, 21, std=1.0)
    v = torch.rand(R, C, generator=_gen(3)).cuda() * 2 - 1
    tokens = torch.randint(0, C, (R,), generator=_gen(4)).cuda()
    one = torch.ones(R, device="cuda")
    B = _r(C) * 12 + 4 * U * 12
    tol = B / h + h * h / 6 * 12
    fwd = lambda z: ops.token_logprobs_fwd(z, tokens)  # noqa: E731
    r = fwd(x)
    up, down = fwd(x + h * v), fwd(x - h * v)
    for name, gl, gh in (("logp", one, None), ("entropy", 0 * one, one)):
        d = ops.token_logprobs_bwd(x, tokens, r.stats, r.entropy, gl, gh)
        num = (getattr(up, name) - getattr(down, name)).double() / (2 * h)
        assert ((d.double() * v.double()).sum(dim=1) - num).abs().max().item() <= tol, name
    for tail in (False, True):
        idx, t = (z.cuda() for z in _teacher(R, C, K, 1.0, tail, 5, empty=0.0))
        _, stats = ops.distill_fwd(x, idx, t, tail=tail)
        d = ops.distill_bwd(x, idx, t, stats, one, tail=tail)
        num = (ops.distill_fwd(x + h * v, idx, t, tail=tail)[0] - ops.distill_fwd(x - h * v, idx, t, tail=tail)[0]).double() / (2 * h)
        assert ((d.double() * v.double()).sum(dim=1) - num).abs().max().item() <= tol, tail


def test_no_rows_and_many_rows():
    from ttts_amd import ops
    e = torch.empty(0, 100, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    r = ops.token_logprobs_fwd(e, none, top_k=4)
    assert r.logp.shape == (0,) and r.top_idx.shape == (0, 4)
    assert ops.token_logprobs_bwd(e, none, r.stats, r.entropy, r.logp).shape == (0, 100)
    i, t = torch.empty(0, 3, dtype=torch.int64, device="cuda"), torch.empty(0, 3, device="cuda")
    loss, stats = ops.distill_fwd(e, i, t)
    assert loss.shape == (0,) and ops.distill_bwd(e, i, t, stats, loss).shape == (0, 100)
    # more rows than a 16-bit grid dimension
    R = 70001
    x = _logits(R, 4, 8, torch.float16, 1)
    tok = torch.randint(0, 4, (R,), generator=_gen(2)).cuda()
    r = ops.token_logprobs_fwd(x, tok, C=4, top_k=2)
    logp, ent, tl, ti, _, _ = _ref_logprobs(x, tok, 4, 2, 1.0)
    _inside(r.logp, logp, _r(4) + 4 * U * logp.abs(), "logp")
    assert torch.equal(r.top_idx.cpu(), ti)


def test_offsets_past_32_bits():
    """The last rows of a logits tensor of more than 2^31 elements (two-byte classes: 4.3 GB)."""
    from ttts_amd import ops
    R, C = 2200, 1000003
    x = torch.zeros(R, C, dtype=torch.float16, device="cuda")
    x[-2:] = (torch.randn(2, C, generator=_gen(8)) * 2).half().cuda()
    tokens = torch.zeros(R, dtype=torch.int64, device="cuda"); tokens[-1] = C - 1
    r = ops.token_logprobs_fwd(x, tokens, top_k=3)
    logp, ent, tl, ti, y, _ = _ref_logprobs(x[-2:], tokens[-2:], C, 3, 1.0)
    _inside(r.logp[-2:], logp, _r(C) + 4 * U * logp.abs(), "logp")
    assert torch.equal(r.top_idx[-2:].cpu(), ti)
    assert abs(r.logp[0].item() + math.log(C)) < _r(C) and r.top_idx[0].tolist() == [0, 1, 2]
    d = ops.token_logprobs_bwd(x, tokens, r.stats, r.entropy, torch.ones(R, device="cuda"), dlogits=x)
    ref = -y.exp()
    ref[0, 0] += 1; ref[1, C - 1] += 1
    _inside(d[-2:], ref, y.exp() * (4 * _r(C) + 200 * U) + 4 * U + _half_step(ref, torch.float16), "dlogits")


def test_streams_and_graphs():
    """On a side stream, and captured: every replay, with other work between them, gives what the eager calls give."""
    from ttts_amd import ops
    R, C, K = 40, 40000, 12                                # rows of several segments: the calls that use a workspace
    xs = [_logits(R, C, C, torch.bfloat16, s) for s in range(3)]
    tokens = torch.randint(0, C, (R,), generator=_gen(1)).cuda()
    idx, t = (z.cuda() for z in _teacher(R, C, K, 1.0, True, 5))
    one = torch.ones(R, device="cuda")

    def step(x):
        r = ops.token_logprobs_fwd(x, tokens, top_k=8)
        d = ops.token_logprobs_bwd(x, tokens, r.stats, r.entropy, one, one)
        loss, stats = ops.distill_fwd(x, idx, t, tail=True)
        return list(r) + [d, loss, stats, ops.distill_bwd(x, idx, t, stats, one, tail=True)]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    static = [xs[0].clone(), xs[0].clone()]
    graphs, outs = [], []
    for s in static:                                       # two graphs alive at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s))
        graphs.append(g)
    for n in range(4):
        for j in (0, 1):
            static[j].copy_(xs[(n + j) % 3])
        graphs[0].replay(); graphs[1].replay()
        step(xs[2])
        torch.cuda.synchronize()
        for j in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[j], want[(n + j) % 3])), (n, j)


def test_refusals_on_the_gpu():
    from ttts_amd import ops
    from ttts_amd.lib import TttsError
    x = torch.zeros(4, 16, device="cuda")
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    idx, t = torch.zeros(4, 3, dtype=torch.int64, device="cuda"), torch.zeros(4, 3, device="cuda")
    bad = [lambda: ops.token_logprobs_fwd(x.double(), tok), lambda: ops.token_logprobs_fwd(x, tok[:3]), lambda: ops.token_logprobs_fwd(x, tok.int()),
           lambda: ops.token_logprobs_fwd(x, tok, C=17), lambda: ops.token_logprobs_fwd(x, tok, C=0), lambda: ops.token_logprobs_fwd(x, tok, top_k=65),
           lambda: ops.token_logprobs_fwd(x, tok, top_k=-1), lambda: ops.token_logprobs_fwd(x, tok, temperature=0.0),
           lambda: ops.token_logprobs_fwd(x, tok, temperature=math.nan), lambda: ops.token_logprobs_fwd(x.t(), tok),
           lambda: ops.token_logprobs_fwd(x[:1].expand(4, 16), tok), lambda: ops.token_logprobs_fwd(x, tok.cpu()), lambda: ops.token_logprobs_fwd(x.cpu(), tok),
           lambda: ops.distill_fwd(x, idx, t[:, :2]), lambda: ops.distill_fwd(x, idx, t.double()), lambda: ops.distill_fwd(x, idx[:, 0], t),
           lambda: ops.distill_fwd(x, torch.zeros(4, 129, dtype=torch.int64, device="cuda"), torch.zeros(4, 129, device="cuda")),
           lambda: ops.distill_fwd(x, idx[:, :0], t[:, :0]), lambda: ops.distill_fwd(x, idx, t, temperature=-1.0)]
    s2, s3, v = torch.zeros(4, 2, device="cuda"), torch.zeros(4, 3, device="cuda"), torch.zeros(4, device="cuda")
    bad += [lambda: ops.token_logprobs_bwd(x, tok, s3, v, v), lambda: ops.token_logprobs_bwd(x, tok, s2, v, v[:2]),
            lambda: ops.token_logprobs_bwd(x, tok, s2, v, v, dlogits=x.half()), lambda: ops.token_logprobs_bwd(x, tok, s2, v, v, dlogits=x[:, :8]),
            lambda: ops.distill_bwd(x, idx, t, s2, v), lambda: ops.distill_bwd(x, idx, t, s3, v, accumulate=True),
            lambda: ops.distill_bwd(x, idx, t, s3, v, accumulate=True, dlogits=x)]
    for n, f in enumerate(bad):
        with pytest.raises(TttsError):
            f()
            pytest.fail("refusal %d did not come" % n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [40, 1026, 8200, 40000])
def test_distill_rows_with_nan_and_no_entries(C, dtype):
    """With the mass that the list leaves out, a row without entries compares all of it: NaN or +inf among its classes shows in its loss."""
    from ttts_amd import ops
    x = _logits(4, C, C, dtype, 5)
    x[1, C // 2], x[2, C - 1] = math.nan, math.inf
    idx, t = torch.full((4, 3), -1).cuda(), torch.zeros(4, 3).cuda()
    loss, stats = ops.distill_fwd(x, idx, t, tail=True)
    d = ops.distill_bwd(x, idx, t, stats, torch.ones(4, device="cuda"), tail=True)
    for r in (1, 2):
        assert torch.isnan(loss[r]) and torch.isnan(d[r]).any(), r
    for r in (0, 3):                                      # the whole mass on all classes: log 1 - log 1
        assert loss[r].abs().item() <= 4 * U and d[r].float().abs().max().item() <= 4 * _r(C), r


GAPS = [20.0, 23.0, 60.0, 80.0, 87.0, 90.0, 105.0, 200.0, 1000.0, -90.0, -1000.0]


def _apart(x, idx, C, T, dtype):
    """Rows of x changed in place so that the named classes lie by GAPS (in logits / T) above the others, and then: a finite mask over the others, the
    lowest value over the others, over all but one of them, and over all but a few others of which some are at -inf."""
    n = len(GAPS)
    for r in range(len(x)):
        named = idx[r][(idx[r] >= 0) & (idx[r] < C)].unique()
        rest = torch.ones(C, dtype=torch.bool)
        rest[named] = False
        if not rest.any():
            continue
        if r < n:
            x[r, :C] = (x[r, :C].float() / 6 * min(T, 1.0)).to(dtype)
            x[r, named] = (x[r, named].float() + GAPS[r] * T).to(dtype)
        else:
            x[r, :C][rest.cuda()] = -1e4 if r == n else LOWEST[dtype]
            if r == n + 2:
                x[r, int(rest.nonzero()[0])] = 1.0
            if r == n + 3:
                x[r, int(rest.nonzero()[-1])] = -math.inf
                x[r, int(rest.nonzero()[len(rest.nonzero()) // 2])] = -math.inf


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C,offset", [(9, 0), (1026, 0), (2000, 1), (2049, 0), (8195, 1), (20000, 0), (40001, 0), (300007, 1)])
@pytest.mark.parametrize("K,T", [(1, 1.0), (5, 0.1), (64, 1.0), (100, 2.0)])
def test_distill_where_named_and_other_classes_lie_far_apart(C, offset, dtype, K, T):
    """The mass that the list leaves out is compared with the other classes' however far they lie below the named ones (or above): their
    maximum and sum are their own.  The named classes' log-sum-exp b is one fp32 number where they lie far above: their share is off
    by the rounding of b / T."""
    from ttts_amd import ops
    R = len(GAPS) + 4
    x = _logits(R, C, C + offset, dtype, C + K, offset)
    idx, t = _teacher(R, C, K, T, True, C + 3 * K, empty=0.1 if K > 1 else 0.0, repeat=K > 4)
    if K == 1:
        t = torch.log(torch.linspace(0.05, 0.95, R)).view(R, 1)
    _apart(x, idx, C, T, dtype)
    g = torch.randn(R, generator=_gen(9))
    loss, stats = ops.distill_fwd(x, idx.cuda(), t.cuda(), C=C, temperature=T, tail=True)
    d = ops.distill_bwd(x, idx.cuda(), t.cuda(), stats, g.cuda(), C=C, temperature=T, tail=True)
    there = (idx >= 0) & (idx < C)
    at = idx.clamp(0, C - 1)
    z = x[:, :C].double().cpu() / T
    named = torch.zeros(R, C, dtype=torch.float64).scatter_add_(1, at, there.double()) > 0
    lp = torch.where(there, t, 0.0).double()
    p = torch.where(there, lp.exp(), 0.0)
    mass = p.sum(dim=1)
    left = (1 - mass).clamp(min=0)
    zr = z.masked_fill(named, -math.inf)
    top = z.amax(dim=1, keepdim=True)
    logz = (z - top).exp().sum(dim=1, keepdim=True).log()
    held = (zr > -math.inf).any(dim=1) & (left > 0)
    left = torch.where(held, left, 0.0)
    top_r = zr.amax(dim=1, keepdim=True).clamp(min=-1e300)
    logz_r = (zr - top_r).exp().sum(dim=1, keepdim=True).log()
    y = z - top - logz
    log_r = torch.where(zr > -math.inf, zr - top_r - logz_r, -math.inf)
    rest = torch.where(held, (top_r - top + logz_r - logz)[:, 0], 0.0)      # log of the student's share of the others
    terms = torch.where(p > 0, p * (lp - y.gather(1, at)), 0.0)
    safe = torch.where(held, left, 1.0)
    ref = terms.sum(dim=1) + left * (safe.log() - rest)
    logs = torch.where(p > 0, p * (lp.abs() + y.gather(1, at).abs()), 0.0).sum(dim=1)
    l_off = (K / 2 + 8) * U * (1 + mass)
    bound = (_r(C) + 16 * U) * (mass + logs + left * (1 + rest.abs())) + (K + 8) * U * logs + l_off * (safe.log().abs() + rest.abs() + 1) + 8 * U
    _inside(loss, ref.float().double(), bound, "row_loss")
    q, r = y.exp(), log_r.exp()
    target = torch.zeros(R, C, dtype=torch.float64).scatter_add_(1, at, p)
    grad = (q * (mass + left)[:, None] - target - left[:, None] * r) * (g.double() / T)[:, None]
    # exponents: of a named class |log q| and, far above the others, b / T (rounded once, and once more taken off); of another |log r| and the
    # distance that still counts as near (32 bits: 22.2)
    b = z.masked_fill(~named, -math.inf).amax(dim=1, keepdim=True).clamp(min=-1e300).abs() + 8
    far = ((top - top_r) > 22)
    span = torch.where(named, y.abs() + torch.where(far, b, 0.0), torch.minimum(log_r.abs() + 23, y.abs() + 23)).nan_to_num(posinf=0.0)
    size = q * (mass + left)[:, None] + target + left[:, None] * r
    err = (l_off * held)[:, None] * (q + r)
    gb = g.double().abs()[:, None] / T
    bound = gb * (size * (4 * _r(C) + (K + 16) * U + 8 * U * (span + 1)) + 2 * err) + _half_step(grad, dtype) + 1e-37
    _inside(d[:, :C], grad, bound, "dlogits")
    base = torch.randn(x.shape, generator=_gen(4)).to(dtype).cuda()
    acc = ops.distill_bwd(x, idx.cuda(), t.cuda(), stats, g.cuda(), C=C, temperature=T, tail=True, dlogits=base.clone(), accumulate=True)
    want = base[:, :C].double().cpu() + grad
    _inside(acc[:, :C], want, bound + _half_step(want, dtype) + 2 * U * want.abs(), "accumulated dlogits")
    assert ops.distill_bwd(x, idx.cuda(), t.cuda(), stats, g.cuda(), C=C, temperature=T, tail=True, dlogits=x) is x and torch.equal(x[:, :C], d[:, :C])


@pytest.mark.parametrize("gap", [30.0, 100.0, 500.0])
def test_distill_gradient_far_apart_agrees_with_differences(gap):
    """As test_gradients_agree_with_differences, the named classes `gap` above the others: the forward's error grows with the loss, left * gap."""
    from ttts_amd import ops
    R, C, h, K = 6, 1500, 2.0 ** -5, 8
    x = _logits(R, C, C, torch.float32, 22, std=1.0)
    idx, t = _teacher(R, C, K, 1.0, True, 6, empty=0.0)
    for r in range(R):
        x[r, idx[r]] += gap
    v = torch.rand(R, C, generator=_gen(3)).cuda() * 2 - 1
    idx, t = idx.cuda(), t.cuda()
    f = lambda z: ops.distill_fwd(z, idx, t, tail=True)[0].double()  # noqa: E731
    _, stats = ops.distill_fwd(x, idx, t, tail=True)
    d = ops.distill_bwd(x, idx, t, stats, torch.ones(R, device="cuda"), tail=True)
    num = (f(x + h * v) - f(x - h * v)) / (2 * h)
    B = (_r(C) + (K + 24) * U) * (gap + 12)
    # x +- h v are rounded: each class by U (gap + 8), which moves the loss by at most that much twice over
    assert ((d.double() * v.double()).sum(dim=1) - num).abs().max().item() <= (B + 2 * U * (gap + 8)) / h + h * h / 6 * 12


@pytest.mark.parametrize("T", [4.3e-39, 1.5e-38, 3.0e38])
def test_temperatures_at_the_ends_of_the_range(T):
    """The least temperature makes the best class certain (ties share), the largest makes all alike."""
    from ttts_amd import ops
    x = _logits(4, 700, 700, torch.float32, 31)
    best = x.argmax(dim=1)
    x[3, (best[3] + 1) % 700] = x[3, best[3]]
    r = ops.token_logprobs_fwd(x, best, top_k=2, temperature=T)
    want = [0.0, 0.0, 0.0, math.log(2.0)] if T < 1 else [math.log(700.0)] * 4
    for n in range(4):
        assert abs(r.logp[n].item() + want[n]) <= 4 * _r(700) and abs(r.entropy[n].item() - want[n]) <= 24 * _r(700), n
    loss, _ = ops.distill_fwd(x, best[:, None].contiguous(), torch.zeros(4, 1, device="cuda"), temperature=T)
    assert (loss.cpu().double() - torch.tensor(want, dtype=torch.float64)).abs().max().item() <= 4 * _r(700)


@pytest.mark.parametrize("dtype,C,used", [(torch.float32, 8256, False), (torch.float32, 8257, False), (torch.float32, 20000, False), (torch.float32, 32832, False),
                                          (torch.float32, 32833, True), (torch.bfloat16, 8256, False), (torch.bfloat16, 8257, True)])
def test_scratch_is_taken_where_it_is_used(dtype, C, used, monkeypatch):
    """Rows that one workgroup ends take none, and the C entries do not ask for any there."""
    from ttts_amd import lib as l
    from ttts_amd import ops
    taken = []
    real = ops._workspace
    monkeypatch.setattr(ops, "_workspace", lambda n, like: (taken.append(n), real(n, like))[1])
    x = _logits(3, C, C, dtype, 8)
    tokens = torch.tensor([0, C - 1, -1]).cuda()
    idx, t = (z.cuda() for z in _teacher(3, C, 7, 1.0, True, 3))
    r = ops.token_logprobs_fwd(x, tokens, top_k=9)
    loss, stats = ops.distill_fwd(x, idx, t, tail=True)
    assert len(taken) == (2 if used else 0)
    logp, _, tl, ti, _, _ = _ref_logprobs(x, tokens, C, 9, 1.0)
    assert torch.equal(r.top_idx.cpu(), ti)
    _inside(r.logp, logp, _r(C) + 4 * U * logp.abs(), "logp")
    outs = [torch.empty_like(z) for z in (r.logp, r.entropy, r.stats, r.top_logp, r.top_idx, loss, stats)]
    p = [z.data_ptr() for z in outs]
    code = l.DTYPE_F32 if dtype == torch.float32 else l.DTYPE_BF16
    stream = torch.cuda.current_stream().cuda_stream
    rc = [l.get().ttts_token_logprobs_fwd(x.data_ptr(), code, C, tokens.data_ptr(), p[0], p[1], p[2], p[3], p[4], 3, C, 9, 1.0, None, 0, stream),
          l.get().ttts_distill_fwd(x.data_ptr(), code, C, idx.data_ptr(), t.data_ptr(), p[5], p[6], 3, C, 7, 1.0, 1, None, 0, stream)]
    if used:
        assert rc == [-1, -1] and "workspace" in l.get().ttts_last_error().decode()
    else:
        assert rc == [0, 0]
        for a, b in zip(outs, (r.logp, r.entropy, r.stats, r.top_logp, r.top_idx, loss, stats)):
            assert torch.equal(a, b)


def test_distill_lowest_values_at_a_temperature_of_their_size():
    """Named classes at the lowest fp32 value, a temperature of 1e38 .. 3e38: they are e^-1 .. e^-4 of the others, not nothing."""
    from ttts_amd import ops
    x = _logits(3, 900, 900, torch.float32, 41)
    idx = torch.tensor([[3, 500], [800, 801], [0, 899]])
    for r in range(3):
        x[r, idx[r]] = torch.finfo(torch.float32).min
    t = torch.log(torch.tensor([[0.2, 0.3], [0.5, 0.1], [0.05, 0.6]]))
    for T in (1e38, 3e38):
        loss, stats = ops.distill_fwd(x, idx.cuda(), t.cuda(), temperature=T, tail=True)
        ref = _ref_distill(x.double().cpu(), idx, t, 900, T, True)[0]
        assert (loss.cpu().double() - ref).abs().max().item() <= 12 * _r(900), T


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("C,offset", [(2, 0), (40, 1), (1026, 0), (1088, 0), (2112, 0), (5000, 1), (9152, 0), (20000, 0), (40001, 1), (150000, 0)])
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_nearly_certain_classes_keep_their_bits(C, offset, dtype, T):
    """The best class 5 to 60 nats ahead of the others: its log-probability, -log(1 + the others), and the entropy are good to a few steps
    of THEMSELVES.  A term of the others is off by its exponent's roundings, 6 U of its distance and a few U; two best classes, and
    four, share the rest."""
    from ttts_amd import ops
    gaps = [5.0, 7.0, 10.0, 14.0, 20.0, 40.0, 60.0]
    R = 2 * len(gaps)
    x = (_logits(R, C, C + offset, dtype, C, offset, std=0.5).float() * T).to(dtype)
    best = torch.randint(0, C, (R,), generator=_gen(7))
    for r in range(R):
        x[r, best[r]] = x[r, :C].float().max().item() + (gaps[r % len(gaps)] + math.log(C)) * T
        if r >= len(gaps):
            for n in range(1, 2 if r % 2 else 4):
                x[r, (best[r] + n * (C // 4 + 1)) % C] = x[r, best[r]]
    r = ops.token_logprobs_fwd(x, best.cuda(), C=C, top_k=3, temperature=T)
    z = x[:, :C].double().cpu() / T
    d = z - z.amax(dim=1, keepdim=True)
    ties = (d == 0).sum(dim=1)
    rest = torch.where(d == 0, 0.0, d.exp()).sum(dim=1)
    logz = torch.where(ties == 1, torch.log1p(rest), torch.log(ties + rest))
    ent = logz - (d * d.exp()).sum(dim=1) / d.exp().sum(dim=1)
    far = torch.where(d == 0, 0.0, d.abs()).amax(dim=1)
    bound = (_r(C) + (6 * far + 20) * U)
    _inside(r.logp, -logz, bound * logz, "logp")
    _inside(r.entropy, ent, 2 * bound * ent, "entropy")
    _inside(r.stats[:, 1], logz, bound * logz, "log Z")
    first = torch.sort(z, dim=1, descending=True, stable=True)
    assert torch.equal(r.top_idx[:, :min(3, C)].cpu(), first.indices[:, :3])
    _inside(r.top_logp[:, 0], -logz, bound * logz, "top_logp")
