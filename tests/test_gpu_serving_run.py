"""The paged cache, its attention, the scoring and the distillation in one run, as they are used: a teacher decodes a ragged batch
over a paged cache and reports each token's alternatives, a student learns from them -- against the same run in 64 bits; and the
GPT's own path: UnifiedVoice.score of one model as the teacher of another's train step."""
import json
import math
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
GOLD = os.path.join(os.path.dirname(__file__), "golden")
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def test_decode_score_distill():
    from ttts_amd import ops
    M, H, Hkv, dh, page, C, K, steps = 5, 4, 2, 64, 16, 1026, 12, 20
    g = _gen(1)
    lens0 = [37, 0, 15, 64, 300]                            # prompts of any length, one place without a prompt
    width = -(-(max(lens0) + steps) // page)
    P = M * width
    table = torch.randperm(P, generator=g).view(M, width)
    kp = torch.full((P, Hkv, page, dh), math.nan, dtype=torch.bfloat16, device="cuda")   # nothing but written rows may be read
    vp = kp.clone()
    bf = lambda t: t.to(torch.bfloat16)  # noqa: E731
    prompt = [bf(torch.randn(n, (H + 2 * Hkv) * dh, generator=g)) for n in lens0]
    new = bf(torch.randn(steps, M, (H + 2 * Hkv) * dh, generator=g))
    head = bf(torch.randn(C, H * dh, generator=g) / 8)
    student = bf(torch.randn(steps * M, C, generator=g) * 2)

    def slots(m, lo, hi):
        pos = torch.arange(lo, hi)
        return table[m, pos // page] * page + pos % page
    # the prompts of all sequences in one padded call
    longest = max(lens0)
    rows = torch.zeros(M, longest, (H + 2 * Hkv) * dh, dtype=torch.bfloat16)
    at = torch.full((M, longest), -1)
    for m, n in enumerate(lens0):
        rows[m, :n] = prompt[m]
        at[m, :n] = slots(m, 0, n)
    packed = rows.view(M * longest, -1).cuda()
    kv = lambda t: (t[:, H * dh:(H + Hkv) * dh].view(-1, Hkv, dh), t[:, (H + Hkv) * dh:].view(-1, Hkv, dh))  # noqa: E731
    ops.kv_page_write(*kv(packed), kp, vp, at.view(-1).cuda())
    block = table.to(torch.int32).cuda()
    head_c = head.cuda()
    att, logits_all, idx_all, logp_all, tokens_all, got = [], [], [], [], [], []
    for t in range(steps):
        x = new[t].cuda()
        pos = torch.tensor(lens0) + t
        slot = table[torch.arange(M), pos // page] * page + pos % page
        ops.kv_page_write(*kv(x), kp, vp, slot.cuda())
        o, _ = ops.attn_paged_decode(x[:, :H * dh].view(M, H, dh), kp, vp, block, (pos + 1).to(torch.int32).cuda(), dh ** -0.5)
        logits = o.reshape(M, H * dh).float() @ head_c.float().t()
        tokens = logits.argmax(dim=1)
        r = ops.token_logprobs_fwd(logits, tokens, top_k=K, temperature=2.0)
        att.append(o); logits_all.append(logits); idx_all.append(r.top_idx); logp_all.append(r.top_logp); tokens_all.append(tokens); got.append(r)
    idx, logp = torch.cat(idx_all), torch.cat(logp_all)
    s = student.cuda()
    loss, stats = ops.distill_fwd(s, idx, logp, temperature=2.0, tail=True)
    g_loss = torch.full((steps * M,), 1.0 / (steps * M), device="cuda")
    grad = ops.distill_bwd(s, idx, logp, stats, g_loss, temperature=2.0, tail=True)
    # the attention of every step in 64 bits: within one rounding of the weights and one of the result (2^-8 each) of sum p |v|
    for t in range(steps):
        for m in range(M):
            seq = torch.cat([prompt[m], new[:t + 1, m]]).double()
            k, v = seq[:, H * dh:(H + Hkv) * dh].view(-1, Hkv, dh), seq[:, (H + Hkv) * dh:].view(-1, Hkv, dh)
            for h in range(H):
                p = torch.softmax(k[:, h // 2] @ new[t, m, h * dh:(h + 1) * dh].double() * dh ** -0.5, dim=0)
                ref, mag = p @ v[:, h // 2], p @ v[:, h // 2].abs()
                off = (att[t][m, h].double().cpu() - ref).abs() - 2.0 ** -8 * (mag + ref.abs()) * 1.02 - 1e-5
                assert off.max().item() <= 0, (t, m, h, off.max().item())
    # from the logits on in 64 bits
    teacher = torch.cat(logits_all).double().cpu() / 2.0
    lp = torch.log_softmax(teacher, dim=1)
    want, order = torch.sort(teacher, dim=1, descending=True, stable=True)
    assert torch.equal(idx.cpu(), order[:, :K])
    assert (logp.double().cpu() - lp.gather(1, order[:, :K])).abs().max().item() <= (C / 64 + 32) * U + 4 * U * 20
    tok = torch.cat(tokens_all).cpu()
    assert torch.equal(tok, idx[:, 0].cpu())
    assert torch.equal(torch.cat([r.logp for r in got]), logp[:, 0])     # the token is its own first alternative
    leaf = student.double().requires_grad_(True)
    y = torch.log_softmax(leaf / 2.0, dim=1)
    p = logp.double().cpu().exp()
    left = 1 - p.sum(dim=1)
    listed = torch.zeros_like(y, dtype=torch.bool).scatter_(1, idx.cpu(), True)
    rest = torch.logsumexp(y.masked_fill(listed, -math.inf), dim=1)
    ref = (p * (p.log() - y.gather(1, idx.cpu()))).sum(dim=1) + left * (left.log() - rest)
    ref.mean().backward()
    # 100 U: the classes' sums (C / 64 + 32 of them), the terms' own roundings, K of the mass; the loss' terms add up to under 10
    assert (loss.double().cpu() - ref.detach()).abs().max().item() <= 100 * U * 10
    size = (y.detach().exp() + torch.zeros_like(y).scatter_(1, idx.cpu(), p) + left[:, None] * (y.detach() - rest.detach()[:, None]).exp()) / (2.0 * steps * M)
    off = (grad.double().cpu() - leaf.grad).abs() - 2.0 ** -8 * leaf.grad.abs() - 400 * U * size - 1e-38
    assert off.max().item() <= 0, off.max().item()


def _models():
    from oracle import gpt_ref
    import ttts_amd.gpt as gpt
    cfg = json.loads(str(np.load(os.path.join(GOLD, "gpt_infer.npz"))["cfg_json"]))
    models = []
    for scale in (0.05, 0.02):
        m = gpt.UnifiedVoice(**cfg, device="cuda:0", dropout_p=0.0)
        m.load_state_dict(gpt_ref.det_state_dict(cfg, scale))
        models.append(m)
    batch = gpt_ref.synthetic_batch(B=2, text_len=9, mel_len=14, seed=5, cfg=cfg)
    return cfg, models, [batch[0].cuda(), batch[1], batch[2].cuda(), batch[3]]


def test_gpt_score_and_teacher():
    """score() is the model's own logits, scored; a train step with its alternatives as the teacher has the two losses' gradient."""
    from ttts_amd.gpt.model import prepare_tokens
    from ttts_amd.lib import TttsError
    cfg, (teacher, student), batch = _models()
    K = 10
    r = teacher.score(*batch, top_k=K)
    _, _, logits = teacher(*batch)
    tokens = prepare_tokens(teacher.cfg, *batch)
    x = logits.detach().permute(0, 2, 1).double().cpu()              # (B, Tm, classes)
    y = torch.log_softmax(x, dim=2)
    C = y.shape[2]
    tar = tokens[3].cpu()
    assert r.logp.shape == tar.shape and r.top_idx.shape == tar.shape + (K,)
    assert (r.logp.double().cpu() - y.gather(2, tar[..., None])[..., 0]).abs().max().item() <= (C / 64 + 32) * U + 80 * U
    assert torch.equal(r.top_idx.cpu(), torch.sort(x, dim=2, descending=True, stable=True).indices[..., :K])
    assert teacher.engine.training                                   # as it was
    eng = student.engine
    dev_tokens = [t.cuda() for t in tokens]
    w, w_mel = 0.7, 0.9
    eng.set_tokens(*dev_tokens)
    eng.forward()
    eng.set_teacher(r.top_idx, r.top_logp, weight=w)
    eng.zero_grad()
    eng.backward(0.0, w_mel)
    B, _, Tm = eng._bufs_key
    rows = B * Tm
    leaf = eng.b["logits_m"][:, :eng.nm].double().cpu().requires_grad_(True)
    ys = torch.log_softmax(leaf, dim=1)
    idx, lp = r.top_idx.view(rows, K).cpu(), r.top_logp.view(rows, K).double().cpu()
    p = lp.exp()
    left = (1 - p.sum(dim=1)).clamp(min=0)
    rest = torch.logsumexp(ys.scatter(1, idx, -math.inf), dim=1)
    kl = ((p * (lp - ys.gather(1, idx))).sum(dim=1) + left * (left.log() - rest)).mean()
    ce = -ys.gather(1, dev_tokens[3].view(-1, 1).cpu()).mean()
    (w_mel * ce + w * kl).backward()
    assert abs(eng.distill_loss.item() - kl.item()) <= 1e-5 * (1 + abs(kl.item()))
    # the cross-entropy's gradient is rounded to bf16, the sum again: 2^-8 of each; the exponentials' own error is below that by far
    ce_part = (ys.detach().exp() - torch.nn.functional.one_hot(dev_tokens[3].view(-1).cpu(), eng.nm)) * w_mel / rows
    off = (eng.b["dlog_m"][:, :eng.nm].double().cpu() - leaf.grad).abs() - 2.0 ** -8 * (leaf.grad.abs() + ce_part.abs()) - 1e-6 / rows
    assert off.max().item() <= 0, off.max().item()
    # a whole step runs, and without a teacher it is what it was
    eng.zero_grad()
    eng.train_step(dev_tokens, w_mel=w_mel, teacher=dict(teacher_idx=r.top_idx, teacher_logp=r.top_logp, weight=w))
    assert torch.isfinite(eng.params).all()
    eng.train_step(dev_tokens, w_mel=w_mel)
    assert eng._teacher is None
    with pytest.raises(TttsError):
        eng.train_step(dev_tokens, capture=True, teacher=dict(teacher_idx=r.top_idx, teacher_logp=r.top_logp))
    with pytest.raises(TttsError):
        eng.set_teacher(r.top_idx[:, :-1], r.top_logp[:, :-1])


def test_teacher_arguments_are_checked_before_the_step():
    from ttts_amd.gpt.model import prepare_tokens
    from ttts_amd.lib import TttsError
    cfg, (teacher, student), batch = _models()
    r = teacher.score(*batch, top_k=5)
    eng = student.engine
    tokens = [t.cuda() for t in prepare_tokens(teacher.cfg, *batch)]
    before = eng.params.clone()
    wide = r.top_idx.repeat(1, 1, 26)
    for bad in (dict(teacher_idx=r.top_idx.int(), teacher_logp=r.top_logp), dict(teacher_idx=r.top_idx, teacher_logp=r.top_logp.double()),
                dict(teacher_idx=r.top_idx.cpu(), teacher_logp=r.top_logp.cpu()), dict(teacher_idx=r.top_idx[..., :0], teacher_logp=r.top_logp[..., :0]),
                dict(teacher_idx=wide, teacher_logp=r.top_logp.repeat(1, 1, 26)), dict(teacher_idx=r.top_idx),
                dict(teacher_idx=r.top_idx, teacher_logp=r.top_logp, temperature=0.0)):
        with pytest.raises(TttsError):
            eng.train_step(tokens, teacher=bad)
        assert eng._teacher is None and torch.equal(eng.params, before) and not eng.grads.any()
    eng.train_step(tokens, teacher=dict(teacher_idx=r.top_idx, teacher_logp=r.top_logp))
    assert math.isfinite(eng.distill_loss.item())
    eng.train_step(tokens)
    assert eng.distill_loss is None                      # no loss of an earlier step's teacher


@pytest.mark.parametrize("temperature", [1e-39, 4.2e-39, 3.2e38, math.nan])
def test_teacher_temperatures_are_checked_before_the_step(temperature):
    """A temperature that the distillation refuses is refused with the tokens, not in the middle of the backward."""
    from ttts_amd.gpt.model import prepare_tokens
    from ttts_amd.lib import TttsError
    cfg, (teacher, student), batch = _models()
    r = teacher.score(*batch, top_k=5)
    eng = student.engine
    before = eng.params.clone()
    with pytest.raises(TttsError, match="set_teacher"):
        eng.train_step([t.cuda() for t in prepare_tokens(teacher.cfg, *batch)],
                       teacher=dict(teacher_idx=r.top_idx, teacher_logp=r.top_logp, temperature=temperature))
    assert eng._teacher is None and torch.equal(eng.params, before) and not eng.grads.any()
