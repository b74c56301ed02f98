"""Measured cases of the serving and distillation operators: the paged key / value cache with the attention of one new token
that reads it, the log-probabilities of given tokens with entropy and alternatives, and the distillation loss on such
alternatives.  `own` False: the operators in elementary torch operations; True: the calls of `ttts_amd.ops`."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ---- cases --------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the new tokens of a decode step enter the cache: 8 sequences of the GPT of this repository (8 heads of 64)
        {"name": "write-step", "op": "write", "rows": 8, "heads": 8, "dh": 64, "page": 16, "pads": 0, "dtype": "bf16"},
        # a padded batch of prompts enters the cache of a wider model in one call; the padding rows have no slot
        {"name": "write-prompts", "op": "write", "rows": 30011, "heads": 8, "dh": 128, "page": 64, "pads": 1717, "dtype": "f16"},
        # one sequence of the GPT of this repository, in the middle of its speech: latency
        {"name": "attend-one", "op": "attend", "seqs": 1, "heads": 8, "kv_heads": 8, "dh": 64, "page": 16, "longest": 613,
         "shortest": 613, "len_seed": 1, "dtype": "bf16"},
        # a served batch of that GPT at every stage, up to its 802 text and 1602 speech positions
        {"name": "attend-batch", "op": "attend", "seqs": 64, "heads": 8, "kv_heads": 8, "dh": 64, "page": 16, "longest": 2404,
         "shortest": 3, "len_seed": 2, "dtype": "bf16"},
        # few long documents, heads shared eight to one
        {"name": "attend-long", "op": "attend", "seqs": 4, "heads": 32, "kv_heads": 4, "dh": 128, "page": 64, "longest": 131071,
         "shortest": 90001, "len_seed": 3, "dtype": "f16"},
        # a large ragged batch with empty places in it, heads shared five to one
        {"name": "attend-ragged", "op": "attend", "seqs": 96, "heads": 40, "kv_heads": 8, "dh": 128, "page": 32, "longest": 4096,
         "shortest": 0, "len_seed": 4, "dtype": "bf16"},
        # what a decode step of this repository's GPT answers beside its tokens: fp32 logits in rows of 1088
        {"name": "logprob-step", "op": "logprob", "rows": 8, "classes": 1026, "pitch": 1088, "top": 5, "train": False,
         "temperature": 1.0, "masked": False, "dtype": "f32"},
        # scoring a training batch of it (8 x 1602 positions) with the alternatives that a student learns from
        {"name": "logprob-score", "op": "logprob", "rows": 12816, "classes": 1026, "pitch": 1088, "top": 20, "train": False,
         "temperature": 1.0, "masked": False, "dtype": "bf16"},
        # scoring with a large text vocabulary, part of it masked out, and many alternatives
        {"name": "logprob-vocabulary", "op": "logprob", "rows": 2048, "classes": 100003, "pitch": 100008, "top": 64, "train": False,
         "temperature": 1.0, "masked": True, "dtype": "bf16"},
        # a policy-gradient step with an entropy bonus: forward and gradient
        {"name": "logprob-train", "op": "logprob", "rows": 4096, "classes": 8194, "pitch": 8256, "top": 0, "train": True,
         "temperature": 0.7, "masked": False, "dtype": "f32"},
        # the GPT of this repository as a student: forward and gradient on 20 alternatives a position
        {"name": "distill-gpt", "op": "distill", "rows": 12816, "classes": 1026, "pitch": 1088, "top": 20, "tail": False,
         "temperature": 1.0, "dtype": "bf16"},
        # a large vocabulary in unpadded rows of odd length, softened, with the mass that the teacher's list leaves out
        {"name": "distill-vocabulary", "op": "distill", "rows": 2048, "classes": 50257, "pitch": 50257, "top": 64, "tail": True,
         "temperature": 2.0, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "logprob", "logprob", "distill"])
    if op == "write":
        rows, heads, dh = _log_int(rng, 1, 30000), rng.choice([1, 2, 3, 8]), rng.choice([32, 64, 128])
        return {"op": op, "rows": rows, "heads": heads, "dh": dh, "page": rng.choice([16, 32, 64, 128]),
                "pads": rng.randrange(0, rows // 8 + 1), "dtype": rng.choice(["bf16", "f16"])}
    if op == "attend":
        kv_heads, dh = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 128])
        seqs = _log_int(rng, 1, 160)
        longest = _log_int(rng, 1, min(100000, 2 ** 28 // (seqs * kv_heads * dh)))
        return {"op": op, "seqs": seqs, "heads": kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 8, 16]), "kv_heads": kv_heads, "dh": dh,
                "page": rng.choice([16, 32, 64, 128]), "longest": longest, "shortest": rng.randrange(0, longest + 1),
                "len_seed": rng.randrange(1 << 20), "dtype": rng.choice(["bf16", "f16"])}
    rows = _log_int(rng, 1, 14000)
    classes = _log_int(rng, 2, min(100000, 10 ** 8 // rows))
    case = {"op": op, "rows": rows, "classes": classes, "pitch": rng.choice([classes, -(-classes // 8) * 8, -(-classes // 64) * 64]),
            "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]), "dtype": rng.choice(["bf16", "f16", "f32"])}
    if op == "logprob":
        case.update(top=rng.choice([0, 1, 5, 20, 64]), train=rng.random() < 0.4, masked=rng.random() < 0.3)
    else:
        case.update(top=rng.randrange(1, min(classes, 64) + 1), tail=rng.random() < 0.5)
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """The sequences' lengths: part of the case, not of the seed.  The first is the longest; every 16th place is empty where the
    range begins at zero."""
    r = random.Random(case["len_seed"])
    lens = [r.randint(case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    lens[0] = case["longest"]
    if case["shortest"] == 0:
        lens = [0 if i % 16 == 7 else n for i, n in enumerate(lens)]
    return lens


def _normal(g, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _logits(case, g, std):
    """Rows of `pitch` columns, the first `classes` of which count; a few classes of each row stand out, as a trained model's do."""
    dt = DTYPES[case["dtype"]]
    x = _normal(g, (case["rows"], case["pitch"]), dt, std)
    n, C = min(3, case["classes"]), case["classes"]
    first = torch.randint(0, C, (case["rows"], 1), generator=g, device="cuda")
    peaks = (first + torch.arange(n, device="cuda") * (C // n)) % C            # n different classes of the row
    x.scatter_(1, peaks, _normal(g, (case["rows"], n), torch.float32, 2.0).add_(4.0 * std).to(dt))
    x[:, case["classes"]:] = 30.0
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "write":
        N, H, dh, page = case["rows"], case["heads"], case["dh"], case["page"]
        pages = -(-N // page) + 5
        packed = _normal(g, (N, 3 * H, dh), dt)                     # query, key and value heads of a token side by side
        s["k"], s["v"] = packed[:, H:2 * H], packed[:, 2 * H:]
        s["k_pages"], s["v_pages"] = _normal(g, (pages, H, page, dh), dt), _normal(g, (pages, H, page, dh), dt)
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:N]
        slots[torch.randperm(N, generator=g, device="cuda")[:case["pads"]]] = -1
        s["slots"] = slots
    elif case["op"] == "attend":
        M, H, Hkv, dh, page = (case[k] for k in ("seqs", "heads", "kv_heads", "dh", "page"))
        lens = _lengths(case)
        per = [-(-n // page) for n in lens]
        width, pages = max(1, max(per)), sum(per) + 3
        s["k_pages"], s["v_pages"] = _normal(g, (pages, Hkv, page, dh), dt), _normal(g, (pages, Hkv, page, dh), dt)
        s["q"] = _normal(g, (M, H, dh), dt, 1.5)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        held = torch.tensor(per, device="cuda")
        at = torch.arange(width, device="cuda")[None, :] + (held.cumsum(0) - held)[:, None]
        inside = torch.arange(width, device="cuda")[None, :] < held[:, None]
        s["block_table"] = torch.where(inside, order[at.clamp(max=pages - 1)], 0).to(torch.int32).contiguous()
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    else:
        R, C = case["rows"], case["classes"]
        s["logits"] = _logits(case, g, 2.0)
        if case["op"] == "logprob":
            if case["masked"]:      # one class in five is forbidden, the same ones in every row; never all of them
                bar = torch.rand(C, generator=g, device="cuda") < 0.2
                bar[int(seed) % C] = False
                s["logits"][:, :C].masked_fill_(bar, -math.inf)
            tokens = torch.randint(0, C, (R,), generator=g, device="cuda")
            blank = torch.rand(R, generator=g, device="cuda") < 0.05          # positions of the padding: no token
            s["tokens"] = torch.where(blank, -1, tokens)
            s["g_logp"], s["g_entropy"] = _normal(g, (R,), torch.float32), _normal(g, (R,), torch.float32, 0.05)
        else:
            teacher = s["logits"][:, :C].float() + _normal(g, (R, C), torch.float32)
            t = torch.log_softmax(teacher / case["temperature"], dim=1) if case["tail"] else teacher
            top, idx = t.topk(case["top"], dim=1)
            absent = torch.rand((R, case["top"]), generator=g, device="cuda") < 0.02
            s["teacher_idx"], s["teacher_logp"] = torch.where(absent, -1, idx), top.contiguous()
            s["g_loss"] = torch.rand(R, generator=g, device="cuda") / R
    return s


# ---- the operators in elementary operations -----------------------------------------------------------------------------
def _plain_write(s):
    page = s["page"]
    keep = s["slots"] >= 0
    slot = s["slots"][keep]
    p, o = torch.div(slot, page, rounding_mode="floor"), slot % page
    s["k_pages"][p, :, o] = s["k"][keep]
    s["v_pages"][p, :, o] = s["v"][keep]
    return [s["k_pages"], s["v_pages"]]


def _plain_attend(s):
    q, table, lens = s["q"], s["block_table"].long(), s["seq_lens"].long()
    M, H, dh = q.shape
    Hkv, page = s["k_pages"].shape[1], s["k_pages"].shape[2]
    L = table.shape[1] * page
    k = s["k_pages"][table].permute(0, 2, 1, 3, 4).reshape(M, Hkv, L, dh).float()
    v = s["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(M, Hkv, L, dh).float()
    qf = q.float().view(M, Hkv, H // Hkv, dh) * dh ** -0.5
    score = torch.matmul(qf, k.transpose(2, 3).contiguous())
    score = score.masked_fill(torch.arange(L, device=q.device) >= lens[:, None, None, None], -math.inf)
    top = score.amax(dim=3, keepdim=True).clamp(min=-3.0e38)
    e = torch.exp(score - top)
    total = e.sum(dim=3, keepdim=True)
    out = torch.matmul(e, v) / total.clamp(min=1e-38)
    lse = (top + torch.log(total)).masked_fill(total == 0, -math.inf)
    return [out.reshape(M, H, dh).to(q.dtype), lse.reshape(M, H)]


def _plain_softmax(x):
    """(e / Z, log(e / Z), e, Z) of the rows of x, in its type."""
    x = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(dim=1, keepdim=True)
    return e / total, x - torch.log(total), e, total


def _plain_logprob(s):
    C = s["classes"]
    raw = s["logits"][:, :C].float()
    p, y, _, _ = _plain_softmax(raw / s["temperature"])
    given = s["tokens"] >= 0
    tok = s["tokens"].clamp(min=0)[:, None]
    logp = torch.where(given, y.gather(1, tok)[:, 0], 0.0)
    py = torch.where(p > 0, p * y, 0.0)
    entropy = -py.sum(dim=1)
    out = [logp, entropy]
    if s["top"]:
        k = min(s["top"], C)
        best, idx = torch.sort(raw, dim=1, descending=True, stable=True)          # equal values stay in the order of their classes
        idx = torch.where(best[:, :k] > -math.inf, idx[:, :k], -1)
        top = torch.where(idx >= 0, y.gather(1, idx.clamp(min=0)), -math.inf)
        pad = s["top"] - k
        out += [torch.nn.functional.pad(top, (0, pad), value=-math.inf), torch.nn.functional.pad(idx, (0, pad), value=-1)]
    if s["train"]:
        gl = torch.where(given, s["g_logp"], 0.0)[:, None]
        d = -gl * p - s["g_entropy"][:, None] * (py + p * entropy[:, None])
        d.scatter_add_(1, tok, gl)
        dl = torch.zeros_like(s["logits"])
        dl[:, :C] = d / s["temperature"]
        out.append(dl)
    return out


def _plain_distill(s):
    C, T = s["classes"], s["temperature"]
    x = s["logits"][:, :C].float() / T
    q, y, e, total = _plain_softmax(x)
    there = s["teacher_idx"] >= 0
    idx = s["teacher_idx"].clamp(min=0)
    if s["tail"]:
        p = torch.where(there, torch.exp(s["teacher_logp"]), 0.0)
        logp = s["teacher_logp"]
    else:
        t = (s["teacher_logp"] / T).masked_fill(~there, -math.inf)
        w = torch.exp(t - t.amax(dim=1, keepdim=True).clamp(min=-3.0e38))
        p = w / w.sum(dim=1, keepdim=True).clamp(min=1e-38)
        logp = torch.log(p)
    loss = torch.where(p > 0, p * (logp - y.gather(1, idx)), 0.0).sum(dim=1)
    mass = p.sum(dim=1, keepdim=True)
    d = q * mass
    d.scatter_add_(1, idx, -p)
    if s["tail"]:
        left = (1.0 - mass).clamp(min=0.0)
        hit = torch.zeros_like(x).scatter_add_(1, idx, there.float()) > 0
        er = e.masked_fill(hit, 0.0)
        zr = er.sum(dim=1, keepdim=True)
        zl = e.masked_fill(~hit, 0.0).sum(dim=1, keepdim=True)
        held = (zr > 0) & (left > 0)
        # log of the student's rest = -log(1 + listed / rest): the difference of two long sums' logarithms would lose it
        loss = loss + torch.where(held, left * (torch.log1p(-mass.clamp(max=1.0)) + torch.log1p(zl / zr)), 0.0)[:, 0]
        d = d + torch.where(held, left * (q - er / zr), 0.0)
    dl = torch.zeros_like(s["logits"])
    dl[:, :C] = d * (s["g_loss"][:, None] / T)
    return [loss, dl]


# ---- the framework's operators ------------------------------------------------------------------------------------------
def _own_write(s):
    from ttts_amd import ops
    ops.kv_page_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"])
    return [s["k_pages"], s["v_pages"]]


def _own_attend(s):
    from ttts_amd import ops
    return list(ops.attn_paged_decode(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["seq_lens"], s["dh"] ** -0.5))


def _own_logprob(s):
    from ttts_amd import ops
    r = ops.token_logprobs_fwd(s["logits"], s["tokens"], C=s["classes"], top_k=s["top"], temperature=s["temperature"])
    out = [r.logp, r.entropy]
    if s["top"]:
        out += [r.top_logp, r.top_idx]
    if s["train"]:
        out.append(ops.token_logprobs_bwd(s["logits"], s["tokens"], r.stats, r.entropy, s["g_logp"], s["g_entropy"], C=s["classes"],
                                          temperature=s["temperature"]))
    return out


def _own_distill(s):
    from ttts_amd import ops
    loss, stats = ops.distill_fwd(s["logits"], s["teacher_idx"], s["teacher_logp"], C=s["classes"], temperature=s["temperature"],
                                  tail=s["tail"])
    return [loss, ops.distill_bwd(s["logits"], s["teacher_idx"], s["teacher_logp"], stats, s["g_loss"], C=s["classes"],
                                  temperature=s["temperature"], tail=s["tail"])]


def run(state):
    if own:
        return {"write": _own_write, "attend": _own_attend, "logprob": _own_logprob, "distill": _own_distill}[state["op"]](state)
    return {"write": _plain_write, "attend": _plain_attend, "logprob": _plain_logprob, "distill": _plain_distill}[state["op"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "write":      # the rows that have a slot, read once and written once, and the slots
        row = 2 * case["heads"] * case["dh"] * b
        return {"bytes": 2 * row * (case["rows"] - case["pads"]) + 8 * case["rows"], "flops": 0}
    if case["op"] == "attend":     # every cached key and value once, the queries, the outputs and their log-sums
        lens = _lengths(case)
        M, H, Hkv, dh = (case[k] for k in ("seqs", "heads", "kv_heads", "dh"))
        tables = 4 * sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * sum(lens) * Hkv * dh * b + 2 * M * H * dh * b + 4 * M * H + tables + 4 * M, "flops": 4 * sum(lens) * H * dh}
    R, C = case["rows"], case["classes"]
    if case["op"] == "logprob":    # the logits once (once more for the gradient, which follows the whole row's sums), and the outputs
        n = R * C * b + R * (8 + 8) + R * case["top"] * 12
        return {"bytes": n + (R * C * b + R * case["pitch"] * b + 16 * R if case["train"] else 0), "flops": R * C * (14 if case["train"] else 8)}
    lists = R * case["top"] * 12
    return {"bytes": 2 * R * C * b + R * case["pitch"] * b + 2 * lists + 16 * R, "flops": R * C * (18 if case["tail"] else 12)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":      # copies: nothing is computed
        return None
    if case["op"] == "attend":
        group, page = case["heads"] // case["kv_heads"], case["page"]
        out = torch.zeros(case["seqs"], case["heads"], case["dh"], dtype=torch.float64, device="cuda")
        lse = torch.full((case["seqs"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
        for m, n in enumerate(_lengths(case)):
            if n == 0:
                continue
            ids = s["block_table"][m, :-(-n // page)].long()
            for h in range(case["kv_heads"]):
                k = s["k_pages"][ids, h].reshape(-1, case["dh"])[:n].double()
                v = s["v_pages"][ids, h].reshape(-1, case["dh"])[:n].double()
                z = (s["q"][m, h * group:(h + 1) * group].double() @ k.t()) / math.sqrt(case["dh"])
                out[m, h * group:(h + 1) * group] = torch.softmax(z, dim=1) @ v
                lse[m, h * group:(h + 1) * group] = torch.logsumexp(z, dim=1)
        return [out, lse]
    R, C, T = case["rows"], case["classes"], case["temperature"]
    parts = []
    for lo in range(0, R, 512):
        rows = slice(lo, min(R, lo + 512))
        y = torch.log_softmax(s["logits"][rows, :C].double() / T, dim=1)
        n = y.shape[0]
        at = torch.arange(n, device="cuda")
        dl = torch.zeros(n, case["pitch"], dtype=torch.float64, device="cuda")
        if case["op"] == "logprob":
            tok = s["tokens"][rows]
            logp = torch.where(tok >= 0, y[at, tok.clamp(min=0)], 0.0)
            ent = torch.special.entr(y.exp()).sum(dim=1)
            part = [logp, ent]
            if case["top"]:
                k = min(case["top"], C)
                top = torch.full((n, case["top"]), -math.inf, dtype=torch.float64, device="cuda")
                top[:, :k] = y.topk(k, dim=1).values
                part += [top, None]
            if case["train"]:
                one = torch.zeros_like(y)
                one[at, tok.clamp(min=0)] = (tok >= 0).double()
                gl = torch.where(tok >= 0, s["g_logp"][rows].double(), 0.0)[:, None]
                surprise = torch.where(y > -math.inf, y, 0.0) + ent[:, None]
                dl[:, :C] = (gl * (one - y.exp()) - s["g_entropy"][rows].double()[:, None] * y.exp() * surprise) / T
                part.append(dl)
        else:
            idx, t = s["teacher_idx"][rows], s["teacher_logp"][rows].double()
            gone = idx < 0
            if case["tail"]:
                p = t.exp().masked_fill(gone, 0.0)
            else:
                p = torch.softmax((t / T).masked_fill(gone, -math.inf), dim=1).nan_to_num(0.0)
            target = torch.zeros_like(y).scatter_add_(1, idx.clamp(min=0), p)
            listed_ = torch.zeros_like(y).scatter_add_(1, idx.clamp(min=0), (~gone).double()) > 0
            loss = (torch.special.xlogy(p, p) - p * y.gather(1, idx.clamp(min=0))).sum(dim=1)
            grad = y.exp() * p.sum(dim=1, keepdim=True) - target
            if case["tail"]:
                left = (1.0 - p.sum(dim=1, keepdim=True)).clamp(min=0.0)
                z = y.masked_fill(listed_, -math.inf)
                some = (z > -math.inf).any(dim=1, keepdim=True)
                lr = torch.logsumexp(z, dim=1, keepdim=True)
                loss = loss + torch.where(some, torch.special.xlogy(left, left) - left * lr, 0.0)[:, 0]
                grad = grad + torch.where(some, left * (y.exp() - (z - lr).exp()), 0.0)
            dl[:, :C] = grad * (s["g_loss"][rows].double()[:, None] / T)
            part = [loss, dl]
        parts.append(part)
    return [None if p[0] is None else torch.cat(p) for p in zip(*parts)]
