"""Operators on rows of vocabulary logits: a teacher's top logits, distillation from them with its gradient, and
the verification of drafted tokens.

Where ``own`` is false each is computed in its plain form, elementary torch operations in 32 bits (the verification
in 64: the steps of a cumulative sum over a vocabulary are closer than 32 bits resolve); where it is true the calls
are the framework's.

Logits are those of a decoder's head: a spread of a few units, a bias that falls with the token's rank, and a few
tokens per row far above the rest.  Some vocabularies end in padding that is masked with -inf.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
NEG = float("-inf")


def listed():
    return [
        # one position's alternatives, as a teacher that answers token by token gives them: all latency
        {"name": "top_token_f32", "op": "top", "dtype": "f32", "n": 1, "vocab": 151936, "pad": 0, "masked": 0, "k": 20, "temp": 1.0},
        # one answer's teacher pass with an odd vocabulary and rows that start off any boundary
        {"name": "top_odd_f16", "op": "top", "dtype": "f16", "n": 37, "vocab": 50257, "pad": 0, "masked": 0, "k": 8, "temp": 2.0},
        # the targets of a packed batch, a large vocabulary with masked padding
        {"name": "top_answer_bf16", "op": "top", "dtype": "bf16", "n": 256, "vocab": 151936, "pad": 0, "masked": 267, "k": 64, "temp": 2.0},
        # a long document's teacher pass, many alternatives kept
        {"name": "top_document_f32", "op": "top", "dtype": "f32", "n": 1024, "vocab": 151936, "pad": 0, "masked": 0, "k": 128, "temp": 1.0},
        # a short answer of a small vocabulary: all latency
        {"name": "distill_short_f32", "op": "distill", "dtype": "f32", "n": 12, "vocab": 8192, "pad": 0, "masked": 0, "k": 20, "temp": 1.0,
         "hard": 0.0, "rest": False, "ragged": False, "grad": True},
        # the targets of one training step, mixed with the labels' cross-entropy
        {"name": "distill_step_f32", "op": "distill", "dtype": "f32", "n": 256, "vocab": 151936, "pad": 0, "masked": 0, "k": 64, "temp": 2.0,
         "hard": 0.25, "rest": True, "ragged": False, "grad": True},
        # another odd vocabulary in strided rows, lists of several lengths, some rows without a teacher
        {"name": "distill_odd_f16", "op": "distill", "dtype": "f16", "n": 101, "vocab": 50257, "pad": 7, "masked": 0, "k": 33, "temp": 1.25,
         "hard": 0.5, "rest": True, "ragged": True, "grad": True},
        # a long document's targets in 16 bits
        {"name": "distill_document_bf16", "op": "distill", "dtype": "bf16", "n": 2048, "vocab": 151936, "pad": 0, "masked": 267, "k": 128, "temp": 1.0,
         "hard": 0.0, "rest": True, "ragged": False, "grad": True},
        # the same losses without a gradient, as an evaluation computes them
        {"name": "distill_eval_f32", "op": "distill", "dtype": "f32", "n": 301, "vocab": 151936, "pad": 0, "masked": 0, "k": 100, "temp": 1.0,
         "hard": 0.5, "rest": True, "ragged": True, "grad": False},
        # one sequence's draft
        {"name": "verify_one_f32", "op": "verify", "dtype": "f32", "b": 1, "d": 4, "vocab": 151936, "pad": 0, "masked": 0, "temp": 1.0,
         "draft": True, "ragged": False},
        # drafts that a lookup made (no draft probabilities), several lengths, an odd vocabulary
        {"name": "verify_lookup_f16", "op": "verify", "dtype": "f16", "b": 17, "d": 3, "vocab": 50257, "pad": 3, "masked": 0, "temp": 0.75,
         "draft": False, "ragged": True},
        # a serving batch
        {"name": "verify_batch_bf16", "op": "verify", "dtype": "bf16", "b": 64, "d": 5, "vocab": 151936, "pad": 0, "masked": 267, "temp": 1.0,
         "draft": True, "ragged": True},
    ]


def draw(rng):
    op = rng.choice(("top", "distill", "verify"))
    dtype = rng.choice(tuple(DTYPES))
    vocab = int(round(math.exp(rng.uniform(math.log(1000), math.log(152000)))))
    masked = rng.choice((0, 0, vocab // 50))
    temp = rng.choice((0.5, 0.75, 1.0, 1.25, 2.0, 4.0))
    pad = rng.choice((0, 0, 0, 1, 5, 64))
    most = 300_000_000 // (vocab * (4 if dtype == "f32" else 2))  # rows
    c = {"op": op, "dtype": dtype, "vocab": vocab, "pad": pad, "masked": masked, "temp": temp}
    if op == "verify":
        d = rng.randint(1, 8)
        b = int(round(math.exp(rng.uniform(0.0, math.log(64)))))
        c.update(b=max(1, min(b, most // (2 * d + 1))), d=d, draft=rng.random() < 0.7, ragged=rng.random() < 0.5)
        if rng.random() < 0.15:
            c["temp"] = 0.0  # greedy
        return c
    c["n"] = max(1, min(most, int(round(math.exp(rng.uniform(0.0, math.log(2048)))))))
    c["k"] = int(round(math.exp(rng.uniform(0.0, math.log(256)))))
    if op == "distill":
        c.update(hard=rng.choice((0.0, 0.25, 0.5, 1.0)), rest=rng.random() < 0.7, ragged=rng.random() < 0.5, grad=rng.random() < 0.8)
    return c


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    v = case["vocab"]
    if case["op"] == "top":
        return {"bytes": case["n"] * (v * es + 8 * case["k"] + 4), "flops": 3 * case["n"] * v}
    if case["op"] == "distill":
        return {"bytes": case["n"] * (v * es * (2 if case["grad"] else 1) + 8 * case["k"] + 24), "flops": (7 if case["grad"] else 3) * case["n"] * v}
    rows = case["b"] * (case["d"] + 1 + (case["d"] if case["draft"] else 0))
    return {"bytes": rows * v * es + case["b"] * (3 * case["d"] + 3) * 4, "flops": 3 * rows * v}


def _logits(g, n, vocab, near=None):
    """[n x vocab] f32 logits of a head; near: another model's logits of the same positions."""
    noise = torch.randn(n, vocab, generator=g, device=DEV)
    if near is not None:
        z = near + 0.7 * noise
    else:
        rank = torch.randperm(vocab, generator=g, device=DEV).float()
        z = 1.5 * noise + (4.0 - 0.6 * torch.log1p(rank))
    top = torch.randint(vocab, (n, 6), generator=g, device=DEV)
    lift = 3.0 + 6.0 * torch.rand(n, 6, generator=g, device=DEV)
    return z.scatter_add_(1, top, lift)


def _rows(z, case):
    """z in the case's type, masked at the end of the vocabulary, in rows of stride vocab + pad."""
    n, v = z.shape
    out = torch.zeros(n, v + case["pad"], dtype=DTYPES[case["dtype"]], device=DEV)[:, :v]
    out.copy_(z)
    if case["masked"]:
        out[:, v - case["masked"]:] = NEG
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    v, s = case["vocab"], {"case": case}
    live = v - case["masked"]
    if case["op"] == "verify":
        b, d = case["b"], case["d"]
        zp = _logits(g, b * (d + 1), v)
        s["logits"] = _rows(zp, case)
        zq = _logits(g, b * d, v, near=zp.view(b, d + 1, v)[:, :d].reshape(b * d, v))
        s["draft"] = _rows(zq, case) if case["draft"] else None
        # the drafted tokens: samples of the draft's distribution, or a lookup's guesses at the target's likely tokens
        pick = s["draft"].float() if case["draft"] else zp.view(b, d + 1, v)[:, :d].reshape(b * d, v) * 1.5
        if case["masked"]:
            pick = pick.clone()
            pick[:, live:] = NEG
        gumbel = -torch.log(-torch.log(torch.rand(b * d, v, generator=g, device=DEV).clamp_(1e-20, 1 - 1e-7)))
        t = case["temp"] if case["temp"] > 0 else 0.5
        s["drafted"] = (pick / t + gumbel).argmax(1).to(torch.int32).view(b, d).contiguous()
        s["lens"] = torch.randint(0, d + 1, (b,), generator=g, device=DEV, dtype=torch.int32) if case["ragged"] else None
        s["uniform"] = torch.rand(b, d + 1, generator=g, device=DEV)
        s["accepted"] = torch.empty(b, dtype=torch.int32, device=DEV)
        s["tokens"] = torch.empty(b, d + 1, dtype=torch.int32, device=DEV)
    else:
        n, k = case["n"], case["k"]
        z = _logits(g, n, v)
        s["logits"] = _rows(z, case)
        s["ids"] = torch.empty(n, k, dtype=torch.int32, device=DEV)
        s["vals"] = torch.empty(n, k, dtype=torch.float32, device=DEV)
        s["rest"] = torch.empty(n, dtype=torch.float32, device=DEV)
        if case["op"] == "distill":
            zt = _logits(g, n, v, near=z)
            zt[:, live:] = NEG
            vals, ids = torch.topk(zt, k, dim=1)
            s["vals"].copy_(vals)
            s["ids"].copy_(ids)
            zt.scatter_(1, ids, NEG)
            s["rest"].copy_(torch.logsumexp(zt / case["temp"], 1))
            del zt
            if case["ragged"]:  # lists of 0 to k tokens; a row without a list has no teacher
                held = torch.randint(0, k + 1, (n, 1), generator=g, device=DEV)
                s["ids"].masked_fill_(torch.arange(k, device=DEV) >= held, -1)
                s["rest"].masked_fill_(held[:, 0] == 0, NEG)
            if not case["rest"]:
                s["rest"] = None
            s["tok"] = torch.randint(0, live, (n,), generator=g, device=DEV, dtype=torch.int32)
            s["weights"] = (0.25 + torch.rand(n, generator=g, device=DEV)) / n
            s["kl"] = torch.empty(n, dtype=torch.float32, device=DEV)
            s["logp"] = torch.empty(n, dtype=torch.float32, device=DEV)
            s["dlogits"] = torch.empty_like(s["logits"].as_strided((n, v), (v, 1))) if case["grad"] else None
    if own:
        import rust_trainer_amd as rt

        s["ctx"] = rt.default_context()
    return s


# ------------------------------------------------------------------ the framework's calls
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own_top(s, case):
    from rust_trainer_amd.distill import top_logits_d

    z = s["logits"]
    top_logits_d(s["ctx"], z.data_ptr(), TYPE_IDS[case["dtype"]], case["n"], case["vocab"], z.stride(0), case["k"], s["vals"].data_ptr(),
                 s["ids"].data_ptr(), s["rest"].data_ptr(), temperature=case["temp"], stream=torch.cuda.current_stream().cuda_stream)
    return s["vals"], s["ids"], s["rest"]


def _own_distill(s, case):
    from rust_trainer_amd.distill import distill_d, teacher_d

    z, dz = s["logits"], s["dlogits"]
    teacher = teacher_d(case["k"], s["ids"].data_ptr(), s["vals"].data_ptr(), _ptr(s["rest"]), case["temp"])
    distill_d(s["ctx"], z.data_ptr(), TYPE_IDS[case["dtype"]], case["n"], case["vocab"], z.stride(0), teacher, s["tok"].data_ptr(),
              s["weights"].data_ptr() if case["grad"] else 0, s["kl"].data_ptr(), s["logp"].data_ptr(), _ptr(dz), dz.stride(0) if case["grad"] else 0,
              hard=case["hard"], stream=torch.cuda.current_stream().cuda_stream)
    return (s["kl"], s["logp"], dz) if case["grad"] else (s["kl"], s["logp"])


def _own_verify(s, case):
    from rust_trainer_amd.distill import verify_draft_d

    z, q = s["logits"], s["draft"]
    verify_draft_d(s["ctx"], z.data_ptr(), TYPE_IDS[case["dtype"]], z.stride(0), _ptr(q), 0 if q is None else q.stride(0), case["b"], case["d"],
                   case["vocab"], s["drafted"].data_ptr(), _ptr(s["lens"]), s["uniform"].data_ptr(), s["accepted"].data_ptr(),
                   s["tokens"].data_ptr(), temperature=case["temp"], stream=torch.cuda.current_stream().cuda_stream)
    return s["accepted"], s["tokens"]


# ------------------------------------------------------------------ plain forms
def _plain_top(s, case):
    z = s["logits"].float()
    vals, ids = torch.sort(z, dim=1, descending=True, stable=True)
    k, left = case["k"], vals[:, case["k"]:] / case["temp"]
    if left.shape[1] == 0:
        rest = torch.full((case["n"],), NEG, device=DEV)
    else:
        m = left.amax(1)
        rest = m + torch.log(torch.exp(left - torch.where(m == NEG, 0.0, m)[:, None]).sum(1))
    return vals[:, :k].contiguous(), ids[:, :k].to(torch.int32), rest


def _plain_distill(s, case):
    n, v, temp, hard = case["n"], case["vocab"], case["temp"], case["hard"]
    z = s["logits"].float()
    held = s["ids"] >= 0
    ids = torch.where(held, s["ids"], 0).long()
    # the teacher's distribution over its listed tokens and the rest; a row's scalars in 64 bits, since a small
    # divergence is what is left of large terms
    t = torch.where(held, s["vals"].double() / temp, NEG)
    r = s["rest"].double()[:, None] if s["rest"] is not None else torch.full((n, 1), NEG, dtype=torch.float64, device=DEV)
    t = torch.cat((t, r), 1)
    tm = t.amax(1, keepdim=True)
    taught = tm > NEG
    logp_t = t - torch.where(taught, tm, 0.0)
    logp_t = logp_t - torch.log(torch.exp(logp_t).sum(1, keepdim=True))
    p = torch.where(taught, torch.exp(logp_t), 0.0)
    # the student's
    m = z.amax(1, keepdim=True)
    e = torch.exp((z - m) / temp)
    listed_ = torch.zeros(n, v + 1, dtype=torch.bool, device=DEV).scatter_(1, torch.where(held, ids, v), True)[:, :v]
    out = torch.where(listed_, 0.0, e).sum(1, keepdim=True, dtype=torch.float64)
    total = torch.where(listed_, e, 0.0).sum(1, keepdim=True, dtype=torch.float64) + out
    logq = torch.cat(((z.gather(1, ids).double() - m) / temp, torch.log(out)), 1) - torch.log(total)
    kl = torch.where(p > 0, p * (torch.where(p > 0, logp_t, 0.0) - logq), 0.0).sum(1).float()
    e1 = torch.exp(z - m)
    total1 = e1.sum(1, keepdim=True, dtype=torch.float64)
    tok = s["tok"].long()[:, None]
    logp = (z.gather(1, tok).double() - m - torch.log(total1))[:, 0].float()
    if not case["grad"]:
        return kl, logp
    w = s["weights"][:, None]
    pr = p[:, -1:]
    share = torch.where(pr > 0, pr / out, 0.0)
    g = e * torch.where(listed_, (1.0 / total).float(), (1.0 / total - share).float())
    g.scatter_add_(1, ids, torch.where(held, -p[:, :-1], 0.0).float())
    g = torch.where(taught, g * (w * ((1.0 - hard) * temp)), 0.0)
    g += (hard * w) * (e1 / total1.float())
    g.scatter_add_(1, tok, -hard * w)
    return kl, logp, g.to(z.dtype if case["dtype"] == "f32" else DTYPES[case["dtype"]])


def _plain_verify(s, case):
    b, d, v, temp = case["b"], case["d"], case["vocab"], case["temp"]
    z = s["logits"].double().view(b, d + 1, v)
    x = s["drafted"].long()
    lens = s["lens"].long() if s["lens"] is not None else torch.full((b,), d, device=DEV)
    steps = torch.arange(d, device=DEV)
    if temp == 0.0:
        best = torch.argmax((z == z.amax(2, keepdim=True)).to(torch.int8), 2)
        ok = x == best[:, :d]
    else:
        p = torch.exp((z - z.amax(2, keepdim=True)) / temp)
        p = p / p.sum(2, keepdim=True)
        if s["draft"] is not None:
            q = s["draft"].double().view(b, d, v)
            q = torch.exp((q - q.amax(2, keepdim=True)) / temp)
            q = q / q.sum(2, keepdim=True)
        else:
            q = torch.zeros(b, d, v, dtype=torch.float64, device=DEV).scatter_(2, x[:, :, None], 1.0)
        u = s["uniform"].double()
        ok = u[:, :d] * q.gather(2, x[:, :, None])[:, :, 0] < p[:, :d].gather(2, x[:, :, None])[:, :, 0]
    ok = ok & (steps < lens[:, None])
    accepted = torch.cumprod(ok.long(), 1).sum(1)
    row = torch.arange(b, device=DEV)
    if temp == 0.0:
        after = best[row, accepted]
    else:
        pa = p[row, accepted]
        qa = torch.where((accepted < lens)[:, None], q[row, accepted.clamp(max=d - 1)], 0.0)
        w = (pa - qa).clamp_min(0.0)
        w = torch.where(w.sum(1, keepdim=True) > 0, w, pa)
        c = torch.cumsum(w, 1)
        after = (c <= u[:, d:] * c[:, -1:]).sum(1).clamp(max=v - 1)
    wide = torch.arange(d + 1, device=DEV)
    tokens = torch.where(wide < accepted[:, None], torch.cat((x, x[:, :1]), 1), torch.where(wide == accepted[:, None], after[:, None], -1))
    return accepted.to(torch.int32), tokens.to(torch.int32)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return (_own_top if op == "top" else _own_distill if op == "distill" else _own_verify)(state, case)
    return (_plain_top if op == "top" else _plain_distill if op == "distill" else _plain_verify)(state, case)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    v, temp = case["vocab"], case["temp"]
    if case["op"] == "top":
        # one whole-number key per logit: its order in the high half, the lower index first in the low half
        z = s["logits"].float()
        bits = (z + 0.0).contiguous().view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = key * (1 << 20) + ((1 << 20) - 1 - torch.arange(v, device=DEV))
        ids = torch.topk(key, case["k"], dim=1).indices
        vals = z.gather(1, ids)
        left = z.double().scatter_(1, ids, NEG)
        return vals.double(), ids.to(torch.int32), torch.logsumexp(left / temp, 1)
    if case["op"] == "distill":
        n, k, hard = case["n"], case["k"], case["hard"]
        z = s["logits"].double().requires_grad_(case["grad"])
        held = s["ids"] >= 0
        spot = torch.where(held, s["ids"].long(), v)
        t = torch.where(held, s["vals"].double() / temp, NEG)
        r = s["rest"].double() if s["rest"] is not None else torch.full((n,), NEG, dtype=torch.float64, device=DEV)
        lt = torch.cat((t, r[:, None]), 1)
        taught = lt.amax(1) > NEG
        lt = torch.log_softmax(torch.where(taught[:, None], lt, 0.0), 1)
        lq = torch.log_softmax(z / temp, 1)
        wide = torch.cat((lq, torch.full((n, 1), NEG, dtype=torch.float64, device=DEV)), 1)
        gone = torch.zeros(n, v + 1, dtype=torch.bool, device=DEV).scatter_(1, spot, True)
        lr = torch.logsumexp(wide.masked_fill(gone, NEG)[:, :v], 1)
        lq_listed = torch.where(held, lq.gather(1, torch.where(held, spot, 0)), 0.0)
        pt = torch.exp(lt)
        own_bits = torch.where(held, pt[:, :k] * (torch.where(held, lt[:, :k], 0.0) - lq_listed), 0.0).sum(1)
        some = torch.isfinite(lt[:, k]) & taught
        tail = torch.where(some, pt[:, k] * (torch.where(some, lt[:, k], 0.0) - torch.where(some, lr, 0.0)), 0.0)
        kl = torch.where(taught, own_bits + tail, 0.0)
        logp = torch.log_softmax(z, 1).gather(1, s["tok"].long()[:, None])[:, 0]
        if not case["grad"]:
            return kl, logp
        loss = (s["weights"].double() * ((1.0 - hard) * temp * temp * kl - hard * logp)).sum()
        (grad,) = torch.autograd.grad(loss, z)
        return kl.detach(), logp.detach(), grad
    b, d = case["b"], case["d"]
    z = s["logits"].double().view(b, d + 1, v)
    lens = s["lens"].tolist() if s["lens"] is not None else [d] * b
    x, u = s["drafted"].tolist(), s["uniform"].double().tolist()
    lq = torch.log_softmax(s["draft"].double().view(b, d, v) / temp, 2) if s["draft"] is not None and temp > 0 else None
    accepted, tokens = [], []
    for i in range(b):
        lp = torch.log_softmax(z[i] / temp, 1) if temp > 0 else None
        a = 0
        while a < lens[i]:
            if temp == 0:
                go = x[i][a] == int((z[i, a] == z[i, a].max()).nonzero()[0])
            else:
                go = u[i][a] * (math.exp(float(lq[i, a, x[i][a]])) if lq is not None else 1.0) < math.exp(float(lp[a, x[i][a]]))
            if not go:
                break
            a += 1
        if temp == 0:
            after = int((z[i, a] == z[i, a].max()).nonzero()[0])
        else:
            w = torch.exp(lp[a])
            if a < lens[i]:
                left = w.clone()
                if lq is not None:
                    left = torch.relu(left - torch.exp(lq[i, a]))
                else:
                    left[x[i][a]] = 0.0
                w = left if float(left.sum()) > 0 else w
            c = torch.cumsum(w, 0)
            after = min(int(torch.searchsorted(c, c[-1] * u[i][d], right=True)), v - 1)
        accepted.append(a)
        tokens.append(x[i][:a] + [after] + [-1] * (d - a))
    return torch.tensor(accepted, dtype=torch.int32, device=DEV), torch.tensor(tokens, dtype=torch.int32, device=DEV)
