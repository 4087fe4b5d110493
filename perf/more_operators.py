"""Operators on a paged cache of keys and values: appending new tokens' rows with the rotation of their positions,
attention of trees (or runs) of new tokens over what is cached, and keeping the accepted tokens of a tree.

Where ``own`` is false each is computed in its plain form, elementary torch operations in 32 bits (the rotations'
angles in 64: at far positions 32 lose them); where it is true the calls are the framework's.

The cache is in 16 bits: pages of keys [pages x KV heads x slots x head size], pages of values [pages x KV heads x
head size x slots] (a value's slots next to each other, as the attention's product reads them).  A sequence holds
``lens`` tokens; its new ones are the rows ``starts[i] .. starts[i + 1] - 1``, in the slots after them.  ``parents`` makes a
tree of them: the new token that a token follows, -1 for the last cached one.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
NEG = float("-inf")
DEPTH = 8  # longest branch of a drafted tree


def listed():
    return [
        # one token of one conversation enters one layer's cache (the heads of this repository's default step): all latency
        {"name": "append_token_f32", "op": "append", "dtype": "f32", "cache": "f16", "b": 1, "len": 4096, "new": 1, "ragged": False, "tree": False,
         "heads": 16, "kv": 8, "d": 128, "rot": 128, "neox": True, "norm": True, "page": 64, "base": 1e6, "gap": 0},
        # drafted trees of a serving batch at far positions, heads without a norm, rows of a fused projection
        {"name": "append_trees_bf16", "op": "append", "dtype": "bf16", "cache": "bf16", "b": 8, "len": 16000, "new": 31, "ragged": False, "tree": True,
         "heads": 32, "kv": 8, "d": 128, "rot": 128, "neox": False, "norm": False, "page": 64, "base": 5e5, "gap": 0},
        # prompts of several lengths, an odd head size that is rotated in part, small pages, rows further apart than they are long
        {"name": "append_odd_f16", "op": "append", "dtype": "f16", "cache": "f16", "b": 13, "len": 333, "new": 157, "ragged": True, "tree": False,
         "heads": 15, "kv": 3, "d": 80, "rot": 32, "neox": True, "norm": False, "page": 32, "base": 1e4, "gap": 37},
        # a long document's prompt in one call
        {"name": "append_prompt_f32", "op": "append", "dtype": "f32", "cache": "f16", "b": 1, "len": 0, "new": 16384, "ragged": False, "tree": False,
         "heads": 16, "kv": 8, "d": 128, "rot": 128, "neox": True, "norm": True, "page": 64, "base": 1e6, "gap": 0},
        # the next token of one conversation: all latency
        {"name": "attend_token_f32", "op": "attend", "dtype": "f32", "cache": "f16", "b": 1, "len": 1000, "new": 1, "ragged": False, "tree": False,
         "heads": 16, "kv": 8, "d": 128, "page": 64, "gap": 0},
        # the next tokens of a serving batch of several lengths
        {"name": "attend_batch_bf16", "op": "attend", "dtype": "bf16", "cache": "bf16", "b": 64, "len": 8192, "new": 1, "ragged": True, "tree": False,
         "heads": 32, "kv": 8, "d": 128, "page": 64, "gap": 0},
        # drafted trees over long contexts
        {"name": "attend_trees_f16", "op": "attend", "dtype": "f16", "cache": "f16", "b": 8, "len": 16000, "new": 63, "ragged": False, "tree": True,
         "heads": 32, "kv": 8, "d": 128, "page": 64, "gap": 0},
        # small trees of several sizes, sequences without new tokens among them, an odd head size, small pages, strided rows
        {"name": "attend_odd_f32", "op": "attend", "dtype": "f32", "cache": "bf16", "b": 13, "len": 3001, "new": 11, "ragged": True, "tree": True,
         "heads": 15, "kv": 3, "d": 80, "page": 32, "gap": 37},
        # the next token over one very long document
        {"name": "attend_document_f16", "op": "attend", "dtype": "f16", "cache": "f16", "b": 1, "len": 131072, "new": 1, "ragged": False, "tree": False,
         "heads": 32, "kv": 8, "d": 128, "page": 128, "gap": 0},
        # a prompt's next piece over what is cached of it
        {"name": "attend_prompt_bf16", "op": "attend", "dtype": "bf16", "cache": "bf16", "b": 1, "len": 6144, "new": 2048, "ragged": False, "tree": False,
         "heads": 32, "kv": 8, "d": 128, "page": 64, "gap": 0},
        # one sequence's accepted branch in every layer: all latency
        {"name": "keep_branch_f16", "op": "keep", "cache": "f16", "layers": 28, "b": 1, "len": 200, "new": 31, "ragged": False, "tree": True, "kept": 4,
         "kv": 8, "d": 128, "page": 64},
        # a serving batch's accepted branches
        {"name": "keep_batch_bf16", "op": "keep", "cache": "bf16", "layers": 28, "b": 32, "len": 130, "new": 63, "ragged": True, "tree": True, "kept": 8,
         "kv": 8, "d": 128, "page": 32},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "append", "attend", "attend", "attend", "keep"))
    cache = rng.choice(("f16", "bf16"))
    d = rng.choice((64, 80, 96, 128, 128, 256))
    c = {"op": op, "cache": cache, "ragged": rng.random() < 0.5, "kv": rng.choice((1, 2, 3, 4, 8)), "d": d, "page": rng.choice((32, 64, 128, 256))}
    if op == "keep":
        c.update(layers=rng.randint(1, 32), tree=True, b=_spread(rng, 1, 32), len=_spread(rng, 1, 200), new=rng.randint(8, 64), kept=rng.randint(1, 8))
        return c
    c["dtype"] = rng.choice((cache, "f32"))
    c["heads"] = c["kv"] * rng.choice((1, 2, 4, 5, 7, 8))
    c["gap"] = rng.choice((0, 0, 0, 1, 8, 37))
    c["tree"] = rng.random() < 0.4
    c["b"] = _spread(rng, 1, 64)
    c["new"] = rng.randint(2, 64) if c["tree"] else rng.choice((1, 1, _spread(rng, 1, 2048)))
    if op == "append":
        # at most the rows of the largest listed prompt, and caches of half a GB
        c["new"] = min(c["new"], max(1, 16384 * 16 * 128 // (c["heads"] * d * c["b"])))
        c["len"] = min(_spread(rng, 1, 16384), max(1, 2 ** 28 // (c["b"] * c["kv"] * d * 2)))
        c.update(rot=rng.choice((d, d, d // 2, 32)), neox=rng.random() < 0.6, norm=rng.random() < 0.4, base=rng.choice((1e4, 5e5, 1e6)))
        return c
    c["len"] = _spread(rng, 1, 65536)
    # at most the largest listed batch's cache and the prompt piece's products
    c["len"] = min(c["len"], max(1, 64 * 8192 * 8 * 128 // 2 // (c["b"] * c["kv"] * d)))
    most = 2048 * 6144 * 32 * 128
    c["new"] = min(c["new"], max(1, most // (c["b"] * c["heads"] * d * (c["len"] + c["new"]))))
    return c


def _sizes(case):
    """Cached tokens and new tokens of each sequence: of the case alone, so that its work is known without a seed."""
    rng = random.Random(case["b"] * 1000003 + case["len"] * 1009 + case["new"] * 31 + case["page"])
    lens, counts = [], []
    for i in range(case["b"]):
        if case["ragged"] and i:
            lens.append(int(case["len"] * rng.uniform(0.0, 1.0) ** 0.5))
            counts.append(rng.randint((case["new"] + 1) // 2, case["new"]) if rng.random() < 0.85 else 0)
        else:
            lens.append(case["len"])
            counts.append(case["new"])
    return lens, counts


def work(case):
    lens, counts = _sizes(case)
    n, row = sum(counts), case["kv"] * case["d"]
    if case["op"] == "keep":
        moved = 2 * case["layers"] * case["b"] * case["kept"] * row
        return {"bytes": 2 * 2 * moved, "flops": moved}
    es, heads = 4 if case["dtype"] == "f32" else 2, case["heads"] * case["d"]
    if case["op"] == "append":
        return {"bytes": n * ((2 * heads + 2 * row) * es + 2 * row * 2), "flops": 4 * n * (heads + row)}
    if case["tree"]:
        seen = sum(m * (c + min(m, DEPTH) / 2) for c, m in zip(lens, counts))
    else:
        seen = sum(m * c + m * (m + 1) / 2 for c, m in zip(lens, counts))
    keys = sum(c + m for c, m in zip(lens, counts) if m)
    return {"bytes": keys * row * 2 * 2 + 2 * n * heads * es, "flops": 4 * seen * heads}


def _tree(rng, m):
    """Parents of a tree of m nodes, no branch longer than DEPTH, and the nodes' depths."""
    parents, depths = [], []
    for i in range(m):
        p = rng.randint(max(-1, i - 12), i - 1)
        while p >= 0 and depths[p] >= DEPTH - 1:
            p = parents[p]
        parents.append(p)
        depths.append(0 if p < 0 else depths[p] + 1)
    return parents, depths


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _strided(g, n, width, gap, dtype):
    """n rows of random numbers, `gap` elements further apart than they are long."""
    t = torch.zeros(n, width + gap, dtype=dtype, device=DEV)[:, :width]
    t.copy_(torch.randn(n, width, generator=g, device=DEV))
    return t


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = random.Random(seed)
    lens, counts = _sizes(case)
    b, page, kv, d = case["b"], case["page"], case["kv"], case["d"]
    s = {"case": case, "counts": counts, "held": lens, "n": sum(counts)}
    # the pages of each sequence, anywhere in the pool
    pages = [-(-(c + m) // page) for c, m in zip(lens, counts)]
    pool = max(1, sum(pages))
    order = list(range(pool))
    rng.shuffle(order)
    wide = max(1, max(pages))
    table, at = [], 0
    for p in pages:
        table.append(order[at:at + p] + [0] * (wide - p))
        at += p
    s["table"], s["lens"] = _ints(table), _ints(lens)
    starts = [0]
    for m in counts:
        starts.append(starts[-1] + m)
    s["starts"] = _ints(starts)
    s["row_seq"] = torch.repeat_interleave(torch.arange(b, device=DEV), torch.tensor(counts, device=DEV))
    s["row_new"] = torch.arange(s["n"], device=DEV) - s["starts"].long()[s["row_seq"]]
    layers = case.get("layers", 1)
    dt = DTYPES[case["cache"]]
    s["k"] = torch.empty(layers, pool, kv, page, d, dtype=dt, device=DEV)
    s["v"] = torch.empty(layers, pool, kv, d, page, dtype=dt, device=DEV)
    for t in (s["k"], s["v"]):
        for layer in t:
            layer.copy_(torch.randn(layer.shape, generator=g, device=DEV))
    if case["tree"]:
        trees = [_tree(rng, m) for m in counts]
        s["parents"] = _ints([p for t in trees for p in t[0]])
        s["positions"] = _ints([c + x for c, t in zip(lens, trees) for x in t[1]])
    else:
        s["parents"] = s["positions"] = None
    if case["op"] == "keep":
        # the accepted branches: nodes at the front of the draft stay where they are, the others come from behind the kept slots
        kept = []
        for m in counts:
            k = rng.randint(1, case["kept"]) if case["ragged"] else case["kept"]
            k = min(k, m)
            front = rng.randint(0, k)
            front = k if m - k < k - front else front
            row = list(range(front)) + sorted(rng.sample(range(k, m), k - front))
            kept.append(row + [-1] * (case["kept"] - k))
        s["kept"] = _ints(kept)
        s["kept_lists"] = kept
        s["after"] = torch.empty(b, dtype=torch.int32, device=DEV)
    else:
        n, h, x = s["n"], case["heads"], DTYPES[case["dtype"]]
        if case["op"] == "append":
            qkv = _strided(g, n, (h + 2 * kv) * d, case["gap"], x)
            s["q"], s["kx"], s["vx"] = qkv[:, :h * d], qkv[:, h * d:(h + kv) * d], qkv[:, (h + kv) * d:]
            if case["norm"]:
                s["q_norm"] = 0.5 + torch.rand(d, generator=g, device=DEV)
                s["k_norm"] = 0.5 + torch.rand(d, generator=g, device=DEV)
        else:
            s["q"] = _strided(g, n, h * d, case["gap"], x)
            s["q"] *= 1.5  # scores of a spread at which some hundreds of keys share a row's weight
        s["out"] = torch.empty(n, h * d, dtype=x, device=DEV)
    if own:
        from rust_trainer_amd.kvcache import KvCache, rope_d, seqs_d

        s["handle"] = KvCache(layers, pool, page, kv, d, type=TYPE_IDS[case["cache"]], pages_d=(s["k"].data_ptr(), s["v"].data_ptr()))
        s["seqs"] = seqs_d(b, s["lens"].data_ptr(), s["table"].data_ptr(), wide, starts_ptr=s["starts"].data_ptr())
        if case["op"] == "append":
            s["rope"] = rope_d(case["rot"], case["base"], neox=case["neox"], q_norm_ptr=s["q_norm"].data_ptr() if case["norm"] else 0,
                               k_norm_ptr=s["k_norm"].data_ptr() if case["norm"] else 0, eps=1e-6)
    return s


# ------------------------------------------------------------------ the framework's calls
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own_append(s, case):
    q, k, v, out = s["q"], s["kx"], s["vx"], s["out"]
    s["handle"].append_d(0, s["seqs"], s["n"], TYPE_IDS[case["dtype"]], s["rope"], k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                         n_head=case["heads"], q_ptr=q.data_ptr(), ldq=q.stride(0), q_out_ptr=out.data_ptr(), ldo=out.stride(0),
                         positions_ptr=_ptr(s["positions"]), stream=torch.cuda.current_stream().cuda_stream)
    return out, s["k"], s["v"]


def _own_attend(s, case):
    q, out = s["q"], s["out"]
    s["handle"].attend_d(0, s["seqs"], s["n"], TYPE_IDS[case["dtype"]], case["heads"], q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0),
                         parents_ptr=_ptr(s["parents"]), stream=torch.cuda.current_stream().cuda_stream)
    return out


def _own_keep(s, case):
    s["handle"].keep_d(s["seqs"], s["kept"].data_ptr(), case["kept"], lens_out_ptr=s["after"].data_ptr(),
                       stream=torch.cuda.current_stream().cuda_stream)
    return s["k"], s["v"], s["after"]


# ------------------------------------------------------------------ plain forms
def _slots(s, case, seq, slot):
    """(page, slot in the page) of slots of sequences."""
    return s["table"].long()[seq, slot // case["page"]], slot % case["page"]


def _plain_append(s, case):
    n, d, rot = s["n"], case["d"], case["rot"]
    pos = s["positions"].double() if s["positions"] is not None else (s["lens"].long()[s["row_seq"]] + s["row_new"]).double()
    i = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    angle = pos[:, None] * case["base"] ** (-2.0 * i / rot)
    c, sn = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]

    def rows(x, heads, w):
        x = x.float().reshape(n, heads, d)
        if w is not None:
            x = x / torch.sqrt((x * x).mean(2, keepdim=True) + 1e-6) * w
        a, z = (x[..., :rot // 2], x[..., rot // 2:rot]) if case["neox"] else (x[..., 0:rot:2], x[..., 1:rot:2])
        y1, y2 = a * c - z * sn, z * c + a * sn
        turned = torch.cat((y1, y2), 2) if case["neox"] else torch.stack((y1, y2), 3).reshape(n, heads, rot)
        return torch.cat((turned, x[..., rot:]), 2)

    page, slot = _slots(s, case, s["row_seq"], s["lens"].long()[s["row_seq"]] + s["row_new"])
    s["k"][0][page, :, slot] = rows(s["kx"], case["kv"], s.get("k_norm")).to(s["k"].dtype)
    s["v"][0][page, :, :, slot] = s["vx"].reshape(n, case["kv"], d).to(s["v"].dtype)
    s["out"].copy_(rows(s["q"], case["heads"], s.get("q_norm")).reshape(n, -1))
    return s["out"], s["k"], s["v"]


def _plain_attend(s, case):
    d, kv, heads, page = case["d"], case["kv"], case["heads"], case["page"]
    group, at = heads // kv, 0
    for i, (held, m) in enumerate(zip(s["held"], s["counts"])):
        if m == 0:
            continue
        total = held + m
        ids = s["table"][i, :-(-total // page)].long()
        k = s["k"][0][ids].float().permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :total]
        v = s["v"][0][ids].float().permute(1, 0, 3, 2).reshape(kv, -1, d)[:, :total]
        q = s["q"][at:at + m].float().reshape(m, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * m, d)
        score = torch.matmul(q, k.transpose(1, 2)).mul_(1.0 / math.sqrt(d))
        if m > 1:
            if s["parents"] is None:
                seen = torch.ones(m, m, dtype=torch.bool, device=DEV).tril()
            else:
                seen = torch.zeros(m, m + 1, dtype=torch.bool, device=DEV)
                up = s["parents"][at:at + m].long()
                node = torch.arange(m, device=DEV)
                for _ in range(DEPTH):
                    seen.scatter_(1, torch.where(node < 0, m, node)[:, None], True)
                    node = torch.where(node < 0, -1, up[node.clamp(min=0)])
                seen = seen[:, :m]
            score[:, :, held:].masked_fill_(~seen.repeat(group, 1), NEG)
        score = torch.exp(score - score.amax(2, keepdim=True))
        o = torch.matmul(score, v) / score.sum(2, keepdim=True)
        s["out"][at:at + m] = o.reshape(kv, group, m, d).permute(2, 0, 1, 3).reshape(m, heads * d).to(s["out"].dtype)
        at += m
    return s["out"]


def _plain_keep(s, case):
    b, most = case["b"], case["kept"]
    kept = s["kept"].long()
    ok = kept >= 0
    seq = torch.arange(b, device=DEV)[:, None].expand(b, most)
    lens = s["lens"].long()[:, None]
    last = s["table"].shape[1] * case["page"] - 1
    src = _slots(s, case, seq, torch.where(ok, lens + kept, lens).clamp(max=last))
    dst = _slots(s, case, seq, (lens + torch.arange(most, device=DEV)).clamp(max=last))
    src, dst = [x[ok] for x in src], [x[ok] for x in dst]
    s["k"][:, dst[0], :, dst[1]] = s["k"][:, src[0], :, src[1]]
    s["v"][:, dst[0], :, :, dst[1]] = s["v"][:, src[0], :, :, src[1]]
    s["after"].copy_(s["lens"] + ok.sum(1))
    return s["k"], s["v"], s["after"]


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return (_own_append if op == "append" else _own_attend if op == "attend" else _own_keep)(state, case)
    return (_plain_append if op == "append" else _plain_attend if op == "attend" else _plain_keep)(state, case)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d, kv, page = case["d"], case["kv"], case["page"]
    table, lens = s["table"].long(), s["lens"].long()
    if case["op"] == "keep":
        # the slots of a whole sequence in order, taken once each before any is written
        k, v = s["k"].clone(), s["v"].clone()
        for i, row in enumerate(s["kept_lists"]):
            for j, node in enumerate(r for r in row if r >= 0):
                to, fr = s["held"][i] + j, s["held"][i] + node
                pt, pf = int(s["table"][i, to // page]), int(s["table"][i, fr // page])
                k[:, pt, :, to % page] = s["k"][:, pf, :, fr % page]
                v[:, pt, :, :, to % page] = s["v"][:, pf, :, :, fr % page]
        return k.double(), v.double(), _ints([c + sum(x >= 0 for x in r) for c, r in zip(s["held"], s["kept_lists"])])
    n, h = s["n"], case["heads"]
    if case["op"] == "append":
        slot = lens[s["row_seq"]] + s["row_new"]
        pos = s["positions"].double() if s["positions"] is not None else slot.double()
        rot = case["rot"]
        freq = torch.tensor([case["base"] ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=DEV)
        turn = torch.polar(torch.ones(n, rot // 2, dtype=torch.float64, device=DEV), pos[:, None] * freq)[:, None, :]

        def rows(x, heads, w):
            x = x.double().reshape(n, heads, d)
            if w is not None:
                x = x * torch.rsqrt(x.square().sum(2, keepdim=True) / d + 1e-6) * w.double()
            pair = x[..., :rot].reshape(n, heads, 2, rot // 2).transpose(2, 3) if case["neox"] else x[..., :rot].reshape(n, heads, rot // 2, 2)
            y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
            y = y.transpose(2, 3) if case["neox"] else y
            return torch.cat((y.reshape(n, heads, rot), x[..., rot:]), 2)

        k, v = s["k"].double(), s["v"].double()
        at = table[s["row_seq"], slot // page] * page + slot % page
        k = k.permute(0, 1, 3, 2, 4).reshape(-1, kv, d)
        k[at] = rows(s["kx"], kv, s.get("k_norm"))
        k = k.reshape(1, -1, page, kv, d).permute(0, 1, 3, 2, 4)
        v = v.permute(0, 1, 4, 2, 3).reshape(-1, kv, d)
        v[at] = s["vx"].double().reshape(n, kv, d)
        v = v.reshape(1, -1, page, kv, d).permute(0, 1, 3, 4, 2)
        return rows(s["q"], h, s.get("q_norm")).reshape(n, -1), k, v
    group, out, at = h // kv, torch.empty(n, h, d, dtype=torch.float64, device=DEV), 0
    parents = s["parents"].tolist() if s["parents"] is not None else None
    for i, (held, m) in enumerate(zip(s["held"], s["counts"])):
        if m == 0:
            continue
        slots = torch.arange(held + m, device=DEV)
        pid, off = table[i, slots // page], slots % page
        hidden = torch.ones(m, held + m, dtype=torch.bool)
        hidden[:, :held] = False
        for a in range(m):
            if parents is None:
                hidden[a, held:held + a + 1] = False
            else:
                node = a
                while node >= 0:
                    hidden[a, held + node] = False
                    node = parents[at + node]
        hidden = hidden.to(DEV)
        q = s["q"][at:at + m].double().reshape(m, h, d)
        for head in range(h):
            k = s["k"][0][pid, head // group, off].double()
            score = (q[:, head] @ k.T / math.sqrt(d)).masked_fill_(hidden, NEG)
            v = s["v"][0][pid, head // group, :, off].double()
            out[at:at + m, head] = torch.softmax(score, 1) @ v
        at += m
    return out.reshape(n, h * d)
