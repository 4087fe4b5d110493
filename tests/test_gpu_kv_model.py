"""A whole model over a paged cache (``GpuModel.extend``) against the same model's passes over whole sequences.

The two form the same rows by different kernels: the cache's rotation takes its angles in 64 bits where the step's tables are
f32, and so a key may round to the next f16 value (2^-11 of it, a score of unit size by that much at most); the
attention kernels sum in other orders.  Rows agree as the model's other paths do, within 1e-3 of the largest
logit (quantised weights, whose activation codes may move by one: 1e-2)."""
import numpy as np
import pytest

import oracle as O
import rust_trainer_amd as rt
from kv_cases import tree
from model_cases import adapters, sequence, tiny_spec
from rust_trainer_amd import gguf as G

pytestmark = pytest.mark.gpu
V = 256


def load(ctx, wtype=O.F32, lora=True, **kw):
    g = G.GgufFile.from_bytes(tiny_spec(wtype, n_vocab=V, **kw).build())
    m = rt.GpuModel.from_gguf(g, ctx=ctx)
    if lora:
        m.attach_lora(4, 8.0, seed=1)
        a = adapters(g, 4, 8.0, seed=11, b_std=0.05)
        for i in range(m.lora_count()):
            inf = m.lora_info(i)
            m.set_lora(i, *a[(inf["layer"], O.LINEARS[inf["which"]])])
    return m


def logits(te):
    """Whole rows of logits from lists of all tokens."""
    out = np.empty(te.vals.shape, np.float64)
    np.put_along_axis(out, te.ids, te.vals, 1)
    return out


def close(got, want, tol):
    assert got.shape == want.shape
    err = np.abs(got - want).max() / np.abs(want).max()
    assert err <= tol, err


def whole(m, toks, pos):
    return logits(m.top_logits(toks, pos, V))


@pytest.mark.parametrize("wtype, tol", [(O.F32, 1e-3), (O.Q8_0, 1e-2), (O.Q4_0, 1e-2)])
@pytest.mark.parametrize("kw", [dict(), dict(arch="llama"), dict(head_dim=128, rope_dim=128), dict(head_dim=48, rope_dim=32, n_head=3, n_head_kv=1), dict(n_layer=1)])
def test_extending_is_running_the_whole(ctx, wtype, tol, kw):
    m = load(ctx, wtype, **kw)
    toks, _, _ = sequence(V, 75, 5)
    want = whole(m, toks, np.arange(75))
    c = m.cache(4, 32)
    table = [[3, 0, 2]]
    got, at = [], 0
    for n in (40, 1, 1, 20, 1, 1, 1, 10):  # a prompt, tokens, pieces
        te = m.extend(c, rt.Seqs([at], table), toks[at:at + n], V)
        got.append(logits(te))
        at += n
    close(np.concatenate(got), want, tol)
    # the last row alone, as a decoder asks for it
    te = m.extend(c, rt.Seqs([65], table), toks[65:], V, positions=[9])
    close(logits(te), want[74:], tol)
    m.close()


def test_two_sequences_share_a_prompt_and_a_draft_is_kept(ctx):
    m = load(ctx)
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, V, 64)
    tails = [rng.integers(0, V, 5), rng.integers(0, V, 9)]
    c = m.cache(8, 32)
    m.extend(c, rt.Seqs([0], [[0, 1]]), prompt, 1, positions=[])
    # both read the prompt's two pages and write their own
    table = [[0, 1, 2, 4], [0, 1, 3, 5]]
    te = m.extend(c, rt.Seqs([64, 64], table, [0, 5, 14]), np.concatenate(tails), V)
    seqs = [np.concatenate((prompt, t)) for t in tails]
    want = np.concatenate([whole(m, s, np.arange(64, s.size)) for s in seqs])
    close(logits(te), want, 1e-3)
    # a drafted tree each: every node's row is that of its branch alone
    lens, nodes = [69, 73], 11
    trees = [tree(rng, nodes, deep=4)[0] for _ in range(2)]
    drafted = rng.integers(0, V, (2, nodes))
    te = m.extend(c, rt.Seqs(lens, table, [0, nodes, 2 * nodes]), drafted.ravel(), V, parents=np.concatenate(trees))
    got = logits(te).reshape(2, nodes, V)
    branches = []
    for i in range(2):
        for j in range(nodes):
            path, node = [], j
            while node >= 0:
                path.append(node)
                node = trees[i][node]
            branches.append(path[::-1])
            s = np.concatenate((seqs[i], drafted[i][path[::-1]]))
            close(got[i, j][None], whole(m, s, [s.size - 1]), 1e-3)
    # the longest branches are accepted, and the next token follows them
    kept = [max(branches[i * nodes:(i + 1) * nodes], key=len) for i in range(2)]
    lens = c.keep(rt.Seqs(lens, table), kept)
    nxt = rng.integers(0, V, 2)
    te = m.extend(c, rt.Seqs(lens, table), nxt, V)
    for i in range(2):
        s = np.concatenate((seqs[i], drafted[i][kept[i]], nxt[i:i + 1]))
        assert lens[i] == s.size - 1
        close(logits(te)[i][None], whole(m, s, [s.size - 1]), 1e-3)
    m.close()


def test_greedy_verification_of_a_tree_is_that_of_its_branch(ctx):
    """The tokens that follow a tree's nodes by their top logits are those that ``verify_draft`` accepts of the branch."""
    m = load(ctx)
    rng = np.random.default_rng(5)
    toks = rng.integers(0, V, 20)
    c = m.cache(2, 32)
    top = m.extend(c, rt.Seqs([0], [[1, 0]]), toks, 1).ids[-1, 0]
    # a tree of right and wrong guesses: the right one continues
    right = [int(top)]
    for _ in range(3):
        right.append(int(m.top_logits(np.concatenate((toks, right)), [19 + len(right)], 1).ids[0, 0]))
    draft = [(right[0] + 1) % V, right[0], right[1], (right[1] + 1) % V, right[2], (right[3] + 1) % V]
    parents = [-1, -1, 1, 1, 2, 4]
    te = m.extend(c, rt.Seqs([20], [[1, 0]]), draft, 1, parents=parents)
    node, accepted, path = -1, 0, []
    want = int(top)
    while True:
        nxt = [j for j in range(6) if parents[j] == node and draft[j] == want]
        if not nxt:
            break
        node, accepted = nxt[0], accepted + 1
        path.append(node)
        want = int(te.ids[node, 0])
    acc, out = m.verify_draft(np.concatenate((toks, [draft[1], draft[2], draft[4], draft[5]])), 4, temperature=0.0)
    assert (accepted, want) == (acc, int(out[acc])) == (3, right[3])
    assert c.keep(rt.Seqs([20], [[1, 0]]), [path])[0] == 23
    m.close()


def test_steps_of_one_shape_replay_a_graph(ctx):
    m = load(ctx)
    toks, pos, tok = sequence(V, 60, 8)
    targets = [rt.Target(int(a), int(b)) for a, b in zip(pos, tok)]
    m.zero_grad()
    lp, _ = m.forward_backward(toks, targets, np.ones(8))
    g = [m.lora(i)[2:] for i in range(m.lora_count())]
    want = whole(m, toks, np.arange(60))
    c, other = m.cache(2, 32), m.cache(2, 32)
    got = []
    before = m.graph_replays
    for i in range(60):
        got.append(logits(m.extend(c, rt.Seqs([i], [[1, 0]]), toks[i:i + 1], V)))
        if i % 7 == 6:  # another cache of the same shape in between, another table
            a = logits(m.extend(other, rt.Seqs([0], [[0, 1]]), toks[:1], V))
            close(a, want[:1], 1e-3)
    assert m.graph_replays > before + 20
    close(np.concatenate(got), want, 1e-3)
    # training after it is as before, to the bit
    for _ in range(2):
        m.zero_grad()
        lp2, _ = m.forward_backward(toks, targets, np.ones(8))
        assert np.array_equal(lp, lp2)
        assert all(np.array_equal(a, b) for i in range(m.lora_count()) for a, b in zip(m.lora(i)[2:], g[i]))
    m.close()


def test_refusals(ctx):
    m = load(ctx)
    c = m.cache(2, 32)
    ok = rt.Seqs([0], [[0, 1]])
    from rust_trainer_amd.kvcache import KvCache
    cfg = m.config
    wrong = [KvCache(cfg["n_layer"] + 1, 2, 32, cfg["n_head_kv"], cfg["head_dim"], ctx=ctx), KvCache(cfg["n_layer"], 2, 32, cfg["n_head_kv"] + 1, cfg["head_dim"], ctx=ctx),
             KvCache(cfg["n_layer"], 2, 32, cfg["n_head_kv"], cfg["head_dim"] + 16, ctx=ctx)]
    for w in wrong:
        with pytest.raises(rt.RtqError, match="model of"):
            m.extend(w, ok, [1, 2], 1)
    own = rt.Context(0)
    with pytest.raises(rt.RtqError, match="context"):
        m.extend(KvCache(cfg["n_layer"], 2, 32, cfg["n_head_kv"], cfg["head_dim"], ctx=own), ok, [1, 2], 1)
    own.close()
    for bad in (dict(tokens=[1, V]), dict(tokens=[-1]), dict(tokens=[]), dict(k=0), dict(k=257), dict(positions=[2]), dict(positions=[-1]), dict(temperature=0.0),
                dict(parents=[0, -1]), dict(parents=[-1, 1]), dict(seqs=rt.Seqs([63], [[0, 1]])), dict(seqs=rt.Seqs([-1], [[0, 1]])), dict(seqs=rt.Seqs([0], [[0, 2]], [0, 40])),
                dict(seqs=rt.Seqs([0], [[2, 1]])), dict(seqs=rt.Seqs([0, 0, 0], [[0], [1], [0]]))):
        a = dict(seqs=ok, tokens=[1, 2], k=1, positions=None, parents=None, temperature=1.0)
        a.update(bad)
        with pytest.raises(rt.RtqError):
            m.extend(c, a["seqs"], a["tokens"], a["k"], a["positions"], a["parents"], a["temperature"])
    m.extend(c, ok, [1, 2], 1)
    m.close()


def test_a_long_prompt_leaves_the_steps_their_size(ctx):
    """A head size without fused attention, whose steps hold [heads x t x t] probabilities: a prompt of 40000 tokens into a cache, and a
    step of 60 is what it was before, to the bit, in memory of a step of 60."""
    import torch

    m = load(ctx, head_dim=48, rope_dim=48)
    toks, pos, tok = sequence(V, 60, 8)
    targets = [rt.Target(int(a), int(b)) for a, b in zip(pos, tok)]

    def step():
        m.zero_grad()
        lp, _ = m.forward_backward(toks, targets, np.ones(8))
        return [lp] + [x for i in range(m.lora_count()) for x in m.lora(i)[2:]]

    want = step()
    rng = np.random.default_rng(0)
    c = m.cache(40, 1024)
    prompt = rng.integers(0, V, 40000)
    te = m.extend(c, rt.Seqs([0], [np.arange(40)]), prompt, 1, positions=[39999])
    assert np.isfinite(te.vals).all()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(2):
        assert all(np.array_equal(a, b) for a, b in zip(step(), want))
    assert torch.cuda.mem_get_info()[0] > free - (1 << 30)
    # the next token of the prompt, and a step again
    assert np.isfinite(m.extend(c, rt.Seqs([40000], [np.arange(40)]), [1], 1).vals).all()
    assert all(np.array_equal(a, b) for a, b in zip(step(), want))
    m.close()


@pytest.mark.parametrize("keep, fused, head_dim", [(False, False, 64), (True, True, 64), (False, None, 48)])
def test_an_extension_is_no_step(ctx, keep, fused, head_dim):
    """What the last step chose (activations kept, fused attention) is told after an extension as before it, and nothing before any step."""
    m = load(ctx, head_dim=head_dim, rope_dim=32)
    m.checkpointing, m.fused_attention = keep, fused
    c = m.cache(8, 32)
    m.extend(c, rt.Seqs([0], [np.arange(8)]), np.arange(100), 1)
    assert m.checkpointing is None and m.fused_attention is None
    toks, pos, tok = sequence(V, 60, 8)
    m.forward_backward(toks, [rt.Target(int(a), int(b)) for a, b in zip(pos, tok)], np.ones(8))
    want = m.checkpointing, m.fused_attention
    assert want == (keep, bool(fused))
    for at, n in ((100, 1), (101, 120)):
        m.extend(c, rt.Seqs([at], [np.arange(8)]), np.arange(n), 1)
        assert (m.checkpointing, m.fused_attention) == want
    m.close()


@pytest.mark.parametrize("longer", [90, 700])
def test_steps_after_prompts_of_any_length(ctx, longer):
    """Steps and prompts in turn, the prompts somewhat or much longer than the steps: each step is what it was, to the bit, and each prompt's last row the
    whole sequence's."""
    m = load(ctx, head_dim=64, n_layer=3)
    toks, pos, tok = sequence(V, 60, 8)
    targets = [rt.Target(int(a), int(b)) for a, b in zip(pos, tok)]
    prompt = np.random.default_rng(1).integers(0, V, longer)
    c = m.cache(22, 32)
    want = last = None
    for _ in range(3):
        m.zero_grad()
        lp, _ = m.forward_backward(toks, targets, np.ones(8))
        got = [lp] + [x for i in range(m.lora_count()) for x in m.lora(i)[2:]]
        want = want or got
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        te = logits(m.extend(c, rt.Seqs([0], [np.arange(22)]), prompt, V, positions=[longer - 1]))
        last = te if last is None else last
        assert np.array_equal(te, last)
    close(last, whole(m, prompt, [longer - 1]), 1e-3)
    m.close()
