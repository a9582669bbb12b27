"""The 8-bit KV cache in use: the lean forward, a captured verify pass and the
speculative loop over it, on a small target.

The comparisons hold a pass over the 8-bit cache against the same pass over a
bf16 cache that holds the values the codes stand for, so quantisation itself
cancels: what remains is each attention's rounding (at most 2^-8 |o| + 2^-8
max |v| a layer) carried through three layers; cosine 0.999 and 2 % of the norm
bound it with room."""
import pytest
import torch

from specfit_b200 import ops, synthetic
from specfit_b200.runtime import Kv8Cache
from specfit_b200.runtime.eagle3_drafter import build_random_drafter
from specfit_b200.runtime.kv_cache import ReservedCache, compact_tree_cache_
from specfit_b200.runtime.lean_forward import LeanQwen3Forward
from specfit_b200.runtime.qwen3_verifier import build_random_offloaded_qwen3, qwen3_moe_config
from specfit_b200.runtime.speculator import B200TreeSpeculator, BernoulliAcceptance
from specfit_b200.runtime.verify_graph import VerifyGraph
from specfit_b200.selection import SelectionCostModel

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
PARENTS = (0, 0, 1, 1, 2, 4, 5)  # a verification tree of the seed and seven nodes


@pytest.fixture(scope="module")
def target():
    cfg = qwen3_moe_config(3, hidden=256, experts=16, top_k=4, moe_inter=128, heads=8, kv_heads=2, head_dim=128,
                           vocab=512)
    m = build_random_offloaded_qwen3(device=DEV, slots_per_layer=16, config=cfg, seed=6, std=0.05)
    m.warm_all_caches()
    # One route per token whatever the hidden state: a near tie in the router
    # would turn a rounding into another expert.
    hooks = []
    state = {"ids": None}
    for l, layer in enumerate(m.model.model.layers):
        def route(mod, args, out, l=l):
            if state["ids"] is None:
                return None
            return out[0], out[1], synthetic.token_routes(state["ids"].reshape(-1), 3, experts=16, top_k=4)[:, l, :]
        hooks.append(layer.mlp.gate.register_forward_hook(route))
    yield cfg, m, state
    for h in hooks:
        h.remove()
    m.close()


def tree_inputs(batch, base, seed):
    q = len(PARENTS) + 1
    ids = torch.randint(0, 512, (batch, q), generator=torch.Generator().manual_seed(seed)).to(DEV)
    mask = torch.zeros(batch, 1, q, base + q, dtype=torch.bool, device=DEV)
    mask[..., :base] = True
    depth = [0]
    for i in range(q):
        if i:
            mask[:, :, i, base:] = mask[:, :, PARENTS[i - 1], base:]
            depth.append(depth[PARENTS[i - 1]] + 1)
        mask[:, :, i, base + i] = True
    pos = (base + torch.tensor(depth, device=DEV)).expand(batch, q)
    return ids, mask, pos


def near(a, b):
    a, b = a.double().flatten(), b.double().flatten()
    cos = float(a @ b / (a.norm() * b.norm()))
    assert cos >= 0.999 and float((a - b).norm() / b.norm()) <= 2e-2, (cos, float((a - b).norm() / b.norm()))


def run(fwd, state, cache, ids, **kw):
    state["ids"] = ids
    try:
        return fwd(input_ids=ids, past_key_values=cache, use_cache=True, **kw).logits.float()
    finally:
        state["ids"] = None


@pytest.mark.parametrize("batch,ctx,block", [(1, 150, 64), (2, 97, 32), (1, 20, 128)])
def test_lean_forward_over_the_8_bit_cache(target, batch, ctx, block):
    cfg, m, state = target
    fwd = LeanQwen3Forward(m.model)
    ids = torch.randint(0, 512, (batch, ctx), generator=torch.Generator().manual_seed(ctx)).to(DEV)
    small = Kv8Cache(config=cfg, capacity=ctx + 64, block=block, tail_room=16)
    plain = ReservedCache(config=cfg, capacity=ctx + 64)
    near(run(fwd, state, small, ids), run(fwd, state, plain, ids))  # a prompt attends to its own bf16 rows
    assert all(l.sealed == ctx // block * block for l in small.layers)
    for a, b in zip(small.layers, plain.layers):
        k, v = ops.kv8_read(a.rows())
        b._kbuf[:, :, :ctx].copy_(k)
        b._vbuf[:, :, :ctx].copy_(v)
    for step in range(3):  # a tree, its accepted path kept, one more token, and so on
        base = small.get_seq_length()
        tids, mask, pos = tree_inputs(batch, base, step)
        near(run(fwd, state, small, tids, attention_mask=mask, position_ids=pos),
             run(fwd, state, plain, tids, attention_mask=mask, position_ids=pos))
        if batch == 1:
            for c in (small, plain):
                compact_tree_cache_(c, base_kv_length=base, verification_positions=(0, 1, 4),
                                    verification_node_count=8)
        else:
            small.crop(base + 1)
            plain.crop(base + 1)
        one = torch.full((batch, 1), 7 + step, device=DEV)
        near(run(fwd, state, small, one), run(fwd, state, plain, one))
        assert small.get_seq_length() == plain.get_seq_length()


def test_a_captured_verify_pass_replays_over_the_8_bit_cache(target):
    cfg, m, state = target
    fwd = LeanQwen3Forward(m.model)
    ids = torch.randint(0, 512, (1, 100), generator=torch.Generator().manual_seed(3)).to(DEV)
    cache = Kv8Cache(config=cfg, capacity=256, tail_room=16)
    fwd(input_ids=ids, past_key_values=cache, use_cache=True)
    inputs = [tree_inputs(1, 100, s) for s in (1, 2)]
    want = []
    for i in inputs:
        want.append(fwd(input_ids=i[0], attention_mask=i[1], position_ids=i[2], past_key_values=cache,
                        use_cache=True).logits.clone())
        cache.crop(100)
    g = VerifyGraph(m.model, cache, q_len=8, device=DEV, forward=fwd)
    g.capture(*inputs[0])
    for k in (0, 1, 0):
        g.load(*inputs[k])
        g.replay()
        assert torch.equal(g.logits, want[k])
    assert cache.get_seq_length() == 100
    g.graph = None
    with pytest.raises(RuntimeError, match="tail_room"):
        VerifyGraph(m.model, cache, q_len=17, device=DEV, forward=fwd).capture(
            torch.zeros(1, 17, dtype=torch.long, device=DEV), torch.ones(1, 1, 17, 117, dtype=torch.bool, device=DEV),
            torch.zeros(1, 17, dtype=torch.long, device=DEV))
    with pytest.raises(RuntimeError, match="scores"):
        VerifyGraph(m.model, Kv8Cache(config=cfg, capacity=64, budget=32, recent=8), q_len=8, device=DEV, forward=fwd)


def test_weights_add_up_and_eviction_keeps_the_pass_going(target):
    cfg, m, state = target
    fwd = LeanQwen3Forward(m.model)
    ids = torch.randint(0, 512, (1, 200), generator=torch.Generator().manual_seed(5)).to(DEV)
    cache = Kv8Cache(config=cfg, capacity=256, budget=96, sinks=4, recent=16)
    run(fwd, state, cache, ids)
    for l in cache.layers:  # four query heads a KV head, 200 rows of weight 1 each
        total = l.mass[:, :, :200].double().sum(-1)
        assert float((total - 4 * 200).abs().max()) <= 4 * 200 * 1e-3
        assert float(l.mass[:, :, 200:].abs().max()) == 0
    keep = [ops.kv_keep_heaviest(l.mass, 200, 96, sinks=4, recent=16) for l in cache.layers]
    rows = [ops.kv8_read(l.rows()) for l in cache.layers]
    assert cache.evict() == 104 and cache.get_seq_length() == 96 and cache.next_position == 200
    for l, kp, (k, v) in zip(cache.layers, keep, rows):
        at = kp.long().unsqueeze(-1).expand(-1, -1, -1, 128)
        nk, nv = ops.kv8_read(l.rows())
        full = l.sealed
        assert torch.equal(nk[:, :, full:], k.gather(2, at)[:, :, full:])
        for new, old in ((nk, k), (nv, v)):  # rows sealed for the first time are rounded to e4m3: half a step
            o = old.gather(2, at)[:, :, :full].float()
            least = 2.0 ** -10 * float(max(l._codes[2][:, :, : full // 64].max(), l._codes[3][:, :, : full // 64].max()))
            assert bool(((new[:, :, :full].float() - o).abs() <= 2.0 ** -4 * o.abs() + least).all())
    # The same token over a bf16 cache that holds the kept rows.
    plain = ReservedCache(config=cfg, capacity=128)
    run(fwd, state, plain, ids[:, :96])
    for a, b in zip(cache.layers, plain.layers):
        k, v = ops.kv8_read(a.rows())
        b._kbuf[:, :, :96].copy_(k)
        b._vbuf[:, :, :96].copy_(v)
    one = torch.full((1, 1), 9, device=DEV)
    pos = torch.full((1, 1), 200, device=DEV)
    near(run(fwd, state, cache, one), run(fwd, state, plain, one, position_ids=pos))


@pytest.mark.parametrize("budget", [None, 40])
def test_speculative_decoding_over_the_8_bit_cache(target, budget):
    import specfit_b200.runtime.speculator as sp

    cfg, m, state = target
    d = build_random_drafter(m.model, seed=9, std=0.05, inter=512, aux_layers=(0, 1, 2))
    cost = SelectionCostModel(synthetic.SELECTION_SIZE_MEAN_NS, synthetic.SELECTION_INTERCEPT_NS,
                              synthetic.SELECTION_EXPERT_NS)
    spec = B200TreeSpeculator(m, d, cost_model=cost, acceptance=BernoulliAcceptance(3), lean=True, kv8=True,
                              kv8_budget=budget)
    ctx = torch.randint(0, 512, (1, 70), generator=torch.Generator().manual_seed(2)).to(DEV)
    seen = []
    real = sp.compact_tree_cache_

    def spy(cache, **kw):
        real(cache, **kw)
        seen.append((cache, cache.get_seq_length(), cache.next_position))
    sp.compact_tree_cache_ = spy
    try:
        res = spec.generate(ctx, 30)
    finally:
        sp.compact_tree_cache_ = real
    assert res.committed == 30 and all(0 <= t < 512 for t in res.tokens)
    cache = seen[-1][0]
    assert isinstance(cache, Kv8Cache)
    assert 70 < cache.next_position <= 100
    positions = [s[2] for s in seen]
    assert positions == sorted(set(positions))  # every cycle commits at least the seed, none is counted twice
    if budget is None:
        assert cache.dropped == 0 and cache.get_seq_length() == cache.next_position
    else:
        assert cache.get_seq_length() == budget and max(s[1] for s in seen[1:]) <= budget + 8


def test_a_replay_over_replaced_buffers_is_refused(target):
    cfg, m, state = target
    fwd = LeanQwen3Forward(m.model)
    ids = torch.randint(0, 512, (1, 100), generator=torch.Generator().manual_seed(3)).to(DEV)
    cache = Kv8Cache(config=cfg, capacity=256, tail_room=16)
    fwd(input_ids=ids, past_key_values=cache, use_cache=True)
    inputs = tree_inputs(1, 100, 1)
    g = VerifyGraph(m.model, cache, q_len=8, device=DEV, forward=fwd)
    g.capture(*inputs)
    want = g.replay().clone()
    run(fwd, state, cache, ids[:, :70])  # wider than the tail
    cache.crop(100)
    with pytest.raises(RuntimeError, match="laid out"):
        g.replay()
    run(fwd, state, cache, ids[:, :1])
    with pytest.raises(RuntimeError, match="laid out"):
        g.replay()
    cache.crop(100)
    run(fwd, state, cache, ids[:, :1])  # the tail is the usual one again
    cache.crop(100)
    again = VerifyGraph(m.model, cache, q_len=8, device=DEV, forward=fwd)
    again.capture(*inputs)
    assert torch.equal(again.replay(), want)
    run(fwd, state, cache, ids[:, :5])  # rows that the replay writes over
    assert torch.equal(again.replay(), want)


@pytest.mark.parametrize("budget", [None, 96])
def test_a_long_pass_goes_through_in_parts(target, monkeypatch, budget):
    """A causal pass and a masked one, whole and in parts of 48 rows."""
    import specfit_b200.runtime.lean_forward as lf

    cfg, m, state = target
    fwd = LeanQwen3Forward(m.model)
    ids = torch.randint(0, 512, (2, 170), generator=torch.Generator().manual_seed(8)).to(DEV)
    outs, weights = [], []
    for rows in (lf.KV8_ROWS, 48):
        monkeypatch.setattr(lf, "KV8_ROWS", rows)
        cache = Kv8Cache(config=cfg, capacity=512, budget=budget, recent=16)
        got = [run(fwd, state, cache, ids), run(fwd, state, cache, ids[:, :101])]
        total = 170 + 101 + 60
        mask = torch.ones(2, 1, 60, total, dtype=torch.bool, device=DEV)
        mask[:, :, :, 271:] = torch.ones(60, 60, dtype=torch.bool, device=DEV).tril()
        pos = torch.arange(271, 331, device=DEV).expand(2, 60)
        got.append(run(fwd, state, cache, ids[:, :60], attention_mask=mask, position_ids=pos))
        outs.append(got)
        if budget:
            weights.append([l.mass[:, :, :total].double() for l in cache.layers])
    for a, b in zip(*outs):
        near(a, b)
    if budget:
        # Every row's weights sum to one; layer 0 sees the same inputs both times.
        for w in weights:
            assert all(float((x.sum(-1) - 4 * 331).abs().max()) <= 4 * 331 * 1e-3 for x in w)
        assert bool(((weights[0][0] - weights[1][0]).abs() <= 1e-3 * weights[0][0] + 1e-3).all())


def test_batches_grow_shrink_and_change_order(target):
    cfg, m, state = target
    fwd = LeanQwen3Forward(m.model)
    ids = torch.randint(0, 512, (2, 90), generator=torch.Generator().manual_seed(4)).to(DEV)
    cache = Kv8Cache(config=cfg, capacity=256, budget=64, recent=16)
    run(fwd, state, cache, ids)
    before = [(ops.kv8_read(l.rows()), l.mass.clone()) for l in cache.layers]
    cache.batch_repeat_interleave(3)
    cache.reorder_cache(torch.tensor([5, 0, 2], device=DEV))  # requests 1, 0, 0
    cache.batch_select_indices(torch.tensor([0, 1], device=DEV))
    for l, ((k, v), mass) in zip(cache.layers, before):
        nk, nv = ops.kv8_read(l.rows())
        assert torch.equal(nk, k.flip(0)) and torch.equal(nv, v.flip(0)) and torch.equal(l.mass, mass.flip(0))
    one = torch.tensor([[3], [4]], device=DEV)
    flipped = run(fwd, state, cache, one.flip(0))
    again = Kv8Cache(config=cfg, capacity=256, budget=64, recent=16)
    run(fwd, state, again, ids)
    near(flipped.flip(0), run(fwd, state, again, one))
