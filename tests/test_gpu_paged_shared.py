"""PagedKV.attend over a plan of shared pages against the plain 64-bit form (oracle/paged_kv.py).

Tolerance, as for attend (test_gpu_paged.py), with A = sum_j p_j |v_j|, S = scale * sum |q k|, u half a step of the output type, and:
  * a component of q, as two (fp16: three) e4m3 parts of a row scaled to [128, 256), ends at the parts' smallest step, 2^-9: off by at most 2^-10 /
    2^7 = 2^-17 of its row's largest where its own bits do not end before: a score by E = 2^-17 scale max|q| max_j sum|k_j|;
  * a weight of (largest in its tile = 256) is rounded to fp16 (2^-11) and to two parts (2^-9) or three (2^-14), and ends at 2^-10 / 2^8 = 2^-18 of
    the tile's largest: over 128 tokens 2^-11 max|v| at most, for all tiles together, as their largest weights add up to one at most.
So |o - o*| <= (u + w + 2^-12 S + 2 E + 2^-18) A + 2^-11 max|v| with w = 2^-9 + 2^-11 (fp16: 2^-11 + 2^-14), and |lse - lse*| <= 2^-13 S + E +
2^-16 (1 + |lse*|).  The term 2^-11 max|v| is a bound on what 128 roundings of one sign could do; that they do not add up so is the second check: the
error's 2-norm stays below (u + w) of A's.  (Not of the output's: every term of the first bound is in units of A, and where a value of -1 of weight 0.503
stands against thousands of +1, u |o| + w A with |o| = 0.007 and A = 1 is 0.0025, 60 times (u + w) |o|.)"""
import random

import pytest
import torch

from oracle import paged_kv as opk
from test_gpu_paged import D, U, _cache, _fill, _host, _poison, _rand

pytestmark = pytest.mark.gpu
W = {torch.bfloat16: 2.0 ** -9 + 2.0 ** -11, torch.float16: 2.0 ** -11 + 2.0 ** -14}


def _check(c, plan, q, scale=None, layer=0, norm=True):
    o, lse = c.attend(layer, q.cuda(), scale=scale, with_lse=True, shared=plan)
    _check_out(c, plan, q, o, lse, scale, layer, norm)
    return o


def _check_out(c, plan, q, o, lse, scale=None, layer=0, norm=True):
    o, lse, u, w = o.cpu(), lse.cpu().double(), U[q.dtype], W[q.dtype]
    assert o.dtype == q.dtype and torch.isfinite(o).all()
    kc, ks, vc, vs = _host(c, layer)
    sc = D ** -0.5 if scale is None else scale
    longest = float((kc.nan_to_num().abs().sum(-1).amax(-1) * ks.nan_to_num()).max())
    err, size, done = 0.0, 0.0, {}
    for b, slot in enumerate(plan.slots):
        if slot not in done:
            done[slot] = c.table[slot].tolist(), int(c.lens[slot])
        row, n = done[slot]
        ro, rl, mag, big = opk.attend(kc, ks, vc, vs, row, n, q[b], scale)
        top = float((vc.nan_to_num().abs().amax((2, 3)) * vs.nan_to_num()).max())
        E = 2.0 ** -17 * sc * q[b].double().abs().amax(-1) * longest
        tol = (u + w + 2.0 ** -12 * big[..., None] + 2 * E[..., None] + 2.0 ** -18) * mag + 2.0 ** -11 * top * (mag > 0)
        off = (o[b].double() - ro).abs()
        assert (off <= tol).all(), (b, (off - tol).max())
        err, size = err + float((off ** 2).sum()), size + float((mag ** 2).sum())
        dead = rl == -float("inf")
        assert (lse[b][dead] == -float("inf")).all() and (o[b].transpose(0, 1)[dead] == 0).all()
        off = (lse[b] - rl).abs()[~dead]
        assert (off <= (2.0 ** -13 * big.T + E.T + 2.0 ** -16 * (1 + rl.abs()))[~dead]).all(), (b, off.max())
    assert not norm or err ** 0.5 <= (u + w) * size ** 0.5


def _tree(page, common, docs, ways, tails, G=1, layers=1, spare=0, poison=True):
    """A common prompt, documents behind it, sequences behind each of them; the slots of the sequences."""
    n, nd = sum(ways), len(docs)
    pages = -(-common // page) + sum(-(-(d + page) // page) for d in docs) + sum(-(-(x + page) // page) for x in tails) + 2 + spare
    c = _cache(layers, pages, G, n + nd + 1, page=page, max_len=common + max(docs) + max(tails) + page)
    root, mid, leaves = n, list(range(n + 1, n + 1 + nd)), list(range(n))
    c.reserve([root], common)
    c.fork([root] * nd, mid)
    c.free([root])
    c.reserve(mid, docs)
    c.fork([m for m, w in zip(mid, ways) for _ in range(w)], leaves)
    c.free(mid)
    c.reserve(leaves, tails)
    _fill(c, common)
    if poison:
        _poison(c)
    return c, leaves


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("H,G,t,dtype", [(24, 4, 1, torch.bfloat16), (6, 1, 3, torch.float16), (2, 2, 1, torch.float16), (8, 1, 2, torch.bfloat16),
                                         (24, 1, 1, torch.bfloat16), (5, 1, 5, torch.bfloat16)])
def test_one_prompt_many_sequences(page, H, G, t, dtype):
    tails = [t + (37 * i) % 150 for i in range(9)]
    c, slots = _tree(page, 700, [0], [9], tails, G)
    plan = c.share(slots, min_saved=1)
    assert plan.runs == 1 and plan.slots == slots
    _check(c, plan, _rand(9, t, H, D, dtype=dtype))


@pytest.mark.parametrize("common", [64, 128, 192, 1000, 2311])
def test_lengths_of_shared_runs(common):
    """Runs of one page, of one tile, that end inside a tile, and tails of one token."""
    c, slots = _tree(64, common, [0], [2], [1, 1])
    _check(c, c.share(slots, min_saved=1), _rand(2, 1, 4, D, seed=2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tree_of_prompts_and_slots_in_any_order(dtype):
    c, slots = _tree(32, 333, [500, 0, 64, 1700, 31], [3, 1, 4, 2, 5], [1 + (53 * i) % 200 for i in range(15)], 2, layers=2)
    order = [slots[(7 * i) % 15] for i in range(15)] + [slots[3], slots[3]]        # a slot three times: even its partial page's tokens are its own
    plan = c.share(order, min_saved=1)
    assert plan.runs > 4
    q = _rand(17, 1, 12, D, seed=3, dtype=dtype)
    o = _check(c, plan, q, layer=1)
    _check(c, plan, q, scale=0.3)
    few = c.share(order, min_saved=1500)
    assert 0 < few.runs < plan.runs
    assert (_check(c, few, q, layer=1).double() - o.double()).abs().max() < 0.05
    none = c.share(order, min_saved=10 ** 9)
    assert none.runs == 0
    ids = torch.tensor(order, device="cuda")
    assert torch.equal(c.attend(1, q.cuda(), shared=none)[0], c.attend(1, q.cuda(), ids)[0])


def test_many_rows_and_many_runs():
    """More than 128 rows of one run (several row blocks), more runs than a warp has lanes, and sequences that share nothing among them."""
    c, slots = _tree(16, 90, [16 * (1 + i % 3) for i in range(40)], [2] * 38 + [60, 1], [3 + i % 20 for i in range(137)])
    plan = c.share(slots, min_saved=1)
    assert plan.runs > 32
    _check(c, plan, _rand(137, 3, 6, D, seed=5))


def test_deep_chain_of_forks():
    """A sequence forked again and again: four runs to a sequence at most, the rest in the tails."""
    c = _cache(1, 200, 1, 12, page=16, max_len=1024)
    c.reserve([0], 50)
    for i in range(1, 10):
        c.fork([i - 1], [i])
        c.reserve([i], 33)
        c.reserve([i - 1], 5)
    _fill(c, 6)
    _poison(c)
    plan = c.share(range(10), min_saved=1)
    assert plan.runs >= 4
    _check(c, plan, _rand(10, 1, 4, D, seed=6))


def test_newest_tokens_inside_shared_pages():
    """Forks that have nothing of their own yet: the tokens of the call lie in the shared pages, each sees up to its own position."""
    for t in (1, 5, 64, 200):
        c, slots = _tree(64, 384, [0], [3], [0, 0, 2], poison=False)
        _check(c, c.share(slots, min_saved=1), _rand(3, t, 4, D, seed=t))


def test_tokens_before_the_first_position():
    """More tokens than a sequence has: those see nothing."""
    c, slots = _tree(16, 32, [0], [2], [0, 1], poison=False)
    o, lse = c.attend(0, _rand(2, 40, 2, D, seed=8).cuda(), shared=c.share(slots, min_saved=1), with_lse=True)
    assert (o[0, :8] == 0).all() and (lse[0, :, :8] == -float("inf")).all() and lse[0, :, 8:].isfinite().all()
    assert (o[1, :7] == 0).all() and lse[1, :, 7:].isfinite().all()


def test_long_prompt_over_all_ctas():
    c, slots = _tree(128, 30000, [0], [3], [1, 200, 17], 2)
    _check(c, c.share(slots), _rand(3, 1, 16, D, seed=9))


def test_one_heavy_key_among_many():
    """A weight near one beside thousands near 2^-13, in another tile and in its own: their sum counts."""
    c = _cache(1, 70, 1, 3, page=128, max_len=8192)
    c.reserve([0], 8000)
    k = torch.zeros(8000, 1, D)
    k[17, 0, :16] = 9.0
    v = torch.ones(8000, 1, D)
    v[17] = -1.0
    c.append(0, k.to(torch.bfloat16).cuda()[None], v.to(torch.bfloat16).cuda()[None])
    c.fork([0, 0], [1, 2])
    q = torch.zeros(3, 1, 1, D)
    q[..., :16] = 1.0
    _check(c, c.share([0, 1, 2]), q.to(torch.bfloat16))


def test_scales_far_apart():
    """V scales up to 2^24 apart, the weight on the small ones and on the large ones."""
    c, slots = _tree(16, 250, [0], [3], [3, 20, 1], poison=False)
    P = c.v_scale.shape[1]
    c.v_scale.copy_(torch.ldexp(torch.ones(P), torch.arange(P) % 5 * 6 - 20)[None, :, None])
    c.k_scale.copy_(torch.ldexp(torch.ones(P), torch.arange(P) % 3 * 2 - 9)[None, :, None])
    _poison(c)
    _check(c, c.share(slots, min_saved=1), _rand(3, 1, 4, D, seed=7))
    # all of the weight on a page of small values, whole tiles of large ones around it: its relative error is that of a sequence of its own
    c, slots = _tree(128, 512, [0], [2], [1, 1], poison=False)
    c.k_pages.copy_(torch.zeros(c.k_pages.shape).to(torch.float8_e4m3fn))
    c.k_pages[0, 1, 0, 7] = 200 * torch.ones(D)
    c.k_scale.fill_(1)
    c.v_scale.fill_(2.0 ** 12)
    c.v_scale[0, 1] = 2.0 ** -12
    q = torch.full((2, 1, 1, D), 0.25).bfloat16()
    o = c.attend(0, q.cuda(), shared=c.share(slots, min_saved=1))[0]
    want = c.v_pages[0, 1, 0, 7].double() * 2.0 ** -12
    assert ((o.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -9 + 2.0 ** -11) * want.abs() + 2.0 ** -30).all()


def test_rows_of_a_wide_range():
    """A row with one component 2^12 times the others: what its parts hold of them."""
    c, slots = _tree(32, 200, [0], [4], [1, 2, 3, 4], poison=False)
    c.k_pages[..., 5] = torch.zeros(()).to(torch.float8_e4m3fn).cuda()
    q = _rand(4, 1, 3, D, seed=11, dtype=torch.float16)
    q[:, :, 1, 5] = 2.0 ** 12
    q[:, :, 2] *= 2.0 ** -14
    # (E is not small here: 2^-17 * 2^12 / 16 * sum|k| of about 200 is 0.4, so the second check, which has no E, says nothing)
    _check(c, c.share(slots, min_saved=1), q, norm=False)


def test_values_that_are_not_finite():
    c, slots = _tree(16, 160, [0], [3], [4, 4, 4], poison=False)
    plan = c.share(slots, min_saved=1)
    q = _rand(3, 2, 4, D, seed=8)
    clean = c.attend(0, q.cuda(), shared=plan)[0]
    q[1, 0, 2, 9], q[2, 1, 1, 3] = float("inf"), float("nan")
    o = c.attend(0, q.cuda(), shared=plan)[0]
    bad = torch.zeros(3, 2, 4, dtype=torch.bool)
    bad[1, 0, 2] = bad[2, 1, 1] = True
    assert torch.equal(o.isnan().all(-1).cpu(), bad) and torch.equal(o[~bad.cuda()], clean[~bad.cuda()])
    q = _rand(3, 2, 4, D, seed=8).cuda()
    nan = torch.full((1,), float("nan")).to(torch.float8_e4m3fn).cuda()
    page = int(c.table[0, 3])
    c.v_pages[0, page, 0, 5, 7] = nan
    o = c.attend(0, q, shared=plan)[0]
    assert o[..., 7].isnan().all() and torch.equal(o[..., :7], clean[..., :7])
    c.v_pages[0, page, 0, 5, 7] = torch.zeros((), device="cuda").to(torch.float8_e4m3fn)
    own = int(c.table[1, 10])
    c.k_pages[0, own, 0, 1, 7] = nan               # a token of one sequence alone
    o = c.attend(0, q, shared=plan)[0]
    assert o[1].isnan().all() and o[0].isfinite().all() and o[2].isfinite().all()


def test_plans_after_changes():
    c, slots = _tree(32, 300, [64, 100], [3, 3], [1] * 6, spare=40)
    q = _rand(6, 1, 4, D, seed=12)
    plan = c.share(slots, min_saved=1)
    c.reserve(slots, 40)                           # growing leaves it good
    _fill(c, 3)
    _poison(c)
    _check(c, plan, q)
    c.compact()
    _check(c, plan, q)
    c.truncate([slots[0]], [10])
    with pytest.raises(ValueError, match="share again"):
        c.attend(0, q.cuda(), shared=plan)
    assert c.share(slots, plan, 1) is plan
    _check(c, plan, q)
    c.free([slots[1]])
    with pytest.raises(ValueError, match="share again"):
        c.attend(0, q.cuda(), shared=plan)
    c.share(slots, into=plan, min_saved=1)         # an ended sequence among them: zeros
    o, lse = c.attend(0, q.cuda(), shared=plan, with_lse=True)
    assert not o[1].any() and (lse[1] == -float("inf")).all()
    _check(c, plan, q)


def test_captured_and_replayed_with_a_new_plan():
    c, slots = _tree(64, 1000, [0], [4], [3, 9, 1, 2], spare=10)
    q = _rand(4, 1, 8, D, seed=13).cuda()
    plan = c.share(slots, min_saved=1)
    c.attend(0, q, shared=plan)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = c.attend(0, q, shared=plan, with_lse=True)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            c.share(slots)
    other = torch.cuda.Stream()
    for step in range(3):
        c.reserve(slots, 1)
        _fill(c, 20 + step)
        _poison(c)
        q.copy_(_rand(4, 1, 8, D, seed=20 + step))
        if step == 2:                              # other sequences in the same slots
            c.free([slots[0]])
            c.reserve([slots[0]], 77)
            c.share(slots, into=plan, min_saved=1)
            _fill(c, 30)
            _poison(c)
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(other):             # and another call at the same time
            o2 = c.attend(0, q, shared=plan)[0]
        torch.cuda.synchronize()
        assert torch.equal(o, o2)
        _check_out(c, plan, q.cpu(), o, lse)


def test_replayed_with_a_plan_that_has_no_runs():
    """And with one that is no longer good: what the pages then hold is not the sequences', but the replay ends and the others are right."""
    c, slots = _tree(64, 1000, [0], [4], [3, 9, 1, 2], spare=10)
    q = _rand(4, 1, 8, D, seed=13).cuda()
    plan, none = c.share(slots, min_saved=1), c.share(slots)
    assert plan.runs == 1 and none.runs == 0
    for p in (plan, none):
        c.attend(0, q, shared=p)
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = c.attend(0, q, shared=plan, with_lse=True)
    with torch.cuda.graph(h):
        o2, lse2 = c.attend(0, q, shared=none, with_lse=True)
    c.share(slots, plan)
    c.share(slots[::-1], none, min_saved=1)
    assert plan.runs == 0 and none.runs == 1
    g.replay()
    h.replay()
    torch.cuda.synchronize()
    _check_out(c, plan, q.cpu(), o, lse)
    _check_out(c, none, q.cpu(), o2, lse2)
    c.share(slots, plan, min_saved=1)
    c.free([slots[1]])
    assert not plan.good
    g.replay()
    torch.cuda.synchronize()
    assert not o[1].any() and (lse[1] == -float("inf")).all()
    plan.slots[1] = plan.slots[0]
    o[1], lse[1], q[1] = o[0], lse[0], q[0]
    _check_out(c, plan, q.cpu(), o, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_same_bits_again_and_again(dtype):
    """Ends of tiles, where what the pages hold behind a sequence (NaN here) is blotted out while the values of the tile before may still be on their way."""
    rng = random.Random(7)
    for tree in range(60):
        page, G, R, t = rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4]), rng.choice([1, 2, 6, 8, 24]), rng.choice([1, 1, 1, 2, 5])
        docs = [rng.choice([0, page, rng.randint(0, 600)]) for _ in range(rng.randint(1, 4))]
        ways = [rng.randint(1, 9) for _ in docs]
        c, slots = _tree(page, rng.choice([page, rng.randint(page, 1500)]), docs, ways, [rng.randint(0, 300) for _ in range(sum(ways))], G)
        plan = c.share(slots, min_saved=1)
        q = _rand(len(slots), t, G * R, D, seed=tree, dtype=dtype)
        if not plan.runs:
            continue
        calls = [c.attend(0, q.cuda(), shared=plan, with_lse=True) for _ in range(24)]
        for o, lse in calls:
            assert torch.equal(o, calls[0][0]) and torch.equal(lse, calls[0][1]), tree
        if tree % 10 == 0:
            _check_out(c, plan, q, *calls[0])


@pytest.mark.parametrize("page,common,docs,ways,R,t,tails,slots", [
    (32, 1095, [159, 441, 0], [3, 9, 9], 24, 5, [3, 181, 105, 175, 10, 2, 190, 3, 3, 103, 0, 231, 3, 0, 2, 42, 0, 2, 3, 3, 3],
     [16, 11, 5, 8, 14, 2, 13, 12, 6, 7, 1, 17, 10, 15, 4, 19, 3, 0, 18, 20, 9]),
    (128, 128, [232, 128, 215, 358], [6, 9, 3, 8], 1, 1,
     [0, 1, 111, 171, 0, 3, 83, 129, 0, 276, 1, 288, 12, 2, 2, 2, 0, 245, 1, 260, 5, 0, 2, 38, 51, 2],
     [14, 11, 5, 16, 0, 19, 21, 4, 6, 3, 7, 10, 12, 15, 2, 8, 25, 13, 9, 22, 23, 17, 20, 18, 24, 1])])
def test_values_of_the_tile_before_on_their_way(page, common, docs, ways, R, t, tails, slots):
    """Two batches whose last tiles were blotted out too early (the values behind a sequence came after it) in one call of some tens."""
    c, _ = _tree(page, common, docs, ways, tails, 4)
    plan = c.share(slots, min_saved=100)
    q = _rand(len(slots), t, 4 * R, D, dtype=torch.float16)
    calls = []
    for _ in range(300):
        calls = calls[:1] + [c.attend(0, q.cuda(), shared=plan, with_lse=True)]
        assert torch.equal(calls[-1][0], calls[0][0]) and torch.equal(calls[-1][1], calls[0][1])
    _check_out(c, plan, q, *calls[0])


def test_refused_calls():
    c, slots = _tree(16, 100, [0], [3], [1, 1, 1])
    other, _ = _tree(16, 100, [0], [3], [1, 1, 1])
    plan = c.share(slots, min_saved=1)
    q = _rand(3, 1, 4, D).cuda()
    for bad in (lambda: c.attend(0, q[:2], shared=plan), lambda: other.attend(0, q, shared=plan), lambda: c.attend(0, q, shared=slots),
                lambda: c.attend(0, q, torch.zeros(3, dtype=torch.int32, device="cuda"), shared=plan), lambda: c.share([]),
                lambda: c.share([99]), lambda: c.share(slots, min_saved=0), lambda: c.share(slots[:2], into=plan),
                lambda: other.share(slots, into=plan), lambda: c.share([0.5])):
        with pytest.raises(ValueError):
            bad()
    assert c.attend(0, q[:, :0], shared=plan)[0].shape == (3, 0, 4, D)


@pytest.mark.parametrize("t,dtype", [(1, torch.bfloat16), (3, torch.float16)])
def test_scores_below_what_fp32_holds(t, dtype):
    """Scales and queries so small that every score is 0: what a row does not see still has no weight, and all the others are alike."""
    c, slots = _tree(32, 200, [0], [3], [t, t + 40, t + 3], 2)
    plan = c.share(slots, min_saved=1)
    _check(c, plan, _rand(3, t, 4, D, seed=14, dtype=dtype), scale=1e-44)
    q = _rand(3, t, 4, D, seed=15, dtype=dtype) * 2.0 ** (-100 if dtype == torch.bfloat16 else -20)
    q[0] = 0
    c.k_scale[c.k_scale.isfinite()] = 2.0 ** -64       # the scale of pages of zeros, and the smallest there is
    _check(c, plan, q, scale=1e-20)


def test_pages_that_nothing_was_written_to():
    """Scales of 0 and codes of 0, as in a call made before the first append: zeros, each token with the same weight."""
    c = _cache(1, 20, 1, 3, page=32, max_len=320)
    c.reserve([0], 200)
    c.fork([0, 0], [1, 2])
    c.reserve([0, 1, 2], [1, 70, 2])
    _check(c, c.share([0, 1, 2], min_saved=1), _rand(3, 1, 4, D, seed=16))
