"""The 8-bit page cache: append, attend and the page operations against plain 64-bit forms (oracle/paged_kv.py).

append and the page operations are exact: codes and scales equal the definition's bit for bit (a power-of-two scale makes
every step but the one rounding exact).  attend, with u half a step of the output type and A = sum_j p_j |v_j|:
  * o is rounded once: u |o| <= u A;
  * a weight enters the product as three e4m3 parts of 4 bits each: off by at most 2^-12 relatively, or 2^-26 of its block of
    keys' largest weight where the parts run into the code's smallest step (128 keys at most: 2^-19 A' with A' the largest
    |v| of the block, covered by the absolute term);
  * a query enters as three e4m3 parts: exact for 8 and 11 significant bits; a score's 256 products are summed in the tensor
    core's fp32 accumulator: off by at most 2^-13 S with S = scale * sum |q k|, even if it cut its addends to 14 bits of the
    largest (they are exact products); a weight by twice that relatively.
So |o - o*| <= (u + 2^-11 + 2^-12 S) A + 2^-19 max|v|, and |lse - lse*| <= 2^-13 S + 2^-16 (1 + |lse*|)."""
import pytest
import torch

from oracle import paged_kv as opk

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
D = 256


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


def _cache(layers, pages, heads, slots, **kw):
    _dev()
    from heimdall_b200 import PagedKV
    return PagedKV(layers, pages, heads, slots, **kw)


def _rand(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _fill(c, seed=0):
    """Random codes and scales in every page, NaN codes among those that no test below may read."""
    g = torch.Generator().manual_seed(seed)
    for x in (c.k_pages, c.v_pages):
        r = (torch.randn(x.shape, generator=g) * 64).clamp(-448, 448).to(torch.float8_e4m3fn)
        x.copy_(r)
    for s in (c.k_scale, c.v_scale):
        s.copy_(torch.ldexp(torch.ones(s.shape), torch.randint(-9, -3, s.shape, generator=g)))


def _poison(c):
    """NaN codes and NaN scales wherever no token of a slot is."""
    lens, table = c.lens.tolist(), c.table.tolist()
    used = {}
    for n, row in zip(lens, table):
        for j, p in enumerate(row):
            if p >= 0:
                used[p] = max(used.get(p, 0), min(c.page, n - j * c.page))
    for p in range(c.k_pages.shape[1]):
        n = used.get(p, 0)
        for x in (c.k_pages, c.v_pages):
            x[:, p, :, n:] = torch.full((1,), float("nan")).to(torch.float8_e4m3fn).to(x.device)
        if n == 0:
            c.k_scale[:, p] = float("nan")
            c.v_scale[:, p] = float("nan")


def _host(c, layer=0):
    return [x[layer].cpu().double() for x in (c.k_pages, c.k_scale, c.v_pages, c.v_scale)]


def _same(a, b):
    return torch.equal(a.nan_to_num(nan=1e9), b.nan_to_num(nan=1e9))


def _check_append(c, before, slots, news, k, v, layer=0):
    kc, ks, vc, vs = before
    at = 0
    for slot, n in zip(slots, news):
        row, ln = c.table[slot].tolist(), int(c.lens[slot])
        opk.append(kc, ks, row, ln, k[at:at + n])
        opk.append(vc, vs, row, ln, v[at:at + n])
        at += n
    for got, want in zip(_host(c, layer), (kc, ks, vc, vs)):
        assert _same(got, want)


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_packed_prompts_and_steps(page, dtype):
    c = _cache(2, 40, 2, 5, page=page, max_len=20 * 16)
    news = [1, 0, page, page + 1, 3 * page - 1 if page < 128 else 200]
    c.reserve(range(5), news)
    T = sum(news)
    k, v = _rand(T, 2, D, seed=1, dtype=dtype) * 3, _rand(T, 2, D, seed=2, dtype=dtype)
    cu = torch.tensor([0] + news).cumsum(0).cuda()
    before = _host(c, 1)
    c.append(1, k.cuda(), v.cuda(), cu_seqlens=cu)
    _check_append(c, before, range(5), news, k, v, 1)
    assert not c.k_pages[0].view(torch.uint8).any() and not c.v_scale[0].any()
    for step in range(3):          # growing values: the pages' scales grow with them, earlier codes are rounded again
        c.reserve([3, 0, 1], 1)
        k, v = _rand(3, 1, 2, D, seed=3 + step, dtype=dtype) * 2.0 ** step, _rand(3, 1, 2, D, seed=9 + step, dtype=dtype) * 40.0 ** step
        before = _host(c, 1)
        c.append(1, k.cuda(), v.cuda(), torch.tensor([3, 0, 1], device="cuda"))
        _check_append(c, before, [3, 0, 1], [1, 1, 1], k[:, 0], v[:, 0], 1)


def test_append_special_values():
    c = _cache(1, 4, 1, 1, page=16)
    c.reserve([0], 20)
    x = torch.zeros(20, 1, D)
    x[3, 0, 5], x[4, 0, 6], x[4, 0, 7], x[5, 0, 0] = float("inf"), -float("inf"), float("nan"), 7.0
    x[16] = 0.0
    x[17, 0, 0] = 2.0 ** -120
    k = x.to(torch.bfloat16)
    before = _host(c)
    c.append(0, k.cuda()[None], -k.cuda()[None])
    _check_append(c, before, [0], [20], k, -k)
    assert c.k_scale[0, 0, 0] == 2.0 ** -6 and c.k_scale[0, 1, 0] == 2.0 ** -64
    big = torch.full((1, 1, 1, D), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16)
    c.reserve([0], 1)
    before = _host(c)
    c.append(0, big.cuda(), big.cuda())
    _check_append(c, before, [0], [1], big[0], big[0])


def test_append_strides_order_and_bounds():
    c = _cache(1, 6, 2, 3, page=16, max_len=48)
    kr = _rand(3, 2, 5, D, seed=1).cuda()                      # head-major, as the roped keys are
    v = _rand(3, 5, 2, D, seed=2).cuda()
    c.reserve(range(3), 5)
    before = _host(c)
    c.append(0, kr.transpose(1, 2), v)
    _check_append(c, before, range(3), [5] * 3, kr.transpose(1, 2).reshape(15, 2, D).cpu(), v.reshape(15, 2, D).cpu())
    keep = _host(c)
    c.append(0, kr.transpose(1, 2), v, torch.tensor([7, -1, 3], device="cuda"))          # no such slots
    c.append(0, kr.transpose(1, 2)[:0], v[:0])
    c.append(0, kr.transpose(1, 2)[:, :0], v[:, :0])
    assert all(_same(a, b) for a, b in zip(_host(c), keep))
    w = _rand(2, 5, 2, D, seed=3).cuda()
    before = _host(c)
    c.append(0, w, w, torch.tensor([1, 1], device="cuda"))      # a slot named twice: the first writes
    _check_append(c, before, [1], [5], w[0].cpu(), w[0].cpu())
    before = _host(c)                                           # more tokens than the slot has: only its last 5 fit
    w = _rand(1, 9, 2, D, seed=4).cuda()
    c.append(0, w, w)
    _check_append(c, before, [0], [9], w[0].cpu(), w[0].cpu())
    c.free([0])
    c.table[0, 0], c.lens[0] = 99, 4                            # a page number outside the pool: nothing is stored
    before = _host(c)
    c.append(0, w[:, :4], w[:, :4])
    assert all(_same(a, b) for a, b in zip(_host(c), before))


# ------------------------------------------------------------------------------------------------ attend
def _check_attend(c, q, slots, scale=None, layer=0, **kw):
    ids = None if slots is None else torch.tensor(slots, device="cuda")
    o, lse = c.attend(layer, q.cuda(), ids, scale, with_lse=True)
    o, lse, u = o.cpu(), lse.cpu().double(), U[q.dtype]
    assert o.dtype == q.dtype and torch.isfinite(o).all()
    kc, ks, vc, vs = _host(c, layer)
    for b in range(q.shape[0]):
        slot = b if slots is None else slots[b]
        ok = 0 <= slot < c.lens.numel()
        ro, rl, mag, big = opk.attend(kc, ks, vc, vs, c.table[slot].tolist() if ok else [], int(c.lens[slot]) if ok else 0, q[b], scale)
        top = float((vc.nan_to_num().abs().amax((2, 3)) * vs.nan_to_num()).max())
        tol = (u + 2.0 ** -11 + 2.0 ** -12 * big[..., None]) * mag + 2.0 ** -19 * top * (mag > 0)
        off = (o[b].double() - ro).abs()
        assert (off <= tol).all(), (b, (off - tol).max())
        dead = rl == -float("inf")
        assert (lse[b][dead] == -float("inf")).all() and (o[b].transpose(0, 1)[dead] == 0).all()
        off = (lse[b] - rl).abs()[~dead]
        assert (off <= (2.0 ** -13 * big.T + 2.0 ** -16 * (1 + rl.abs()))[~dead]).all(), (b, off.max())
    return o


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("H,G,t,dtype", [(24, 4, 1, torch.bfloat16), (6, 1, 4, torch.float16), (2, 2, 3, torch.bfloat16),
                                         (8, 1, 5, torch.bfloat16), (24, 1, 1, torch.float16), (3, 3, 1, torch.bfloat16)])
def test_attend(page, H, G, t, dtype):
    lens = [1, 16, 127, 128, 129, 300, 0, 515]
    c = _cache(1, 140, G, len(lens), page=page, max_len=1024)
    for step in (0, 1):                   # two rounds, so that the pages of a sequence are not in a row
        c.reserve(range(len(lens)), [n // 2 if step else n - n // 2 for n in lens])
    _fill(c)
    _poison(c)
    _check_attend(c, _rand(len(lens), t, H, D, dtype=dtype), None)


def test_attend_longer_and_slots_in_any_order():
    lens = [5000, 1, 2999, 64]
    c = _cache(2, 150, 2, 6, page=64, max_len=8192)
    c.reserve([4, 0, 2, 5], lens)
    _fill(c, 1)
    _poison(c)
    q = _rand(7, 1, 12, D, seed=5)
    _check_attend(c, q, [4, 0, 2, 5, 4, 1, 9], layer=1)           # one slot twice, an empty one, one that is not there
    _check_attend(c, q[:1], [4], layer=1)      # in another batch a sequence is cut elsewhere: the same to rounding, not to the bit
    _check_attend(c, q[:2] * 6, [4, 2], scale=0.3, layer=1)


@pytest.mark.parametrize("H,t,page", [(6, 4, 16), (6, 2, 64), (12, 2, 32), (5, 3, 128)])
def test_attend_several_tokens_over_long_and_short_sequences(H, t, page):
    """Rows in every size of block (16 and 24 at a time), runs of many tiles and of many segments in one CTA."""
    lens = [7000, 4, 130, 40, 2900] + [5 + 3 * i for i in range(40)] + [1500]
    c = _cache(1, sum(-(-n // page) for n in lens), 1, len(lens), page=page, max_len=7040)
    c.reserve(range(len(lens)), lens)
    _fill(c, 9)
    _check_attend(c, _rand(len(lens), t, H, D, seed=11, dtype=torch.float16), None)


def test_attend_many_sequences():
    n = 150
    lens = [(37 * i) % 200 for i in range(n)]
    c = _cache(1, 700, 1, n, page=32, max_len=256)
    c.reserve(range(n), lens)
    _fill(c, 2)
    _poison(c)
    _check_attend(c, _rand(n, 1, 2, D, seed=6), None)


def test_attend_more_sequences_than_threads():
    """Slots in any order, as 64-bit numbers, more sequences than a CTA has threads; the longest is cut over many CTAs."""
    n = 900
    lens = [(37 * i) % 60 for i in range(n)]
    lens[700] = 4000
    c = _cache(1, 1200, 1, n, page=64, max_len=4096)
    c.reserve(range(n), lens)
    _fill(c, 12)
    _poison(c)
    slots = [(i * 7) % n for i in range(n)]
    _check_attend(c, _rand(n, 1, 2, D, seed=13), slots)


@pytest.mark.parametrize("n,page", [(75, 32), (1100, 16), (33, 128)])
def test_append_many_sequences(n, page):
    news = [(11 * i) % 40 * (n < 100 or i % 5 == 0) for i in range(n)]
    c = _cache(1, n * 3, 1, n + 2, page=page, max_len=max(page, 96))
    slots = [(i * 2 + 1) % (n + 2 if n % 2 else n + 1) for i in range(n)]
    c.reserve(slots, [i % 7 for i in range(n)])
    c.reserve(slots, news)
    _fill(c, 14)
    T = sum(news)
    k, v = _rand(T, 1, D, seed=15) * 5, _rand(T, 1, D, seed=16)
    before = _host(c)
    c.append(0, k.cuda(), v.cuda(), torch.tensor(slots, device="cuda"), torch.tensor([0] + news).cumsum(0).cuda())
    _check_append(c, before, slots, news, k, v)


@pytest.mark.parametrize("page,G", [(16, 5), (16, 4), (32, 3), (32, 2), (128, 3)])
def test_append_long_prompts_of_several_heads(page, G):
    """So many pages that a CTA takes several heads of a page, whose number need not go into theirs; pages half full and values of
    which a page's scale grows among them."""
    lens, had = [page * 70 + 5, 1, page * 55 - 3, 0, page * 30], [3, page - 1, page // 2, 7, 0]
    c = _cache(1, 200, G, 5, page=page, max_len=page * 80)
    c.reserve(range(5), had)
    k = _rand(1, 1, 1, D, seed=17).expand(5, page, G, D)
    c.append(0, k.cuda(), k.cuda())
    c.reserve(range(5), lens)
    T = sum(lens)
    k, v = (_rand(T, G, D, seed=18 + i) * torch.logspace(-3, 3, G)[:, None].to(torch.bfloat16) for i in range(2))
    before = _host(c)
    c.append(0, k.cuda(), v.cuda(), cu_seqlens=torch.tensor([0] + lens).cumsum(0).cuda())
    _check_append(c, before, range(5), lens, k, v)


def test_calls_without_sequences_or_tokens():
    c = _cache(1, 4, 2, 2, page=16, max_len=32)
    c.reserve([0], 3)
    c.reserve([], 1), c.free([]), c.fork([], []), c.truncate([], 0)
    before = _host(c)
    none, cu = torch.zeros(0, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    k = torch.zeros(0, 2, D, dtype=torch.bfloat16, device="cuda")
    c.append(0, k, k, none, cu)
    c.append(0, k[None], k[None])
    c.append(0, k.view(0, 1, 2, D), k.view(0, 1, 2, D))
    for B, t in ((0, 1), (2, 0), (0, 0)):
        o, lse = c.attend(0, torch.zeros(B, t, 4, D, dtype=torch.bfloat16, device="cuda"), none if B == 0 else None, with_lse=True)
        assert o.shape == (B, t, 4, D) and lse.shape == (B, 4, t)
    assert all(_same(x, y) for x, y in zip(_host(c), before)) and c.length(0) == 3
    for slot in (-1, 2):
        with pytest.raises(ValueError):
            c.length(slot)


def test_attend_one_heavy_key_among_many():
    """A weight near one beside thousands near 2^-13: their sum counts."""
    c = _cache(1, 64, 1, 1, page=128, max_len=8192)
    c.reserve([0], 8000)
    k = torch.zeros(8000, 1, D)
    k[17, 0, :16] = 9.0 * 16 / 16
    v = torch.ones(8000, 1, D)
    v[17] = -1.0
    c.append(0, k.to(torch.bfloat16).cuda()[None], v.to(torch.bfloat16).cuda()[None])
    q = torch.zeros(1, 1, 1, D)
    q[..., :16] = 1.0
    _check_attend(c, q.to(torch.bfloat16), None)


def test_attend_scales_far_apart():
    c = _cache(1, 16, 1, 1, page=16)
    c.reserve([0], 250)
    _fill(c, 3)
    c.v_scale.copy_(torch.ldexp(torch.ones(16), torch.arange(16) % 5 * 6 - 20)[None, :, None])
    c.k_scale.copy_(torch.ldexp(torch.ones(16), torch.arange(16) % 3 * 2 - 9)[None, :, None])
    _poison(c)
    _check_attend(c, _rand(1, 1, 4, D, seed=7), None)


def test_attend_missing_pages_and_non_finite_values():
    c = _cache(1, 20, 1, 2, page=16)
    c.reserve([0, 1], [150, 70])
    _fill(c, 4)
    c.table[0, 3], c.table[0, 9], c.table[1, :] = -1, 20, -1
    q = _rand(2, 2, 4, D, seed=8)
    _check_attend(c, q, None)
    c.table[0, 3] = 3
    nan = torch.full((1,), float("nan")).to(torch.float8_e4m3fn).cuda()
    c.v_pages[0, 3, 0, 5, 7] = nan
    o = c.attend(0, q.cuda())[0]
    assert torch.isnan(o[0, :, :, 7]).all() and torch.isfinite(o[0, :, :, :7]).all() and (o[1] == 0).all()
    c.v_pages[0, 3, 0, 5, 7] = 0.5 * torch.ones((), device="cuda").to(torch.float8_e4m3fn).float()
    c.k_pages[0, 3, 0, 5, 7] = nan
    assert torch.isnan(c.attend(0, q.cuda())[0][0]).all()
    c.k_pages[0, 3, 0, 5, 7] = 1.0
    q[0, 0, 1, 9], q[0, 1, 2, 3] = float("inf"), float("nan")
    o = c.attend(0, q.cuda())[0][0]
    bad = torch.zeros(2, 4, dtype=torch.bool)
    bad[0, 1] = bad[1, 2] = True
    assert torch.equal(torch.isnan(o).all(-1).cpu(), bad) and torch.isfinite(o[~bad.cuda()]).all()


def test_attend_strided_query():
    c = _cache(1, 20, 2, 2, page=64)
    c.reserve([0, 1], [150, 700])
    _fill(c, 5)
    x = _rand(2, 4, 3, D, seed=9).cuda()                       # [B,H,t,D], as the roped queries are
    a = c.attend(0, x.transpose(1, 2))[0]
    assert torch.equal(a, c.attend(0, x.transpose(1, 2).contiguous())[0])
    odd = torch.empty(2, 3, 4, D + 1, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(x.transpose(1, 2))
    assert torch.equal(a, c.attend(0, odd)[0])


def test_attend_is_the_same_every_time():
    c = _cache(1, 300, 4, 3, page=64)
    c.reserve(range(3), [9000, 3001, 40])
    _fill(c, 6)
    q = _rand(3, 1, 24, D, seed=10).cuda()
    a = c.attend(0, q)[0]
    for _ in range(5):
        assert torch.equal(a, c.attend(0, q)[0])


# ------------------------------------------------------------------------------------------------ pages
def _sequence(c, slot, layer):
    """What a slot holds, in values."""
    n = int(c.lens[slot])
    row = c.table[slot].long()[:-(-n // c.page)]
    return [(p[layer][row].double() * s[layer][row].double()[..., None, None]).transpose(1, 2).reshape(-1, c.heads, D)[:n].cpu()
            for p, s in ((c.k_pages, c.k_scale), (c.v_pages, c.v_scale))]


def _all(c, slots):
    return [_sequence(c, s, layer) for s in slots for layer in range(c.layers)]


def _equal(a, b):
    return all(torch.equal(x, y) for p, q in zip(a, b) for x, y in zip(p, q))


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_fork_truncate_free_and_compact_keep_what_the_sequences_hold(page):
    c = _cache(3, 60, 2, 8, page=page, max_len=6 * page)
    lens = [page * 3 + 5, page * 2, 1, page * 5 - 1]
    c.reserve(range(4), lens)
    _fill(c, 7)
    held = _all(c, range(4))
    stale = c.k_pages[:, 40].clone()
    c.fork([0, 0, 1, 3], [4, 5, 6, 7])
    assert c.lens.tolist() == lens + [lens[0], lens[0], lens[1], lens[3]]
    assert _equal(_all(c, range(4)), held) and _equal(_all(c, [4, 5]), held[0:3] + held[0:3])
    assert _equal(_all(c, [6]), held[3:6]) and _equal(_all(c, [7]), held[9:12])
    assert torch.equal(c.table.cpu(), torch.from_numpy(c.host.table)) and torch.equal(c.k_pages[:, 40], stale)
    c.reserve([4], 1)                                  # a fork's own tokens leave its parent alone
    k = _rand(1, 1, 2, D, seed=8).cuda() * 100
    c.append(0, k, k, torch.tensor([4], device="cuda"))
    assert _equal(_all(c, [0, 5]), held[0:3] + held[0:3])
    c.truncate([5, 0], [page + 2, page + 3])
    cut = lambda s, n: [[x[:n] for x in p] for p in s]
    assert _equal(_all(c, [5]), cut(held[0:3], page + 2)) and _equal(_all(c, [0]), cut(held[0:3], page + 3))
    c.free([1, 2])
    live = c.compact()
    assert c.table.max() < live == c.host.pages - c.free_pages
    assert torch.equal(c.table.cpu(), torch.from_numpy(c.host.table)) and c.lens.tolist()[:4] == [page + 3, 0, 0, lens[3]]
    assert _equal(_all(c, [3, 7]), held[9:12] + held[9:12]) and _equal(_all(c, [6]), held[3:6])
    assert _equal(_all(c, [5]), cut(held[0:3], page + 2))
    c.free(range(8))
    assert c.free_pages == 60 and (c.table == -1).all() and (c.lens == 0).all() and c.compact() == 0


def test_many_pages_in_one_call():
    """More changes than one launch carries."""
    c = _cache(1, 3000, 1, 40, page=16, max_len=1600)
    c.reserve(range(0, 40, 2), 1500)
    c.reserve(range(1, 40, 2), 700)
    _fill(c, 8)
    odd = _all(c, range(1, 40, 2))
    assert torch.equal(c.table.cpu(), torch.from_numpy(c.host.table))
    c.free(range(0, 40, 2))
    c.compact()
    assert torch.equal(c.table.cpu(), torch.from_numpy(c.host.table)) and _equal(_all(c, range(1, 40, 2)), odd)
    c.fork([1] * 20, range(0, 40, 2))
    assert torch.equal(c.table.cpu(), torch.from_numpy(c.host.table)) and _equal(_all(c, range(0, 40, 2)), odd[:1] * 20)


def test_refusals():
    c = _cache(1, 4, 2, 2, page=16, max_len=32)
    k = _rand(2, 1, 2, D).cuda()
    with pytest.raises(RuntimeError, match="full"):
        _cache(1, 1, 2, 2, page=16, max_len=32).reserve([0, 1], 16)
    for kind, call in ((ValueError, lambda: c.append(1, k, k)), (ValueError, lambda: c.append(0, k, k[:1])), (ValueError, lambda: c.append(0, k[0], k[0])),
                       (ValueError, lambda: c.append(0, k[:, :, :1], k[:, :, :1])), (NotImplementedError, lambda: c.append(0, k.float(), k.float())),
                       (ValueError, lambda: c.append(0, k, k.half())), (RuntimeError, lambda: c.append(0, k.cpu(), k.cpu())),
                       (ValueError, lambda: c.append(0, k, k, torch.tensor([0], device="cuda"))),
                       (NotImplementedError, lambda: c.append(0, k.clone().requires_grad_(), k)),
                       (ValueError, lambda: c.append(0, torch.cat([k, k]), torch.cat([k, k]))),
                       (ValueError, lambda: c.attend(0, k[:, :, :1])), (ValueError, lambda: c.attend(-1, k)), (ValueError, lambda: c.attend(0, k[0])),
                       (NotImplementedError, lambda: c.attend(0, k.float())), (NotImplementedError, lambda: c.attend(0, k.expand(2, 1, 2, D).repeat(1, 1, 25, 1))),
                       (ValueError, lambda: c.attend(0, k, scale=0.0)), (NotImplementedError, lambda: c.attend(0, k.clone().requires_grad_())),
                       (ValueError, lambda: c.attend(0, k, torch.tensor([0, 1, 1], device="cuda"))), (ValueError, lambda: c.layer(1))):
        with pytest.raises(kind):
            call()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(g):
            c.reserve([1], 0)


# ------------------------------------------------------------------------------------------------ together
def test_serving_steps_captured_and_replayed():
    """A decode step (append and attend of two layers) captured once and replayed as the sequences grow, on a stream of its
    own, equals the eager steps."""
    dev = _dev()
    B, G, H, steps = 3, 2, 6, 20
    caches = [_cache(2, 60, G, B, page=16, max_len=256) for _ in range(2)]
    g = torch.Generator().manual_seed(0)
    lens = [30, 1, 47]
    cu = torch.tensor([0] + lens).cumsum(0).to(dev)
    k0, v0 = (torch.randn(2, sum(lens), G, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    for c in caches:
        c.reserve(range(B), lens)
        for i in range(2):
            c.append(i, k0[i], v0[i], cu_seqlens=cu)
    q, k, v = (torch.zeros(2, B, 1, h, D, dtype=torch.bfloat16, device=dev) for h in (H, G, G))

    def step(c):
        out = []
        for i in range(2):
            c.append(i, k[i], v[i])
            out.append(c.attend(i, q[i])[0])
        return out
    xs = [[torch.randn(x.shape, generator=g).to(torch.bfloat16).to(dev) for x in (q, k, v)] for _ in range(steps)]
    graph, stream = None, torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for a, b, d in xs:
        q.copy_(a), k.copy_(b), v.copy_(d)
        caches[0].reserve(range(B), 1)
        want = step(caches[0])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            caches[1].reserve(range(B), 1)
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    got = step(caches[1])
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    for x, y in zip(_host(caches[0], 1), _host(caches[1], 1)):
        assert _same(x, y)


def test_calls_in_a_row_without_waiting():
    """Kernels start under the end of the one before: what they enqueue back to back is what they do one by one."""
    from heimdall_b200 import prompt_attention
    dev = _dev()
    g = torch.Generator().manual_seed(3)
    G, H, n = 2, 12, 12
    ks = [torch.randn(2, 1, G, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(n)]
    qs = [torch.randn(2, 1, H, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(n)]
    x = torch.randn(300, G, D, generator=g).to(torch.bfloat16).to(dev)
    cu = torch.tensor([0, 300], device=dev, dtype=torch.int32)

    def steps(wait):
        c = _cache(1, 120, G, 4, page=16, max_len=700)
        c.reserve([0, 1], 300)
        out, q = [], torch.empty_like(qs[0])
        for i in range(n):
            for b in (0, 1):
                if i == 0:
                    c.append(0, x, x, torch.tensor([b], device=dev), cu)
                    wait()
            c.reserve([0, 1], 1)
            wait()
            q.copy_(qs[i])
            c.append(0, ks[i], ks[i])
            wait()
            out.append(c.attend(0, q)[0])
            wait()
            c.fork([0], [2]), wait()
            out.append(c.attend(0, q[:1], torch.tensor([2], device=dev))[0])
            wait()
            out.append(prompt_attention(torch.cat([q[0]] * 40), torch.cat([x] * 2)[:40], torch.cat([x] * 2)[:40], cu.clamp(max=40))[0])
            c.free([2]), wait()
            if i % 3 == 2:
                c.truncate([1], c.length(1) - 2), wait()
                c.compact(), wait()
        torch.cuda.synchronize()
        return out, _host(c)
    a, pa = steps(torch.cuda.synchronize)
    for _ in range(3):
        b, pb = steps(lambda: None)
        assert all(torch.equal(u, w) for u, w in zip(a, b)) and all(_same(u, w) for u, w in zip(pa, pb))


def test_captured_behind_copies_and_other_streams():
    """What comes before a call in a graph may be a copy from the host, a memset or work of another stream: it is waited for."""
    from heimdall_b200 import prompt_attention
    dev = _dev()
    c = _cache(1, 40, 2, 2, page=64)
    c.reserve([0, 1], [300, 65])
    _fill(c, 20)
    host = [_rand(2, 1, h, D, seed=21 + h).pin_memory() for h in (2, 8)]
    k, q = (x.to(dev) for x in host)
    big, slots = _rand(1 << 24, seed=22).to(dev), torch.tensor([0, 1], device=dev, dtype=torch.int32)
    cu = torch.tensor([0, 1, 2], device=dev, dtype=torch.int32)
    side = torch.cuda.Stream()

    def calls():
        k.copy_(host[0], non_blocking=True)                     # a copy node, then append
        c.append(0, k, k, slots)
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):                           # something slow on the other stream, which q waits for
            big.mul_(1.0)
            q.copy_(host[1], non_blocking=True)
        slots.zero_()
        slots[1:].fill_(1)
        main.wait_stream(side)
        o = c.attend(0, q, slots)[0]
        q.copy_(host[1], non_blocking=True)
        return o, prompt_attention(q.view(2, 8, D), k.view(2, 2, D), k.view(2, 2, D), cu)[0]
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for i in range(5):
        for j, x in enumerate(host):
            x.copy_(_rand(*x.shape, seed=30 + 2 * i + j) * 3)
        k.zero_(), q.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        held = [x.clone() for x in got]
        want = calls()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, want)), i


def test_two_captured_graphs_side_by_side():
    dev = _dev()
    cs = [_cache(1, 200, 2, 2, page=32) for _ in range(2)]
    qs = [_rand(2, 1, 8, D, seed=i).to(dev) for i in range(2)]
    for i, c in enumerate(cs):
        c.reserve(range(2), [2000 + i, 3001])
        _fill(c, 10 + i)
    want = [c.attend(0, q)[0] for c, q in zip(cs, qs)]
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in cs], []
    for g, c, q in zip(graphs, cs, qs):
        with torch.cuda.graph(g, pool=pool):
            outs.append(c.attend(0, q)[0])
    for _ in range(5):
        for g, o, w in zip(graphs, outs, want):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, w)
    s = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):                    # eager calls of two caches at once
        got = []
        for st, c, q in zip(s, cs, qs):
            with torch.cuda.stream(st):
                got.append(c.attend(0, q)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_teacher_over_pages():
    """retrieval.teacher with a paged layer for a cache: the prompt as with the bf16 cache, later tokens from the codes."""
    dev = _dev()
    from heimdall_b200.retrieval import teacher
    B, H, G = 2, 8, 2
    c = _cache(2, 40, G, B, page=64, max_len=512)
    layers, dicts = [c.layer(0), c.layer(1)], [{}, {}]
    for t in (130, 1, 3, 1):
        for i in range(2):
            qr, kr, v = (_rand(B, h, t, D, seed=100 * t + 10 * i + h).to(dev) for h in (H, G, G))
            v = v.transpose(1, 2).contiguous()
            want = teacher(qr, kr, v, dicts[i])
            got = teacher(qr, kr, v, layers[i])
            # e4m3 moves every key and value by at most 2^-4 of itself: scores by 2^-4 S (S about 10: 0.6 at worst, 0.05 rms),
            # so the outputs agree to some percent; the prompt, which reads no codes, to bf16
            err = ((got.double() - want.double()).norm() / want.double().norm()).item()
            assert err < (8e-3 if t == 130 else 0.15), (t, i, err)
    assert c.lens.tolist() == [135, 135]
    with pytest.raises(NotImplementedError):
        teacher(qr, kr, v, layers[0], dict(k=1, block=16, window=16, sinks=4))
    layers[0].n -= 2
    with pytest.raises(ValueError, match="in step"):
        teacher(qr, kr, v, layers[0])


def test_a_change_of_pages_that_fails_on_the_device_ends_the_cache(monkeypatch):
    """The host's table would be ahead of the device's: no later call goes on from there."""
    import heimdall_b200.paged as paged
    c = _cache(1, 8, 2, 3, page=16, max_len=32)
    c.reserve([0], 20)
    real = paged._lib.call

    def failing(name, *a):
        if name == "bf_paged_pages":
            raise RuntimeError("the launch failed")
        return real(name, *a)
    k = _rand(1, 1, 2, D).cuda()
    with monkeypatch.context() as m:
        m.setattr(paged._lib, "call", failing)
        with pytest.raises(RuntimeError, match="the launch failed"):
            c.fork([0], [1])
    for call in (lambda: c.reserve([0], 1), lambda: c.free([1]), lambda: c.fork([0], [2]), lambda: c.truncate([0], 3), c.compact,
                 lambda: c.append(0, k, k), lambda: c.attend(0, k)):
        with pytest.raises(RuntimeError, match="cannot be used any more"):
            call()


@pytest.mark.parametrize("t,H", [(1, 2), (4, 6)])
@pytest.mark.parametrize("dtype,e", [(torch.bfloat16, 8), (torch.bfloat16, 16), (torch.bfloat16, 20), (torch.bfloat16, 30),
                                     (torch.float16, 8), (torch.float16, 15)])
def test_attend_query_rows_of_a_wide_range(dtype, e, t, H):
    """One component of 2^e among others of order one, against keys that are zero there.

    The parts of a query end at 2^-17 of a row scaled to [128, 256): a component is off by at most half of that, 2^-18 / 128 = 2^-25 of
    the row's largest, a score by that times scale * sum |k|, a weight by twice that relatively, as long as it is small."""
    c = _cache(1, 20, 1, 1, page=64)
    c.reserve([0], 700)
    _fill(c, 23)
    c.k_pages[0, :, :, :, 37] = 0.0
    c.k_scale.fill_(2.0 ** -7)
    q = _rand(1, t, H, D, seed=24, dtype=dtype)
    q[..., 37] = 2.0 ** e
    q[:, -1, -1] = _rand(D, seed=25, dtype=dtype)                  # and a row without one
    o, lse = c.attend(0, q.cuda(), with_lse=True)
    kc, ks, vc, vs = _host(c)
    ro, rl, mag, big = opk.attend(kc, ks, vc, vs, c.table[0].tolist(), 700, q[0], None)
    span = D ** -0.5 * float((kc * ks[..., None, None]).abs().sum(-1).max())
    lost = 2.0 ** -25 * span * q[0].abs().amax(-1).double()        # [t, H]
    known = lost < 2.0 ** -4                                       # 2 x is a bound of e^x - 1 and 1 - e^-x well beyond that
    assert known[-1, -1] and (known.all() or e > 16)
    assert torch.isfinite(o).all()
    top = float((vc.abs().amax((2, 3)) * vs).max())
    tol = (U[dtype] + 2.0 ** -11 + 2.0 ** -12 * big[..., None] + 2 * 2 * lost[..., None]) * mag + 2.0 ** -19 * top
    assert ((o[0].cpu().double() - ro).abs() <= tol)[known].all()
    off, tol = (lse[0].cpu().double() - rl).abs(), 2.0 ** -13 * big.T + lost.T + 2.0 ** -16 * (1 + rl.abs())
    assert (off <= tol)[known.T].all(), (off - tol).max()


def test_append_cumulative_lengths_beyond_the_tensors_and_out_of_order():
    """Entries are clamped into [0, T].  Out of order they do not say which tokens are whose: what is written then lies in the named
    sequences' newest positions and nowhere else."""
    k, v = _rand(50, 2, D, seed=40), _rand(50, 2, D, seed=41)
    c = _cache(1, 30, 2, 4, page=16, max_len=160)
    c.reserve(range(4), [20, 40, 11, 7])
    _fill(c, 42)
    before = _host(c)
    c.append(0, k.cuda(), v.cuda(), torch.tensor([0, 1, 2], device="cuda"), torch.tensor([-3, 5, 42, 90], device="cuda"))
    _check_append(c, before, [0, 1, 2], [5, 37, 8], k, v)
    x = torch.full((50, 2, D), 7.0, dtype=torch.bfloat16, device="cuda")
    keep = [y.clone() for y in (c.k_pages, c.v_pages)]
    c.append(0, x, x, torch.tensor([0, 1, 2], device="cuda"), torch.tensor([0, 45, 9, 50], device="cuda"))
    for old, new in zip(keep, (c.k_pages, c.v_pages)):
        for slot, most in ((0, 20), (1, 5), (2, 41), (3, 0)):
            n = int(c.lens[slot])
            for j, p in enumerate(c.table[slot].tolist()[:-(-n // 16)]):
                a, b = old[0, p].view(torch.uint8), new[0, p].view(torch.uint8)
                assert torch.equal(a[:, max(n - j * 16, 0):], b[:, max(n - j * 16, 0):])          # behind the sequence's end
                if (j + 1) * 16 <= n - most or most == 0:           # pages of none of its newest tokens
                    assert torch.equal(a, b)
        assert torch.equal(old[0, 10:].view(torch.uint8), new[0, 10:].view(torch.uint8))       # pages of no sequence


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("apart", [4, 10, 16, 22])
def test_attend_small_scales_with_the_weight_beside_large_ones(apart, page):
    """Nearly all weight on pages whose V scale is 2^-apart of another's in the same tile; the largest scale of the last tile is on a page
    that the first tokens of the call do not see.  A weight times its V scale is held to 2^-26 of the tile's largest weight times its
    largest V scale: that times sum |code|, tile by tile, is the whole of the absolute term."""
    G, H, t, n = 2, 4, 3, 15 * 16 + 1
    c = _cache(1, 16, G, 1, page=page, max_len=256)
    c.reserve([0], n)
    _fill(c, 43)
    row = c.table[0].tolist()[:-(-n // page)]
    big = [row[j] for j in range(1, len(row), 4)] + [row[-1]]
    c.k_scale.fill_(2.0 ** -7)
    c.v_scale.fill_(2.0 ** -apart)
    c.v_scale[0, big, 1] = 0.5
    c.v_scale[0, big, 0] = 1.0
    c.k_pages[0, :, :, :, 0] = 256.0
    c.k_pages[0, big, :, :, 0] = -256.0
    q = _rand(1, t, H, D, seed=44)
    q[..., 0] = 80.0                                          # scores of 10 and -10 from this component
    o, _ = c.attend(0, q.cuda())
    kc, ks, vc, vs = _host(c)
    ro, _, mag, size = opk.attend(kc, ks, vc, vs, c.table[0].tolist(), n, q[0])
    for h in range(H):
        g = h // (H // G)
        k = (kc[row, g] * ks[row, g][:, None, None]).reshape(-1, D)[:n]
        code, scale = vc[row, g].reshape(-1, D)[:n].abs(), vs[row, g].repeat_interleave(page)[:n]
        for i in range(t):
            m = n - t + 1 + i
            p = torch.softmax(k[:m] @ q[0, i, h].double() / 16, 0)
            floor = torch.zeros(D, dtype=torch.float64)
            for a in range(0, m, 128):
                floor += 2.0 ** -26 * p[a:a + 128].max() * scale[a:a + 128].max() * code[a:min(m, a + 128)].sum(0)
            tol = (U[q.dtype] + 2.0 ** -11 + 2.0 ** -12 * size[i, h]) * mag[i, h] + floor
            off = (o[0, i, h].cpu().double() - ro[i, h]).abs()
            assert (off <= tol).all(), (h, i, (off - tol).max())
            w = p * scale[:m]
            assert w[scale[:m] < 0.25].sum() > 0.5 * w.sum() and floor.max() < 0.5 * mag[i, h].max()   # so that their part cannot be missing


@pytest.mark.parametrize("t", [25, 130, 600])
@pytest.mark.parametrize("H,G,page", [(3, 1, 16), (2, 2, 64)])
def test_attend_of_many_tokens_at_once(t, H, G, page):
    """A chunk of a prompt over the pages: many blocks of rows of one sequence, the last one not full, and tokens before the first."""
    lens = [t + 45, 100]
    c = _cache(1, sum(-(-n // page) for n in lens) + 1, G, 2, page=page, max_len=704)
    c.reserve([0, 1], lens)
    _fill(c, 45)
    _poison(c)
    _check_attend(c, _rand(2, t, H, D, seed=46, dtype=torch.float16 if t == 130 else torch.bfloat16), None)
