"""prompt_attention (causal attention of packed prompts) against its definition in 64 bits (oracle/paged_kv.py).

Tolerances, element by element, with u half a step of the output type (bf16 2^-8, fp16 2^-11) and A = sum_j p_j |v_j|:
  * the weights enter the product rounded to q's type: each is off by at most u, so o by u A;
  * o is rounded once: u |o| <= u A;
  * a score is a sum of 256 exact products in fp32: off by at most 256 * 2^-24 * S with S = scale * sum |q k|, and a weight
    by twice that relatively (it and the normaliser); exp2 and the sums add less than 2^-18 relatively.
So |o - o*| <= (2 u + 2^-15 S + 2^-18) A, and |lse - lse*| <= 2^-16 S + 2^-18 (1 + |lse*|)."""
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


def _cu(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def _inputs(T, Tk, H, G, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda n, h: torch.randn(n, h, D, generator=g).to(dtype)
    return r(T, H), r(Tk, G), r(Tk, G)


def _check(o, lse, q, k, v, cu, cuk=None, scale=None):
    ro, rl, mag, big = opk.prompt_attention(q, k, v, cu, cuk, scale)
    o, u = o.cpu(), U[q.dtype]
    assert o.dtype == q.dtype and torch.isfinite(o).all()
    tol = (2 * u + 2.0 ** -15 * big[..., None] + 2.0 ** -18) * mag
    assert ((o.double() - ro).abs() <= tol).all(), ((o.double() - ro).abs() - tol).max()
    if lse is not None:
        lse = lse.cpu().double()
        dead = rl == -float("inf")
        assert (lse[dead] == -float("inf")).all()
        off = (lse - rl).abs()[~dead]
        assert (off <= (2.0 ** -16 * big.T + 2.0 ** -18 * (1 + rl.abs()))[~dead]).all(), off.max()


def _run(q, k, v, cu, cuk=None, scale=None, **kw):
    from heimdall_b200 import prompt_attention
    dev = _dev()
    t = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)
    return prompt_attention(q.to(dev), k.to(dev), v.to(dev), t(cu), t(cuk), scale, with_lse=True, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,G", [(1, 1), (3, 1), (6, 1), (24, 4), (4, 4), (10, 2)])
@pytest.mark.parametrize("lens", [[1], [127], [128], [129], [300, 1, 0, 77, 256], [0, 5, 0]])
def test_packed_prompts(lens, H, G, dtype):
    T = sum(lens)
    q, k, v = _inputs(T, T, H, G, dtype)
    o, lse = _run(q, k, v, _cu(lens))
    _check(o, lse, q, k, v, _cu(lens))


@pytest.mark.parametrize("nq,nk", [([1, 5, 130], [400, 5, 131]), ([64, 0, 3], [1000, 7, 0]), ([140, 20], [100, 3]), ([129], [257])])
def test_queries_after_earlier_keys_and_rows_that_see_nothing(nq, nk):
    q, k, v = _inputs(sum(nq), sum(nk), 6, 2, torch.bfloat16, 1)
    o, lse = _run(q, k, v, _cu(nq), _cu(nk))
    _check(o, lse, q, k, v, _cu(nq), _cu(nk))
    at = 0
    for a, b in zip(nq, nk):         # the rows without a key
        none = max(0, a - b)
        assert (o[at:at + none] == 0).all() and (lse[:, at:at + none] == -float("inf")).all()
        at += a


@pytest.mark.parametrize("lens", [[1500, 700], [2047]])
def test_longer_prompts(lens):
    T = sum(lens)
    q, k, v = _inputs(T, T, 12, 2, torch.bfloat16, 2)
    o, lse = _run(q, k, v, _cu(lens))
    rows = torch.randperm(T, generator=torch.Generator().manual_seed(3))[:60].tolist()
    cu = _cu(lens)
    for i in rows:
        b = max(x for x in range(len(lens)) if cu[x] <= i)
        n = i + 1 - cu[b]
        _check(o[i:i + 1], lse[:, i:i + 1], q[i:i + 1], k[cu[b]:i + 1], v[cu[b]:i + 1], [0, 1], [0, n])


def test_rows_behind_the_last_sequence_are_zero():
    q, k, v = _inputs(300, 300, 6, 2, torch.bfloat16, 4)
    o, lse = _run(q, k, v, [0, 100, 140])
    _check(o[:140], lse[:, :140], q[:140], k[:140], v[:140], [0, 100, 140])
    assert (o[140:] == 0).all() and (lse[:, 140:] == -float("inf")).all()
    o, lse = _run(q, k, v, [0])
    assert (o == 0).all() and (lse == -float("inf")).all()


def test_lengths_beyond_the_tensors_are_cut():
    q, k, v = _inputs(100, 100, 6, 2, torch.bfloat16, 5)
    o, lse = _run(q, k, v, [0, 60, 4000])
    _check(o, lse, q, k, v, [0, 60, 100])
    o, lse = _run(q, k, v, [0, 60, 40, 100])       # a descending entry counts as the one before it
    _check(o, lse, q, k, v, [0, 60, 60, 100])
    o, lse = _run(q, k, v, [20, 60, 90])           # rows before the first sequence belong to none
    _check(o[20:90], lse[:, 20:90], q[20:90], k[20:90], v[20:90], [0, 40, 70])
    assert (o[:20] == 0).all() and (o[90:] == 0).all() and (lse[:, :20] == -float("inf")).all()
    o, lse = _run(q, k, v, [-7, 60, 100])
    _check(o, lse, q, k, v, [0, 60, 100])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_sequence_sees_nothing_of_its_neighbours(bad):
    """Non-finite keys, values and queries of other sequences, and of the rows behind the last one, change no bit."""
    lens = [90, 200, 33]
    q, k, v = _inputs(400, 400, 6, 2, torch.bfloat16, 6)
    cu = _cu(lens)
    o, lse = _run(q, k, v, cu)
    for x in (q, k, v):
        x[90:290] = bad
        x[323:] = bad
    o2, lse2 = _run(q, k, v, cu)
    for a, b in ((0, 90), (290, 323)):
        assert torch.equal(o[a:b], o2[a:b]) and torch.equal(lse[:, a:b], lse2[:, a:b])
    assert (o2[323:] == 0).all()


def test_later_keys_have_no_part():
    """What a key or value that a query does not see holds, changes nothing: finite values, NaN and infinities in keys."""
    q, k, v = _inputs(300, 300, 6, 2, torch.bfloat16, 7)
    o, _ = _run(q, k, v, [0, 300])
    k2, v2 = k.clone(), v.clone()
    k2[200:], v2[200:] = 3e4, 3e4
    assert torch.equal(_run(q, k2, v2, [0, 300])[0][:200], o[:200])
    k2[200:] = float("nan")
    o2 = _run(q, k2, v, [0, 300])[0]
    assert torch.equal(o2[:200], o[:200]) and torch.isnan(o2[200:]).all()
    k2[200:] = float("inf")
    assert torch.equal(_run(q, k2, v, [0, 300])[0][:200], o[:200])


@pytest.mark.parametrize("scale", [0.5, 2.0 ** -8])
def test_scale_and_large_scores(scale):
    q, k, v = _inputs(200, 200, 6, 2, torch.bfloat16, 8)
    q = q * 8
    o, lse = _run(q, k, v, [0, 150, 200], scale=scale)
    _check(o, lse, q, k, v, [0, 150, 200], scale=scale)


def test_strided_inputs():
    """Views of one fused projection, heads before tokens, and a last dimension that has to be copied."""
    dev = _dev()
    from heimdall_b200 import prompt_attention
    g = torch.Generator().manual_seed(9)
    x = torch.randn(150, 10, D, generator=g).to(torch.bfloat16)
    cu = torch.tensor([0, 70, 150], device=dev)
    xd = x.to(dev)
    o, lse = prompt_attention(xd[:, :6], xd[:, 6:8], xd[:, 8:], cu, with_lse=True)
    _check(o, lse, x[:, :6], x[:, 6:8], x[:, 8:], [0, 70, 150])
    hm = xd.transpose(0, 1).contiguous().transpose(0, 1)
    o2, _ = prompt_attention(hm[:, :6], hm[:, 6:8], hm[:, 8:], cu)
    assert torch.equal(o, o2)
    odd = torch.empty(150, 10, D + 1, dtype=torch.bfloat16, device=dev)[..., 1:]
    odd.copy_(xd)
    o3, _ = prompt_attention(odd[:, :6], odd[:, 6:8], odd[:, 8:], cu)
    assert torch.equal(o, o3)
    e = xd[:, 6:7].expand(150, 2, D)
    o4, lse4 = prompt_attention(xd[:, :6], e, xd[:, 8:], cu, with_lse=True)
    _check(o4, lse4, x[:, :6], x[:, 6:7].expand(150, 2, D), x[:, 8:], [0, 70, 150])


def test_refusals():
    dev = _dev()
    from heimdall_b200 import prompt_attention
    q, k, v = (x.to(dev) for x in _inputs(10, 10, 4, 2, torch.bfloat16))
    cu = torch.tensor([0, 10], device=dev)
    with pytest.raises(NotImplementedError, match="backward"):
        prompt_attention(q.clone().requires_grad_(), k, v, cu)
    with torch.no_grad():
        prompt_attention(q.clone().requires_grad_(), k, v, cu)
    for kind, a in ((ValueError, (q[0], k, v, cu)), (ValueError, (q, k, v[:5], cu)), (ValueError, (q, k.half(), v, cu)),
                    (NotImplementedError, (q.float(), k.float(), v.float(), cu)), (ValueError, (q[:, :3], k, v, cu)),
                    (NotImplementedError, (q[..., :128], k[..., :128], v[..., :128], cu)), (ValueError, (q[:5], k, v, cu)),
                    (ValueError, (q, k, v, cu[None])), (ValueError, (q, k, v, cu.float())), (ValueError, (q, k, v, cu[:0])),
                    (ValueError, (q, k, v, cu, torch.tensor([0, 5, 10], device=dev))), (RuntimeError, (q.cpu(), k, v, cu))):
        with pytest.raises(kind):
            prompt_attention(*a)
    for s in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            prompt_attention(q, k, v, cu, scale=s)


@pytest.mark.parametrize("H,G", [(6, 1), (4, 2), (3, 1)])
@pytest.mark.parametrize("nq,nk", [([5, 130], [3000, 2100]), ([1], [5000]), ([260, 3, 40], [2304, 0, 1999]), ([300], [2200])])
def test_few_queries_of_many_keys(nq, nk, H, G):
    """Blocks of many key tiles beside short ones, rows that see nothing and rows of no sequence."""
    T, Tk = sum(nq) + 7, sum(nk) + 9
    q, k, v = _inputs(T, Tk, H, G, torch.bfloat16, 14)
    o, lse = _run(q, k, v, _cu(nq), _cu(nk))
    _check(o[:-7], lse[:, :-7], q[:-7], k, v, _cu(nq), _cu(nk))
    assert (o[-7:] == 0).all() and (lse[:, -7:] == -float("inf")).all()
    o2, lse2 = _run(q, k, v, _cu(nq), _cu(nk))
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_many_sequences():
    """More sequences than a warp has lanes, most of them short, some empty."""
    lens = [(11 * i) % 23 for i in range(100)] + [200] + [(7 * i) % 5 for i in range(40)]
    T = sum(lens)
    q, k, v = _inputs(T, T, 3, 1, torch.bfloat16, 12)
    o, lse = _run(q, k, v, _cu(lens))
    _check(o, lse, q, k, v, _cu(lens))
    q, k, v = _inputs(T, T, 4, 2, torch.bfloat16, 13)
    o, lse = _run(q, k, v, _cu(lens))
    _check(o, lse, q, k, v, _cu(lens))


def test_more_sequences_than_shared_memory_lists():
    lens = [(5 * i) % 4 for i in range(1200)]
    T = sum(lens)
    q, k, v = _inputs(T, T, 2, 1, torch.bfloat16, 15)
    o, lse = _run(q, k, v, _cu(lens))
    _check(o, lse, q, k, v, _cu(lens))


def test_very_many_sequences_few_of_them_with_tokens():
    lens = [(1 + i % 3) * (i % 97 == 5) for i in range(40000)] + [130]
    T = sum(lens)
    q, k, v = _inputs(T, T, 3, 1, torch.float16, 16)
    o, lse = _run(q, k, v, _cu(lens))
    _check(o, lse, q, k, v, _cu(lens))


def test_no_tokens():
    dev = _dev()
    from heimdall_b200 import prompt_attention
    z = lambda h: torch.zeros(0, h, D, dtype=torch.bfloat16, device=dev)
    o, lse = prompt_attention(z(4), z(2), z(2), torch.zeros(3, dtype=torch.int32, device=dev), with_lse=True)
    assert o.shape == (0, 4, D) and lse.shape == (4, 0)
    q = torch.ones(4, 4, D, dtype=torch.bfloat16, device=dev)
    o, lse = prompt_attention(q, z(2), z(2), torch.tensor([0, 4], device=dev), torch.tensor([0, 0], device=dev), with_lse=True)
    assert (o == 0).all() and (lse == -float("inf")).all()


def test_two_streams_and_a_captured_call():
    dev = _dev()
    from heimdall_b200 import prompt_attention
    a = [x.to(dev) for x in _inputs(700, 700, 6, 2, torch.bfloat16, 10)]
    b = [x.to(dev) for x in _inputs(300, 300, 6, 2, torch.bfloat16, 11)]
    ca, cb = torch.tensor([0, 300, 700], device=dev, dtype=torch.int32), torch.tensor([0, 300], device=dev, dtype=torch.int32)
    want = prompt_attention(*a, ca)[0], prompt_attention(*b, cb)[0]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        with torch.cuda.stream(s1):
            x = prompt_attention(*a, ca)[0]
        with torch.cuda.stream(s2):
            y = prompt_attention(*b, cb)[0]
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = prompt_attention(*a, ca)[0]
    for z in (a[0], a[1], a[2]):
        z.copy_(z.flip(0))
    ca.copy_(torch.tensor([0, 400, 650], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, prompt_attention(*a, ca)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("below", [5, 9, 11, 13, 15, 16.5])
@pytest.mark.parametrize("n", [2, 300, 2500])
def test_one_heavy_key_beside_light_ones(n, below, dtype):
    """A key of weight near one whose value is zero: the output is what the others, each of weight e^-below, bring.

    Their weights are rounded to q's type.  In bf16 that is half a step of each, whatever its size.  fp16 has steps of 2^-24 below
    2^-14, and a weight enters as 2^7 times itself relative to a reference that is at most the row's maximum: off by at most u of itself
    or by 2^-25 / 2^7 = 2^-32 of the largest weight."""
    q, k, v = torch.zeros(1, 2, D), torch.zeros(n, 1, D), torch.ones(n, 1, D)
    q[..., 0], k[:, 0, 0] = 16.0, -below
    at = n // 3
    k[at], v[at] = 0.0, 0.0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    o, lse = _run(q, k, v, [0, 1], [0, n])
    ro, rl, mag, big = opk.prompt_attention(q, k, v, [0, 1], [0, n])
    u = U[dtype]
    top = torch.exp(-rl).T[..., None]                     # the heavy key's weight
    tol = (2 * u + 2.0 ** -15 * big[..., None] + 2.0 ** -18) * mag + (2.0 ** -32 * top * (n - 1) + 2.0 ** -25 if dtype == torch.float16 else 0.0)
    off = (o.cpu().double() - ro).abs()
    assert (off <= tol).all(), (off / ro).max()
    assert ((lse.cpu().double() - rl).abs() <= 2.0 ** -16 * big.T + 2.0 ** -18 * (1 + rl.abs())).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("e", [0, 12, 16, 20, 24])
def test_large_scores_that_grow_from_tile_to_tile(e, dtype):
    """Maxima that rise a little with every tile of keys, at scores from one to 2^24: weights are at most one, so an output is between the
    smallest and the largest value; rounded weights and their sum, each off by u, and the output's own rounding leave 4 u of that."""
    n = 900
    q, k = torch.zeros(n, 2, D), torch.zeros(n, 1, D)
    q[..., 0] = 2.0 ** (e // 2)
    k[:, 0, 0] = 2.0 ** (e - e // 2)
    q[..., 1], k[:, 0, 1] = 1.0, torch.arange(n) // 100 * 4.0
    v = 1.0 + (torch.arange(n)[:, None, None] % 7).expand(n, 1, D) / 8.0
    o, lse = _run(q.to(dtype), k.to(dtype), v.to(dtype), [0, n], scale=1.0)
    o = o.cpu().double()
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    assert (o >= 1.0 - 4 * U[dtype]).all() and (o <= 1.75 * (1 + 4 * U[dtype])).all()
