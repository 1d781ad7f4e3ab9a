"""Adapters.add against its formula in 64 bits.

Tolerance.  u is half a step of the output type, S = |s| sum_r |B_r| sum_i |A_ri x_i|, P = |s| sum_r |B_r h_r|:
  * a chain of sums for h has at most d_in / 16 + 64 additions (steps of 16 values, then warps and parts), each off by at most 2^-23 of the sum of the
    magnitudes: (d_in / 32 + 32) 2^-22 S;
  * h enters as two parts: 2^-16 (bf16) or 2^-21 (fp16) of itself; the second product has at most 16 additions: 2^-18 P in all;
  * out is rounded once: u |out|, and 2^-25 in fp16 below its normal range.
With whole numbers that all sums hold exactly, out is the rounded exact value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _make(ranks, d_in, d_out, dtype=torch.bfloat16, scale=None, seed=0):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from heimdall_b200 import Adapters
    g = torch.Generator().manual_seed(seed)
    a = [(torch.randn(r, d_in, generator=g) * d_in ** -0.5).to(dtype).cuda() for r in ranks]
    b = [(torch.randn(d_out, r, generator=g) * r ** -0.5).to(dtype).cuda() for r in ranks]
    s = [0.5 + 0.25 * i for i in range(len(ranks))] if scale is None else scale
    return Adapters(a, b, s), a, b, s


def _data(T, d_in, d_out, dtype=torch.bfloat16, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, d_in, generator=g).to(dtype).cuda(), torch.randn(T, d_out, generator=g).to(dtype).cuda()


def _check(got, x, y, ids, a, b, s):
    want, S, P = y.double(), torch.zeros_like(y, dtype=torch.float64), torch.zeros_like(y, dtype=torch.float64)
    for i in range(len(a)):
        rows = torch.nonzero(ids == i)[:, 0]
        xd, ad, bd = x[rows].double(), a[i].double(), b[i].double()
        h = xd @ ad.T
        want[rows] += s[i] * (h @ bd.T)
        S[rows] = abs(s[i]) * (xd.abs() @ ad.abs().T) @ bd.abs().T
        P[rows] = abs(s[i]) * h.abs() @ bd.abs().T
    two = 2.0 ** -16 if x.dtype == torch.bfloat16 else 2.0 ** -21
    tol = U[x.dtype] * want.abs() + (x.shape[1] / 32 + 32) * 2.0 ** -22 * S + (two + 2.0 ** -18) * P + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,ranks,d_in,d_out", [
    (1, [16], 64, 8), (1, [3], 8, 264), (17, [8, 16, 1], 1000, 1000), (64, [16] * 40, 512, 600), (200, [128, 5, 64], 2056, 520), (256, [16] * 3, 1024, 256),
    (257, [16] * 3, 1000, 264), (300, [32, 7], 64, 1032), (777, [64, 16, 100], 520, 328), (2500, [128, 8, 33, 64], 136, 72), (1500, [16] * 700, 64, 16)])
def test_against_the_formula(T, ranks, d_in, d_out, dtype):
    ad, a, b, s = _make(ranks, d_in, d_out, dtype)
    x, y = _data(T, d_in, d_out, dtype)
    g = torch.Generator().manual_seed(T)
    for ids in (torch.randint(-1, len(ranks), (T,), generator=g), torch.arange(T) * len(ranks) // T, torch.full((T,), len(ranks) - 1)):
        ids = ids.cuda()
        _check(ad.add(y, x, ids), x, y, ids, a, b, s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,ranks,d_in,d_out", [(5000, [128, 64, 16, 1], 4104, 392), (2600, [64] * 7, 8, 8), (2049, [8], 1160, 136), (20100, [32, 16], 1032, 264)])
def test_groups_that_several_ctas_share(T, ranks, d_in, d_out, dtype):
    """More steps than CTAs, groups cut anywhere, groups of a CTA's own between two that it shares, and groups of one step."""
    ad, a, b, s = _make(ranks, d_in, d_out, dtype)
    x, y = _data(T, d_in, d_out, dtype, seed=T)
    ids = torch.randint(-1, len(ranks), (T,), generator=torch.Generator().manual_seed(T)).cuda()
    ids[T // 3:T // 2] = 0
    first = ad.add(y, x, ids)
    _check(first, x, y, ids, a, b, s)
    assert torch.equal(first, ad.add(y, x, ids))           # the parts are added in their order, whoever is last
    assert torch.equal(first, ad.add(y, x, ids, out=y))


@pytest.mark.parametrize("T", [40, 700])
def test_whole_numbers_are_exact(T):
    from heimdall_b200 import Adapters
    _make([1], 8, 8)
    g = torch.Generator().manual_seed(3)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g)
    ranks, d_in, d_out = [16, 40, 128], 328, 136
    a, b = [whole(r, d_in) for r in ranks], [whole(d_out, r) for r in ranks]
    for dtype in (torch.bfloat16, torch.float16):
        cu = lambda ts: [t.to(dtype).cuda() for t in ts]
        x, y, ids = whole(T, d_in), whole(T, d_out) * 64, torch.randint(-1, 3, (T,), generator=g)
        got = Adapters(cu(a), cu(b), [0.5, -2.0, 0.25]).add(*cu([y, x]), ids.cuda())
        want = y.double()
        for i, s in enumerate((0.5, -2.0, 0.25)):
            rows = ids == i
            want[rows] += s * ((x[rows].double() @ a[i].double().T) @ b[i].double().T)
        assert torch.equal(got.cpu(), want.to(dtype))


@pytest.mark.parametrize("T", [1, 30, 600])
def test_no_adapter_and_numbers_out_of_range(T):
    ad, a, b, s = _make([16, 8], 64, 48)
    x, y = _data(T, 64, 48)
    x[0] = float("nan")                         # not read
    y[-1, 3] = float("inf")
    ids = torch.full((T,), -1)
    ids[1::3], ids[2::3] = 2, 2 ** 31 - 1
    assert torch.equal(ad.add(y, x, ids.int().cuda()), y)
    ids[2::3] = 2 ** 40                         # not 0 after a cut to 32 bits
    ids[1::3] = -2 ** 33 + 1
    z = y.clone()
    assert ad.add(z, x, ids.cuda(), out=z) is z and torch.equal(z, y)


@pytest.mark.parametrize("T", [24, 500])
def test_values_that_are_not_finite_stay_in_their_rows(T):
    ad, a, b, s = _make([16, 16], 128, 64)
    x, y = _data(T, 128, 64)
    ids = (torch.arange(T) % 2).cuda()
    clean = ad.add(y, x, ids)
    x[4, 7], x[9, 0] = float("nan"), float("inf")
    got = ad.add(y, x, ids)
    assert got[4].isnan().all() and got[9].isnan().all()
    rest = [t for t in range(T) if t not in (4, 9)]
    assert torch.equal(got[rest], clean[rest])
    x[4], x[9] = 0, 0
    got = ad.add(y, x, ids)
    assert torch.equal(got[[4, 9]], y[[4, 9]])


@pytest.mark.parametrize("T", [50, 700])
def test_large_and_small_products_in_fp16(T):
    """h beyond fp16's range and far below it: its rows are scaled."""
    ad, a, b, s = _make([16], 64, 32, torch.float16)
    x, y = _data(T, 64, 32, torch.float16)
    x[::2] *= 30000 / 5
    x[1::2] *= 2.0 ** -13
    ids = torch.zeros(T, dtype=torch.int32, device="cuda")
    from heimdall_b200 import Adapters
    big = [t * 20 for t in a]
    small = [t * 2.0 ** -8 for t in b]
    _check(Adapters(big, small, s).add(y, x, ids), x, y, ids, big, small, s)


@pytest.mark.parametrize("B,t", [(3, 7), (4, 130)])
def test_strides_shapes_and_in_place(B, t):
    ad, a, b, s = _make([16, 32], 136, 72)
    g = torch.Generator().manual_seed(9)
    both = torch.randn(B, t, 136 + 72 + 8, generator=g).bfloat16().cuda()
    x, y = both[..., :136], both[..., 136:208]
    ids = torch.randint(-1, 2, (B, t), generator=g).cuda()
    flat = lambda z: z.reshape(B * t, -1)
    got = ad.add(y, x, ids)
    assert got.shape == y.shape and got.is_contiguous()
    _check(flat(got), flat(x), flat(y), ids.reshape(-1), a, b, s)
    odd = torch.empty(B * t * 136 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(B, t, 136).copy_(x)
    assert torch.equal(ad.add(y, odd, ids), got)
    assert torch.equal(ad.add(y, x.transpose(0, 1).contiguous().transpose(0, 1), ids.int()), got)
    z = y.contiguous()
    assert torch.equal(ad.add(z, x, ids, out=z), got)
    one = ids[:, :1].expand(B, t)
    _check(flat(ad.add(y, x, one)), flat(x), flat(y), one.reshape(-1), a, b, s)
    with pytest.raises(ValueError, match="overlap"):
        buf = torch.zeros(B * t * 72 + 72, dtype=torch.bfloat16, device="cuda")
        ad.add(buf[72:].view(B, t, 72), x, ids, out=buf[:-72].view(B, t, 72))


def test_empty_and_refused_calls():
    ad, *_ = _make([16], 64, 32)
    x, y = _data(6, 64, 32)
    ids = torch.zeros(6, dtype=torch.int64, device="cuda")
    assert ad.add(y[:0], x[:0], ids[:0]).shape == (0, 32)
    for bad in ((y, x[:, :56], ids), (y[:5], x, ids), (y, x, ids[:5]), (y, x.half(), ids), (y.half(), x, ids), (y, x, ids.float())):
        with pytest.raises(ValueError):
            ad.add(*bad)
    with pytest.raises(ValueError):
        ad.add(y, x, ids, out=y.float())
    with pytest.raises(NotImplementedError, match="no backward"):
        ad.add(y, x.clone().requires_grad_(), ids)
    with pytest.raises(RuntimeError):
        ad.add(y.cpu(), x, ids)


@pytest.mark.parametrize("T", [40, 600])
def test_captured_replayed_and_on_two_streams(T):
    ad, a, b, s = _make([16, 16, 64], 512, 264)
    x, y = _data(T, 512, 264)
    ids = (torch.arange(T) % 4 - 1).cuda().int()
    ad.add(y, x, ids)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = ad.add(y, x, ids)
        out2 = ad.add(out, x, ids)
    x.mul_(-1.5)
    ids.copy_((torch.arange(T) % 3).int())
    torch.cuda.synchronize()
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):          # another call at the same time
            z = ad.add(y, x, ids)
    torch.cuda.synchronize()
    _check(out, x, y, ids, a, b, s)
    _check(out2, x, out, ids, a, b, s)
    assert torch.equal(z, out)


def test_layer_with_adapters():
    """BifrostAttention with adapters on all projections: one call for a batch equals the layer with each request's merged weights, to the roundings of
    the merged weights and of the projections (2^-8 each of bf16 values that enter sums)."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from heimdall_b200 import Adapters, BifrostAttention, BifrostLayer
    from params import layer_params, proj_params
    p, pp = layer_params(4, 2, 256, 512, 64, 4, 0, 1), proj_params(4, 2, 256, 512, 1, 64, 1e7)
    L = BifrostLayer.from_params(p, torch.device("cuda"))
    g = torch.Generator().manual_seed(4)
    w = {"q": pp.q_w, "k": pp.k_w, "v": pp.v_w, "o": pp.o_w}
    low = {n: ([(torch.randn(8, t.shape[1], generator=g) * t.shape[1] ** -0.5).bfloat16().cuda() for _ in range(2)],
               [(torch.randn(t.shape[0], 8, generator=g) * 0.05).bfloat16().cuda() for _ in range(2)]) for n, t in w.items()}
    layer = lambda ws, **kw: BifrostAttention(*(ws[n] for n in "qkvo"), pp.q_norm_w, pp.k_norm_w, L, pp.rot, pp.theta, pp.eps, pp.gated, **kw)
    A = layer(w, adapters={n: Adapters(*ab, 2.0) for n, ab in low.items()})
    x = torch.randn(3, 90, 512, generator=g).bfloat16().cuda()
    ids = torch.tensor([1, -1, 0], device="cuda")
    y = A.forward(x, {}, 0, adapter_ids=ids)
    for b, i in enumerate(ids.tolist()):
        ws = {n: t.cuda().float() + (0 if i < 0 else 2.0 * low[n][1][i].float() @ low[n][0][i].float()) for n, t in w.items()}
        one = layer(ws).forward(x[b:b + 1], {}, 0)
        assert ((y[b:b + 1].double() - one.double()).norm() / one.double().norm()) < 0.02
    assert torch.equal(A.forward(x, {}, 0)[1], y[1])
    with pytest.raises(ValueError):
        layer(w, adapters={"q": Adapters(*low["k"])})
    for bad in (ids[:2], ids.float(), ids[:, None].expand(3, 4)):
        with pytest.raises(ValueError):
            A.project(x, 0, adapter_ids=bad)
    assert torch.equal(A.project(x, 0, adapter_ids=ids.int())[5], A.project(x, 0, adapter_ids=ids[:, None].expand(3, 90))[5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,rank", [(1, 16), (1, 3), (24, 16), (24, 48), (300, 16)])
def test_a_token_alone_with_its_adapter_that_is_not_finite(T, rank, dtype):
    """A x of infinities, or of sums beyond fp32, makes the whole row NaN, as it does beside other tokens of the adapter.  (Weights of one sign: infinities
    of both signs would become NaN by themselves.)"""
    from heimdall_b200 import Adapters
    _, a, b, s = _make([rank] * T, 64, 48, dtype)
    a, b = [t.abs() + 2.0 ** -6 for t in a], [t.abs() + 2.0 ** -6 for t in b]
    ad = Adapters(a, b, s)
    x, y = _data(T, 64, 48, dtype)
    ids = torch.arange(T).cuda()
    clean = ad.add(y, x, ids)
    for row, value in ((T // 2, float("nan")), (T - 1, -float("inf")), (0, float("inf"))):
        x[row, 5] = value
    bad = sorted({0, T // 2, T - 1})
    got = ad.add(y, x, ids)
    assert got[bad].isnan().all()
    rest = [t for t in range(T) if t not in bad]
    assert torch.equal(got[rest], clean[rest])
    if dtype == torch.bfloat16:                  # finite values whose A x is beyond fp32
        x, y = _data(T, 64, 48)
        x[0] = 3e38
        got = Adapters([16 * t + 1 for t in a], b, s).add(y, x, ids)
        assert got[0].isnan().all() and got[1:].isfinite().all()
