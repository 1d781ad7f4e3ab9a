"""A decode step as a server of many requests runs it: every sequence at its own position and with its own adapters, over a cache in which the
sequences are forks of one prompt.  Each stage is compared with its formula in 64 bits on the values that entered it (the stages' own tests derive the
tolerances), so that the chain as a whole is checked without an error of one stage standing for another's."""
import pytest
import torch

from oracle import paged_kv as opk
from params import layer_params, proj_params
from test_gpu_norm_rope import _check_all
from test_gpu_paged import _host
from test_gpu_paged_shared import _check_out

pytestmark = pytest.mark.gpu
H, G, D, DIM, SECTIONS, RANKS = 4, 2, 256, 512, (11, 11, 10), (8, 24)


def _layer(seed=4):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from heimdall_b200 import Adapters, BifrostAttention, BifrostLayer
    p, pp = layer_params(H, G, D, DIM, 64, 4, 0, 1), proj_params(H, G, D, DIM, 1, 64, 1e7)
    g = torch.Generator().manual_seed(seed)
    w = {"q": pp.q_w, "k": pp.k_w, "v": pp.v_w, "o": pp.o_w}
    low = {n: ([(torch.randn(r, t.shape[1], generator=g) * t.shape[1] ** -0.5).bfloat16().cuda() for r in RANKS],
               [(torch.randn(t.shape[0], r, generator=g) * 0.1).bfloat16().cuda() for r in RANKS]) for n, t in w.items()}
    A = BifrostAttention(pp.q_w, pp.k_w, pp.v_w, pp.o_w, pp.q_norm_w, pp.k_norm_w, BifrostLayer.from_params(p, torch.device("cuda")), pp.rot,
                         pp.theta, pp.eps, pp.gated, rope_sections=SECTIONS, adapters={n: Adapters(*ab, [2.0, 0.5]) for n, ab in low.items()})
    return A, low


def _check_linear(got, x, w, low, ids):
    """y0 = W x in fp32 (two roundings of bf16 with the adapter's sum, each half a step: of y0 and of the result), 2^-16 of the adapter's product and the sums' own 2^-22
    of the magnitudes for each of (d / 16) additions."""
    x, w = x.double().reshape(-1, x.shape[-1]), w.double()
    y0, size = x @ w.T, x.abs() @ w.abs().T
    add = torch.zeros_like(y0)
    part = torch.zeros_like(y0)
    for t, i in enumerate(ids.reshape(-1).tolist()):
        if 0 <= i < len(RANKS):
            h, s = low[0][i].double() @ x[t], (2.0, 0.5)[i]
            add[t], part[t] = s * low[1][i].double() @ h, s * low[1][i].double().abs() @ (low[0][i].double().abs() @ x[t].abs())
    got = got.double().reshape(y0.shape)
    tol = 2.0 ** -8 * ((y0 + add).abs() + 1.01 * y0.abs()) + 2.0 ** -15 * part + (w.shape[1] / 16 + 32) * 2.0 ** -22 * (size + part)
    assert ((got - y0 - add).abs() <= tol).all(), ((got - y0 - add).abs() / tol).max()


def _prompt(A, n, ways, spare=64, page=32):
    """A cache whose slots 0 .. ways - 1 continue one prompt of n tokens (image patches in its midst: three axes of positions)."""
    from heimdall_b200 import PagedKV
    c = PagedKV(layers=1, pages=-(-n // page) + ways * (2 + spare // page), heads=G, slots=ways + 1, page=page, max_len=n + spare)
    g = torch.Generator().manual_seed(n)
    x = torch.randn(1, n, DIM, generator=g).bfloat16().cuda()
    pos = torch.arange(n).repeat(3, 1, 1)
    patch = torch.arange(64)
    for axis, at in enumerate((0 * patch, patch // 8, patch % 8)):
        pos[axis, 0, 100:164] = 100 + at
    pos[:, :, 164:] -= 64 - 8
    q, k, v, qr, kr, qg = A.project(x, 0, pos.cuda(), torch.tensor([0], device="cuda"))
    from heimdall_b200 import retrieval
    o = retrieval.teacher(qr, kr, v, c.layer(0))
    assert A.output(o.float(), qg, x, torch.tensor([0], device="cuda")).isfinite().all()
    c.fork([0] * (ways - 1), list(range(1, ways)))
    return c, int(pos.max()) + 1


def test_step_of_many_requests():
    from heimdall_b200 import retrieval
    A, low = _layer()
    ways = 7
    c, at = _prompt(A, 6200, ways)
    g = torch.Generator().manual_seed(5)
    for step, t in enumerate((1, 3, 1)):
        x = torch.randn(ways, t, DIM, generator=g).bfloat16().cuda()
        ids = torch.tensor([1, -1, 0, 0, 1, 5, 0], device="cuda")[:, None].expand(ways, t)
        pos = (at + torch.arange(t)[None, :] + 5 * torch.arange(ways)[:, None]).expand(3, ways, t).contiguous().cuda()
        q, k, v, qr, kr, qg = A.project(x, 0, pos, ids)
        _check_linear(qg, x, A.q_w, low["q"], ids)
        _check_linear(v, x, A.v_w, low["v"], ids)
        kl = A._linear("k", x, ids)
        _check_linear(kl, x, A.k_w, low["k"], ids)
        _check_all([qg.view(ways, t, H, 2 * D), kl.view(ways, t, G, D), A.q_norm_w, A.k_norm_w, pos, A.inv_freq, A.axes], (q, k, qr, kr), A.eps)
        o = retrieval.teacher(qr, kr, v, c.layer(0, share=True))
        plan = c._layer_plans[ways][0]
        assert plan.runs == 1 and plan.slots == list(range(ways))
        qt = qr.transpose(1, 2).contiguous()
        again, lse = c.attend(0, qt, shared=plan, with_lse=True)
        assert torch.equal(o, again)
        _check_out(c, plan, qt.cpu(), o, lse)
        y = A.output(o.float(), qg, x, ids)
        gate = torch.sigmoid(qg.view(ways, t, H, 2 * D)[..., D:].double())
        z = (o.double() * gate).reshape(ways, t, H * D)
        zb = torch.empty(ways, t, H * D, device="cuda", dtype=torch.bfloat16)
        from heimdall_b200 import _lib
        from heimdall_b200.functional import ptr, stream_handle
        _lib.call("bf_attn_epilogue", ptr(o.float().contiguous()), ptr(qg), 1, ways, t, H, D, ptr(zb), stream_handle())
        assert ((zb.double() - z).abs() <= 2.0 ** -6 * z.abs() + 1e-30).all()          # the gate and the product in bf16, as the reference has them
        _check_linear(y, zb, A.o_w, low["o"], ids)
        at += t
    assert c.length(3) == 6200 + 5


def test_layer_makes_its_plan_anew():
    """After forks and cuts into shared pages, not after cuts of a sequence's own tokens (rejected drafts)."""
    from heimdall_b200 import retrieval
    A, _ = _layer()
    c, _ = _prompt(A, 13000, 4)
    g = torch.Generator().manual_seed(6)

    def step(B, t=1):
        q, k, v, qr, kr, qg = A.project(torch.randn(B, t, DIM, generator=g).bfloat16().cuda())
        o = retrieval.teacher(qr, kr, v, c.layer(0, share=True))
        plan = c.share(range(B))
        _, lse = c.attend(0, qr.transpose(1, 2), shared=plan, with_lse=True)
        if plan.runs:
            _check_out(c, plan, qr.transpose(1, 2).cpu(), o, lse)
        return c._layer_plans[B][0], c._layer_plans[B][0].plan.clone()

    plan, first = step(4, 5)
    assert plan.runs == 1
    c.truncate([0, 2], [13002, 13001])
    assert plan.good                               # drafts were taken back, the plan is as good as before
    c.truncate([1, 3], [13002, 13002])
    c.truncate([0, 1, 3], [13001] * 3)
    same, second = step(4)
    assert same is plan and torch.equal(first, second)
    c.truncate([1], [12345])
    assert not plan.good
    c.truncate([0, 2, 3], [12345] * 3)
    same, third = step(4)
    assert same is plan and plan.good and not torch.equal(first, third)
    c.free([3])
    assert not plan.good
    c.fork([0], [3])                               # shares what slot 0 has by now
    same, fourth = step(4)
    assert same is plan and plan.good and plan.runs == 1
    c.free([1, 2, 3])
    assert step(1)[0].runs == 0


def test_captured_step_with_its_plan():
    """The step is captured with its plan and replayed; the call that would have to make a plan is refused in a capture."""
    from heimdall_b200 import retrieval
    A, _ = _layer()
    c, at = _prompt(A, 1200, 3)
    x = torch.randn(3, 1, DIM, generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
    ids, pos = torch.tensor([0, 1, -1], device="cuda"), torch.full((3, 3, 1), at, device="cuda")
    q, k, v, qr, kr, qg = A.project(x, 0, pos, ids)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            c._layer_plan(3)
        z = x + 0
    plan = c.share(range(3), min_saved=1)
    assert plan.runs == 1 and c.share(range(3)).runs == 0
    run = lambda: (lambda p: (c.append(0, p[4].transpose(1, 2).contiguous(), p[2]),
                              A.output(c.attend(0, p[3].transpose(1, 2), shared=plan)[0].float(), p[5], x, ids))[1])(A.project(x, 0, pos, ids))
    c.reserve(range(3), 1)
    first = run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = run()
    c.truncate(range(3), [1200] * 3)
    c.reserve(range(3), 1)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    for _ in range(2):                             # new tokens at new positions, the same plan
        c.reserve(range(3), 1)
        x.normal_()
        pos.add_(1)
        g.replay()
        torch.cuda.synchronize()
        kc, ks, vc, vs = _host(c, 0)
        p = A.project(x, 0, pos, ids)
        ro, rl, mag, big = opk.attend(kc, ks, vc, vs, c.table[1].tolist(), int(c.lens[1]), p[3].transpose(1, 2)[1].cpu(), None)
        o = c.attend(0, p[3].transpose(1, 2), shared=plan)[0]
        assert ((o[1].cpu().double() - ro).abs() <= 2.0 ** -6 * mag + 2.0 ** -8 * mag.max()).all()
        assert torch.equal(y, A.output(o.float(), p[5], x, ids))
