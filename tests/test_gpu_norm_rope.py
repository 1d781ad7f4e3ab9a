"""norm_rope_heads against its formula in 64 bits.

Tolerance, with u half a step of the output type: the square sum (8 in a row, then 5 levels), rsqrt (2 ulp) and three products are off by less
than 2^-20 relatively; cos and sin by less than 2^-21 (angles reduced in 64 bits, then 2 ulp); a rotation adds two products.  So an
output is off by at most u |o| + 2^-19 (|y_f| + |y_{f+F}|), and 2^-25 in fp16 below its normal range."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 256
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _inputs(B, t, H, G, F, n, gated=True, dtype=torch.bfloat16, far=300000, seed=0):
    _dev()
    g = torch.Generator().manual_seed(seed)
    qg = torch.randn(B, t, H, (2 if gated else 1) * D, generator=g).to(dtype)
    kl = torch.randn(B, t, G, D, generator=g).to(dtype) * 5
    qw, kw = torch.randn(D, generator=g) * 0.2, torch.randn(D, generator=g) * 0.2
    pos = torch.randint(0, far, (n, B, t), generator=g)
    inv = (1e7 ** (-torch.arange(F, dtype=torch.float64) / max(F, 1))).float()
    axes = torch.randint(0, n, (F,), generator=g).tolist()
    return [x.cuda() for x in (qg, kl, qw, kw, pos, inv)] + [axes]


def _formula(x, w, pos, inv, axes, eps=1e-6):
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1 + w.double())
    F = len(axes)
    o, a = y.clone(), torch.zeros_like(y)
    if F:
        ang = (pos[axes].double() * inv.double()[:, None, None]).permute(1, 2, 0)[:, :, None]
        o[..., :F] = y[..., :F] * torch.cos(ang) - y[..., F:2 * F] * torch.sin(ang)
        o[..., F:2 * F] = y[..., F:2 * F] * torch.cos(ang) + y[..., :F] * torch.sin(ang)
        a[..., :F] = a[..., F:2 * F] = y[..., F:2 * F].abs()
    return y, o.transpose(1, 2), (y.abs() + a).transpose(1, 2)


def _check(got, want, size):
    u = U[got.dtype]
    err = (got.double() - want).abs()
    assert (err <= u * want.abs() + 2.0 ** -19 * size + (2.0 ** -25 if got.dtype == torch.float16 else 0)).all(), err.max()


def _check_all(args, out, eps=1e-6, memory=True):
    qg, kl, qw, kw, pos, inv, axes = args
    q, k, qr, kr = out
    for x, w, plain, turned in ((qg[..., :D], qw, q, qr), (kl, kw, k, kr)):
        y, o, size = _formula(x, w, pos.reshape(-1, *pos.shape[-2:]), inv, axes, eps)
        _check(turned, o, size)
        if memory:
            _check(plain, y, y.abs())
        else:
            assert plain is None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,t,H,G,F,n,gated,memory", [
    (1, 1, 24, 4, 32, 3, True, True), (64, 1, 24, 4, 32, 3, True, False), (3, 131, 6, 1, 32, 3, True, True), (1, 1000, 8, 8, 8, 2, False, True),
    (2, 77, 1, 1, 128, 4, True, True), (1, 33, 5, 3, 64, 1, True, False), (2, 9, 7, 2, 0, 1, False, True), (1, 9000, 2, 1, 16, 3, True, True)])
def test_against_the_formula(B, t, H, G, F, n, gated, memory, dtype):
    from heimdall_b200 import norm_rope_heads
    args = _inputs(B, t, H, G, F, n, gated, dtype)
    out = norm_rope_heads(*args[:5], args[5] if F else None, axes=args[6] or None if n == 1 else args[6], gated=gated, memory=memory)
    _check_all(args, out, memory=memory)


def test_positions_32_bits_strides_and_far_positions():
    from heimdall_b200 import norm_rope_heads
    args = _inputs(2, 40, 4, 2, 32, 3, far=2 ** 31 - 1)
    a = norm_rope_heads(*args[:6], axes=args[6])
    _check_all(args, a)
    b = norm_rope_heads(*args[:4], args[4].int(), args[5], axes=args[6])
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    # query, gate, keys as views of one projection; positions expanded over the batch
    g = torch.Generator().manual_seed(5)
    both = torch.randn(2, 40, 4 * 512 + 2 * 256 + 8, generator=g).bfloat16().cuda()
    qg, kl = both[..., :2048].unflatten(2, (4, 512)), both[..., 2048:2560].unflatten(2, (2, 256))
    pos = args[4][:, :1].expand(3, 2, 40)
    c = norm_rope_heads(qg, kl, args[2], args[3], pos, args[5], axes=args[6])
    _check_all([qg, kl, args[2], args[3], pos, args[5], args[6]], c)
    # an odd offset in memory: copied
    odd = torch.randn(2 * 40 * 2 * 256 + 1, generator=g).bfloat16().cuda()[1:].view(2, 40, 2, 256)
    d = norm_rope_heads(qg, odd, args[2], args[3], pos, args[5], axes=args[6])
    _check_all([qg, odd, args[2], args[3], pos, args[5], args[6]], d)


def test_rows_of_zeros_and_of_special_values():
    from heimdall_b200 import norm_rope_heads
    args = _inputs(1, 4, 2, 1, 32, 3)
    args[0][0, 0] = 0
    args[0][0, 1, 0, 3] = float("nan")
    args[0][0, 2, 1, 300] = float("inf")          # the gate: not read
    q, k, qr, kr = norm_rope_heads(*args[:6], axes=args[6])
    assert not q[0, 0].any() and not qr[0, :, 0].any()
    assert q[0, 1, 0].isnan().all() and qr[0, 0, 1].isnan().all() and not q[0, 1, 1].isnan().any()
    args[0][0, 1, 0, 3] = 0
    _check_all(args, norm_rope_heads(*args[:6], axes=args[6]))


def test_empty_and_refused_calls():
    from heimdall_b200 import norm_rope_heads
    args = _inputs(2, 5, 4, 2, 32, 3)
    empty = norm_rope_heads(args[0][:, :0], args[1][:, :0], args[2], args[3], args[4][..., :0], args[5], axes=args[6])
    assert empty[2].shape == (2, 4, 0, 256)
    qg, kl, qw, kw, pos, inv, axes = args
    for bad in (lambda: norm_rope_heads(qg, kl, qw, kw, pos, inv),                                # three axes, none named
                lambda: norm_rope_heads(qg, kl, qw, kw, pos[:, :, :4], inv, axes=axes),
                lambda: norm_rope_heads(qg, kl, qw, kw, pos.float(), inv, axes=axes),
                lambda: norm_rope_heads(qg, kl, qw, kw, pos, inv, axes=axes[:-1]),
                lambda: norm_rope_heads(qg, kl, qw, kw, pos, inv, axes=[3] + axes[1:]),
                lambda: norm_rope_heads(qg, kl, qw, kw, pos, inv, axes=axes, gated=False),
                lambda: norm_rope_heads(qg, kl.half(), qw, kw, pos, inv, axes=axes),
                lambda: norm_rope_heads(qg, kl, qw[:-1], kw, pos, inv, axes=axes)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        norm_rope_heads(qg, kl, qw, kw, pos, inv[:30], axes=axes[:30])
    with pytest.raises(NotImplementedError, match="no backward"):
        norm_rope_heads(qg, kl, qw.requires_grad_(), kw, pos, inv, axes=axes)


def test_captured_and_replayed_on_another_stream():
    from heimdall_b200 import norm_rope_heads
    args = _inputs(3, 7, 6, 2, 32, 3)
    norm_rope_heads(*args[:6], axes=args[6])
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        out = norm_rope_heads(*args[:6], axes=args[6])
    args[4].add_(11)
    args[0].mul_(2)
    g.replay()
    _check_all(args, out)


def test_layer_with_positions_on_several_axes():
    """BifrostAttention.project: text positions give what the one-axis prologue gives, to its second rounding."""
    _dev()
    from heimdall_b200 import BifrostAttention, BifrostLayer
    from params import layer_params, proj_params
    p = layer_params(4, 2, 256, 512, 64, 4, 0, 1)
    pp = proj_params(4, 2, 256, 512, 1, 64, 1e7)
    L = BifrostLayer.from_params(p, torch.device("cuda"))
    A = BifrostAttention(pp.q_w, pp.k_w, pp.v_w, pp.o_w, pp.q_norm_w, pp.k_norm_w, L, pp.rot, pp.theta, pp.eps, pp.gated, rope_sections=(11, 11, 10))
    x = torch.randn(2, 50, 512, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    text = torch.arange(7, 57, device="cuda").expand(3, 2, 50)
    a, b = A.project(x, 7), A.project(x, 0, text)
    c = A.project(x, 0, text[0])
    for i, (u, v, w) in enumerate(zip(a, b, c)):
        assert torch.equal(v, w)
        if i in (2, 5):
            assert torch.equal(u, v)
        else:       # each side rounds q and k once (up to a step between them), qr and kr of the first side twice
            assert ((u.double() - v.double()).norm() / v.double().norm()) < 2.0 ** -8
    image = text.clone()
    image[1, :, 10:20] += 3
    image[2, :, 10:20] += 5
    d = A.project(x, 0, image)
    _check_all([d[5].view(2, 50, 4, 512), torch.nn.functional.linear(x, A.k_w).view(2, 50, 2, 256), A.q_norm_w, A.k_norm_w, image, A.inv_freq, A.axes],
               (d[0], d[1], d[3], d[4]), pp.eps)
    y = A.forward(x, {}, 0, image)
    assert y.shape == (2, 50, 512) and y.isfinite().all()
    with pytest.raises(ValueError):
        BifrostAttention(pp.q_w, pp.k_w, pp.v_w, pp.o_w, pp.q_norm_w, pp.k_norm_w, L, pp.rot, pp.theta, pp.eps, pp.gated, rope_sections=(11, 11, 11))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("F,memory", [(32, True), (32, False), (8, True), (64, False), (0, True)])
def test_infinities_reach_what_the_formula_says(F, memory, dtype):
    """An infinity makes its own dim NaN, its partner where both are turned, and the rest of its head 0."""
    from heimdall_b200 import norm_rope_heads
    args = _inputs(1, 3, 2, 1, F, 1, dtype=dtype)
    for t, at in enumerate((3, 200, 2 * F)):
        args[0][0, t, 0, at] = float("inf")
    args[1][0, 1, 0, 255] = -float("inf")
    out = norm_rope_heads(*args[:5], args[5] if F else None, axes=args[6] or None, memory=memory)
    for x, w, plain, turned in ((args[0][..., :D], args[2], out[0], out[2]), (args[1], args[3], out[1], out[3])):
        y, o, size = _formula(x, w, args[4], args[5], args[6])
        for got, want, mag in ((turned, o, size),) + (((plain, y, y.abs()),) if memory else ()):
            assert torch.equal(got.isnan(), want.isnan())
            _check(got[~got.isnan()], want[~want.isnan()], mag[~want.isnan()])


def test_weights_and_positions_on_any_boundary():
    """The norm weights, the frequencies and the positions may begin anywhere in a larger buffer."""
    from heimdall_b200 import norm_rope_heads
    args = _inputs(2, 5, 4, 2, 32, 3)
    want = norm_rope_heads(*args[:6], axes=args[6])
    off = [torch.cat([z.new_zeros(1), z.reshape(-1)])[1:].view(z.shape) for z in args[2:6]]
    assert off[0].data_ptr() % 16 and off[2].is_contiguous()
    for a, b in zip(norm_rope_heads(*args[:2], *off, axes=args[6]), want):
        assert torch.equal(a, b)
