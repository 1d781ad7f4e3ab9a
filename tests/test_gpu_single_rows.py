"""The serving calls on a single row cut out of a wider one, whose width is no multiple of 8: the strides of dimensions of one mean nothing, and the results
are those of the same values laid out on their own, bit by bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 256


def _cut(*shape, seed, dtype=torch.bfloat16, width=217):
    """Random values of this shape, whose dimensions but the last one or two are one: the same in a wider row, and on their own."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    n = 1
    for s in shape:
        n *= s
    wide = torch.randn(3, n + width, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    lead = [1 for s in shape[:-1] if s == 1]
    row = wide[0:1, :n].reshape(*lead, *shape[len(lead):])
    row = row.as_strided(row.shape, [n + width] * len(lead) + list(row.stride()[len(lead):]))
    assert (n + width) % 8 and row.is_contiguous() and row.data_ptr() == wide.data_ptr()
    return row, row.clone(memory_format=torch.contiguous_format).view(-1).view(shape)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapters_of_one_token(dtype):
    x, x1 = _cut(1, 136, seed=1, dtype=dtype)
    y, y1 = _cut(1, 72, seed=2, dtype=dtype)
    from heimdall_b200 import Adapters
    g = torch.Generator().manual_seed(3)
    ad = Adapters([torch.randn(16, 136, generator=g).to(dtype).cuda()], [torch.randn(72, 16, generator=g).to(dtype).cuda()])
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = ad.add(y1, x1, ids)
    assert torch.equal(ad.add(y, x, ids), want) and torch.equal(ad.add(y, x, ids, out=y), want)


def test_norm_and_rotation_of_one_token():
    from heimdall_b200 import norm_rope_heads
    qg, qg1 = _cut(1, 1, 2, 2 * D, seed=1)
    kl, kl1 = _cut(1, 1, 1, D, seed=2)
    w, pos = torch.zeros(D, device="cuda"), torch.full((1, 1), 77, device="cuda")
    inv = 0.5 ** torch.arange(32, device="cuda", dtype=torch.float32)
    for a, b in zip(norm_rope_heads(qg, kl, w, w, pos, inv), norm_rope_heads(qg1, kl1, w, w, pos, inv)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("share", [False, True])
def test_pages_of_one_sequence(share):
    from heimdall_b200 import PagedKV
    k, k1 = _cut(1, 1, 1, D, seed=1)
    v, v1 = _cut(1, 1, 1, D, seed=2)
    q, q1 = _cut(1, 1, 2, D, seed=3)
    c = PagedKV(1, 4, 1, 2, page=16)
    got = []
    for slot, (a, b, x) in enumerate(((k, v, q), (k1, v1, q1))):
        c.reserve([slot], 1)
        ids = torch.tensor([slot], device="cuda")
        c.append(0, a, b, ids)
        got.append(c.attend(0, x, shared=c.share([slot]))[0] if share else c.attend(0, x, ids)[0])
    assert torch.equal(got[0], got[1])


def test_prompt_of_one_token():
    from heimdall_b200 import prompt_attention
    q, q1 = _cut(1, 1, D, seed=1)
    k, k1 = _cut(1, 1, D, seed=2)
    v, v1 = _cut(1, 1, D, seed=3)
    cu = torch.tensor([0, 1], device="cuda")
    assert torch.equal(prompt_attention(q, k, v, cu)[0], prompt_attention(q1, k1, v1, cu)[0])
