"""``retrieval.teacher`` over the pages of a cache: a layer's progress belongs to the cache, whichever ``layer(i)`` object is used, and
follows what the cache does with its sequences.

Every case runs beside a twin: one layer's tokens written with ``append`` alone and read with ``attend``, from the same inputs.  The pages
of both hold the same bits (append is exact), and outputs are the same calls on the same operands, so they are compared bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D, H, G = 256, 8, 2


def _cache(layers=1, slots=2, **kw):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from heimdall_b200 import PagedKV
    return PagedKV(layers, 60, G, slots, **dict(dict(page=16, max_len=256), **kw))


def _qkv(B, t, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    return r(B, H, t, D), r(B, G, t, D), r(B, t, G, D)


def _direct(c, qr, kr, v, layer=0, reserve=True):
    """The same step with the cache's own calls."""
    B, t = v.shape[:2]
    if reserve:
        c.reserve(range(B), t)
    c.append(layer, kr.transpose(1, 2), v)
    return c.attend(layer, qr.transpose(1, 2))[0]


def _state(c):
    return [x.clone() for x in (c.k_pages.view(torch.uint8), c.v_pages.view(torch.uint8), c.k_scale, c.v_scale, c.table, c.lens)]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(_state(a) if not isinstance(a, list) else a, _state(b) if not isinstance(b, list) else b))


def _teacher(*a):
    from heimdall_b200.retrieval import teacher
    return teacher(*a)


@pytest.mark.parametrize("steps", [(1, 1, 1), (17, 17), (5, 5, 1, 6, 17), (40, 1, 1)])
def test_a_layer_fetched_afresh_goes_on(steps):
    c, twin = _cache(2), _cache()
    for i, t in enumerate(steps):
        qr, kr, v = _qkv(2, t, i)
        for layer in range(2):
            o = _teacher(qr, kr, v, c.layer(layer), None)
        want = _direct(twin, qr, kr, v)
        if i:                       # the first call's outputs are those of the keys and values themselves, not of their codes
            assert torch.equal(o, want), i
        assert c.lens.tolist() == twin.lens.tolist() == [sum(steps[:i + 1])] * 2
    for layer in range(2):
        assert torch.equal(c.k_pages[layer].view(torch.uint8), twin.k_pages[0].view(torch.uint8))
        assert torch.equal(c.v_scale[layer], twin.v_scale[0])


def test_truncate_free_and_fork_are_followed():
    c, twin = _cache(2, 4), _cache(2, 4)
    kept = [c.layer(0), c.layer(1)]

    def step(B, t, seed, layers):
        for i in range(2):
            qr, kr, v = _qkv(B, t, seed + 50 * i)
            o = _teacher(qr, kr, v, layers(i), None)
            want = _direct(twin, qr, kr, v, i, reserve=i == 0)
            yield o, want
    list(step(2, 30, 1, lambda i: kept[i]))
    for o, want in step(2, 4, 2, lambda i: kept[i]):
        assert torch.equal(o, want)
    for x in (c, twin):
        x.truncate([0, 1], [31, 33])             # rejected drafts, not as many of each sequence
    for o, want in step(2, 2, 3, lambda i: c.layer(i) if i else kept[0]):
        assert torch.equal(o, want)
    assert c.lens.tolist() == twin.lens.tolist() == [33, 35, 0, 0]
    for x in (c, twin):
        x.fork([0, 1], [2, 3])
        x.compact()
    for o, want in step(4, 1, 4, lambda i: kept[i]):
        assert torch.equal(o, want)
    for x in (c, twin):
        x.free(range(4))
    list(step(2, 30, 5, lambda i: kept[i]))
    for o, want in step(2, 1, 6, lambda i: kept[i]):
        assert torch.equal(o, want)
    assert _same(c, twin)


def test_a_sequence_behind_another_layer_or_written_directly_is_refused():
    """Where the host cannot tell whether a layer holds a sequence's tokens, the call is refused and changes nothing."""
    c = _cache(2, 3)
    qr, kr, v = _qkv(2, 1, 0)
    c.reserve([0, 1], 1)
    c.append(0, kr.transpose(1, 2), v)            # one-token prompts written directly
    before = _state(c)
    with pytest.raises(ValueError, match="in step|append"):
        _teacher(qr, kr, v, c.layer(0), None)
    assert _same(before, c) and c.length(0) == 1
    layer = c.layer(1)                            # room reserved before the call is used
    _teacher(qr, kr, v, layer, None)
    assert c.length(0) == 1 and layer.n == 1
    c.reserve([0, 1], 1)
    c.append(1, kr.transpose(1, 2), v, torch.tensor([1, 0], device="cuda"))
    before = _state(c)
    with pytest.raises(ValueError, match="in step|append"):
        _teacher(qr, kr, v, layer, None)
    assert _same(before, c)
    c.free([0, 1])
    _teacher(qr, kr, v, c.layer(0), None), _teacher(qr, kr, v, layer, None)
    assert c.lens.tolist() == [1, 1, 0]
    c.reserve([2], 5)                             # another sequence, served directly beside them
    x = _qkv(1, 5, 9)
    for i in range(2):
        c.append(i, x[1].transpose(1, 2), x[2], torch.tensor([2], device="cuda"))
    _teacher(qr, kr, v, c.layer(0), None), _teacher(qr, kr, v, c.layer(1), None)
    assert c.lens.tolist() == [2, 2, 5]


def test_room_for_all_sequences_reserved_at_once():
    """Served side by side: the room of a step is reserved for all, some sequences by teacher, another directly, in either order."""
    c, twin = _cache(1, 3), _cache(1, 3)
    at = torch.tensor([2], device="cuda")
    for i, t in enumerate((20, 1, 1, 2)):
        qr, kr, v = _qkv(3, t, i)
        for x in (c, twin):
            x.reserve(range(3), t)
        one = lambda x: x.append(0, kr[2:].transpose(1, 2), v[2:], at)
        if i % 2:
            one(c)
        o = _teacher(qr[:2], kr[:2], v[:2], c.layer(0), None)
        if i % 2 == 0:
            one(c)
        twin.append(0, kr.transpose(1, 2), v)
        assert _same(c, twin), i
        if i:
            assert torch.equal(o, twin.attend(0, qr[:2].transpose(1, 2))[0]), i


def test_a_refused_call_leaves_the_cache_as_it_was(monkeypatch):
    """What a call refuses it refuses before room is given out; what only a kernel's entry refuses is taken back."""
    import heimdall_b200.paged as paged
    c = _cache(2)
    layers = [c.layer(0), c.layer(1)]
    qr, kr, v = _qkv(2, 20, 0)
    for x in layers:
        _teacher(qr, kr, v, x, None)
    before = _state(c)
    qr, kr, v = _qkv(2, 3, 1)
    wide = torch.cat([qr] * 7, 1)                              # 28 query heads per KV head
    for kind, a in ((NotImplementedError, (qr, kr.clone().requires_grad_(), v)), (NotImplementedError, (qr.clone().requires_grad_(), kr, v)),
                    (NotImplementedError, (wide, kr, v)), (ValueError, (qr, kr[:, :1], v[:, :, :1])), (ValueError, (qr, kr[:, :, :2], v)),
                    (ValueError, (qr[:, :7], kr, v)), (ValueError, (qr[..., :128], kr[..., :128], v[..., :128]))):
        for x in layers:
            with pytest.raises(kind):
                _teacher(*a, x, None)
            assert _same(before, c) and c.length(0) == 20 and x.n == 20 and c.free_pages == 60 - 4
    real = paged._lib.call

    def failing(name, *a):
        if name == "bf_paged_append":
            raise RuntimeError("append")
        return real(name, *a)
    with monkeypatch.context() as m:
        m.setattr(paged._lib, "call", failing)
        with pytest.raises(RuntimeError, match="append"):
            _teacher(qr, kr, v, layers[0], None)
    assert _same(before, c) and c.length(1) == 20 and layers[0].n == 20
    qr, kr, v = _qkv(2, 5, 2)                                  # another number of tokens than the refused call's
    for x in layers:
        _teacher(qr, kr, v, x, None)
    assert c.lens.tolist() == [25, 25] and layers[1].n == 25


def test_appends_of_nothing_leave_no_doubt():
    """A call without sequences or tokens has written nothing, before the first layer() and after it."""
    c = _cache(1)
    qr, kr, v = _qkv(2, 3, 0)
    c.reserve([0, 1], 3)
    none = lambda: (c.append(0, kr.transpose(1, 2)[:0], v[:0]), c.append(0, kr.transpose(1, 2)[:, :0], v[:, :0]))
    none()
    layer = c.layer(0)
    none()
    _teacher(qr, kr, v, layer, None)
    assert c.lens.tolist() == [3, 3] and layer.n == 3
