"""The page allocator of the 8-bit cache against a plain model, the oracle's own properties, and what is refused (CPU)."""
import ctypes
import random

import numpy as np
import pytest
import torch

from heimdall_b200 import PagedKV, _lib, prompt_attention
from heimdall_b200.paged import PageTable
from heimdall_b200.structs import BfPagePool
from oracle import paged_kv as opk


class Model:
    """Sequences as lists of page numbers; a page's holders are counted by looking."""

    def __init__(self, pages, slots, L):
        self.pages, self.L = pages, L
        self.rows, self.lens = [[] for _ in range(slots)], [0] * slots

    def take(self):
        used = {p for r in self.rows for p in r}
        return next(p for p in range(self.pages) if p not in used)

    def reserve(self, slots, n):
        for s, x in zip(slots, n):
            self.lens[s] += x
            while len(self.rows[s]) * self.L < self.lens[s]:
                self.rows[s].append(self.take())

    def free(self, slots):
        for s in slots:
            self.rows[s], self.lens[s] = [], 0

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            row = list(self.rows[a])
            if self.lens[a] % self.L:
                row[-1] = self.take()
            self.rows[b], self.lens[b] = row, self.lens[a]

    def compact(self):
        live = sorted({p for r in self.rows for p in r})
        holes = [p for p in range(len(live)) if p not in set(live)]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]


def check(t, m):
    for s, row in enumerate(m.rows):
        assert t.table[s].tolist() == row + [-1] * (t.width - len(row))
        assert t.lens[s] == m.lens[s]
    count = np.bincount([p for r in m.rows for p in r], minlength=t.pages)
    assert (t.refs == count).all() and t.n_free == int((count == 0).sum())


def play(table, lens, t, todo):
    """The device's part, on host arrays."""
    for s in todo.get("release", []):
        table[s] = -1
        lens[s] = 0
    for a, b, n, old, new in todo.get("fork", []):
        row = table[a].copy()
        if new >= 0:
            assert row[n // t.page] == old
            row[n // t.page] = new
        table[b], lens[b] = row, n
    moves = dict(todo.get("move", np.zeros((0, 2), int)).tolist())
    for i, p in np.ndenumerate(table):
        table[i] = moves.get(int(p), p)
    for at, value in todo.get("set", []):
        if at < table.size:
            table.reshape(-1)[at] = value
        else:
            lens[at - table.size] = value


@pytest.mark.parametrize("seed", range(6))
def test_page_table_follows_a_plain_model(seed):
    rng = random.Random(seed)
    L, slots, width, pages = rng.choice([16, 64]), 7, 5, 24
    t, m = PageTable(pages, slots, L, width), Model(pages, slots, L)
    table, lens = np.full((slots, width), -1), np.zeros(slots, int)
    for _ in range(120):
        op = rng.choice(["reserve", "reserve", "fork", "free", "compact", "truncate"])
        some = rng.sample(range(slots), rng.randint(1, 3))
        try:
            if op == "reserve":
                n = [rng.choice([0, 1, L - 1, L, 2 * L + 1]) for _ in some]
                todo = t.reserve(some, n)
                m.reserve(some, n)
            elif op == "free":
                todo = t.free(some)
                m.free(some)
            elif op == "compact":
                todo = t.compact()
                m.compact()
                assert np.flatnonzero(t.refs).tolist() == list(range(pages - t.n_free))
            elif op == "fork":
                empty = [s for s in range(slots) if t.lens[s] == 0][:2]
                src = [rng.choice([s for s in range(slots) if s not in empty]) for _ in empty] if len(empty) < slots else []
                todo = t.fork(src, empty[:len(src)])
                m.fork(src, empty)
            else:
                before = (t.refs.copy(), t.table.copy())
                new = [rng.randint(0, int(t.lens[s])) for s in some]
                todo = t.truncate(some, new)
                for s, n in zip(some, new):        # a partly filled page belongs to one sequence, the rest stays shared
                    row = t.table[s][t.table[s] >= 0]
                    assert len(row) == -(-n // L) and t.lens[s] == n
                    assert (row[:n // L] == before[1][s][:n // L]).all()
                    if n % L:
                        assert t.refs[row[-1]] == 1
                m.rows = [r[r >= 0].tolist() for r in t.table]
                m.lens = t.lens.tolist()
        except (RuntimeError, ValueError):
            todo = {}
        check(t, m)
        play(table, lens, t, todo)
        assert (table == t.table).all() and (lens == t.lens).all()


def test_refused_page_calls_change_nothing():
    t = PageTable(4, 3, 16, 3)
    t.reserve([0, 1], [20, 16])
    before = (t.refs.copy(), t.table.copy(), t.lens.copy(), t.n_free)
    bad = [(RuntimeError, lambda: t.reserve([1, 2], 16)), (ValueError, lambda: t.reserve([0], 29)), (ValueError, lambda: t.reserve([0, 0], 1)),
           (ValueError, lambda: t.reserve([3], 1)), (ValueError, lambda: t.reserve([-1], 1)), (ValueError, lambda: t.reserve([0], -1)),
           (ValueError, lambda: t.reserve([0, 1], [1, 2, 3])), (ValueError, lambda: t.reserve([0.5], 1)), (ValueError, lambda: t.reserve([0], 0.5)),
           (ValueError, lambda: t.fork([0], [1])), (ValueError, lambda: t.fork([0], [0])), (ValueError, lambda: t.fork([0, 1], [2])),
           (ValueError, lambda: t.fork([0, 1], [2, 2])), (ValueError, lambda: t.truncate([0], [21])), (ValueError, lambda: t.free([0, 0]))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
        assert (t.refs == before[0]).all() and (t.table == before[1]).all() and (t.lens == before[2]).all() and t.n_free == before[3]
    t.fork([0], [2])
    with pytest.raises(RuntimeError):
        t.reserve([2], 20)
    t.truncate([2], 18)
    assert t.n_free == 0 and t.refs.tolist() == [2, 1, 1, 1]


def test_truncate_copies_a_shared_page_once_per_holder_but_the_last():
    t = PageTable(8, 3, 16, 4)
    t.reserve([0], 32)
    t.fork([0, 0], [1, 2])
    todo = t.truncate([0, 1, 2], [20, 21, 22])
    assert todo["fork"].tolist() == [[0, 0, 20, 1, 2], [1, 1, 21, 1, 3]]
    assert t.table[:, 1].tolist() == [2, 3, 1] and t.refs.tolist() == [3, 1, 1, 1, 0, 0, 0, 0]


def test_oracle_codes_and_scales():
    x = torch.tensor([0.0, 448.0, 447.0, -460.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 17.0, 19.0, 1.0625], dtype=torch.float64)
    assert torch.equal(opk.e4m3(x), x.clamp(-448, 448).float().to(torch.float8_e4m3fn).double())
    r = torch.linspace(-448, 448, 100001).double()       # of 32 bits, so that the way through float() rounds once
    assert torch.equal(opk.e4m3(r), r.float().to(torch.float8_e4m3fn).double())
    assert opk.page_scale(torch.tensor([448.0])) == 1.0 and opk.page_scale(torch.tensor([449.0])) == 2.0
    assert opk.page_scale(torch.tensor([7.0, float("inf"), float("nan")])) == 2.0 ** -6
    assert opk.page_scale(torch.zeros(3)) == 2.0 ** -64


def test_entry_points_refuse_on_the_host():
    q, k = torch.zeros(3, 4, 256, dtype=torch.bfloat16), torch.zeros(3, 2, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(q, k, k, torch.tensor([0, 3]))
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKV(1, 4, 2, 1, device="cpu")
    for kw, kind in ((dict(page=48), NotImplementedError), (dict(dim=128), NotImplementedError), (dict(max_len=0), ValueError)):
        with pytest.raises(kind):
            PagedKV(1, 4, 2, 1, **kw)
    with pytest.raises(ValueError):
        PagedKV(0, 4, 2, 1)
    with pytest.raises(ValueError):
        PagedKV(1, 2 ** 24, 8, 1)


def _pool(**kw):
    at = dict(k_pages=256, v_pages=256, k_scale=256, v_scale=256, table=256, lens=256, layers=2, pages=8, heads=4, page=64, dim=256,
              slots=3, width=4)
    at.update(kw)
    p = BfPagePool(*(at[f] for f, _ in BfPagePool._fields_))
    return p, ctypes.addressof(p)


def _code(name, *args):
    with pytest.raises(_lib.BifrostError) as e:
        _lib.call(name, *args)
    return e.value.code


def test_c_entries_check_their_arguments_before_a_launch():
    P = 256            # an aligned address that nothing reads: every call below is refused
    prompt = lambda q=P, st=6144, cu=P, n=1, T=8, Tk=8, H=24, G=4, D=256, dt=1, scale=0.1, o=P: _code(
        "bf_prompt_attn_fwd", q, st, 256, P, 1024, 256, P, 1024, 256, cu, 0, n, T, Tk, H, G, D, dt, scale, o, 0, 0)
    assert prompt(q=0) == 1 and prompt(o=0) == 1 and prompt(cu=0) == 1 and prompt(T=-1) == 1 and prompt(H=23) == 1
    assert prompt(scale=0.0) == 1 and prompt(scale=float("nan")) == 1 and prompt(scale=float("inf")) == 1
    assert prompt(Tk=2 ** 25 + 1) == 2 and prompt(n=2 ** 20 + 1) == 2
    assert prompt(D=128) == 2 and prompt(dt=0) == 2 and prompt(q=P + 8) == 3 and prompt(st=6140) == 3
    keep = []

    def pool(**kw):
        p, at = _pool(**kw)
        keep.append(p)
        return at
    app = lambda pool_, layer=0, k=P, sb=1024, B=2, t=1, dt=1: _code("bf_paged_append", pool_, layer, k, sb, 1024, 256, P, 1024, 1024, 256, 0,
                                                                  0, B, t, dt, 0)
    assert app(0) == 1 and app(pool(lens=0)) == 1 and app(pool(), layer=2) == 1 and app(pool(), layer=-1) == 1
    assert app(pool(page=48)) == 2 and app(pool(dim=128)) == 2 and app(pool(pages=2 ** 24, heads=8)) == 2 and app(pool(k_pages=264)) == 3
    assert app(pool(), B=4) == 1 and app(pool(), k=0) == 1 and app(pool(), k=P + 2) == 3 and app(pool(), sb=1020) == 3 and app(pool(), dt=0) == 2
    att = lambda pool_, q=P, B=2, t=1, H=24, scale=0.1, ws=P, nws=1 << 40, dt=1: _code(
        "bf_paged_attend", pool_, 0, q, 6144, 6144, 256, 0, B, t, H, dt, scale, P, 0, ws, nws, 0)
    assert att(pool(), q=0) == 1 and att(pool(), H=23) == 1 and att(pool(), B=4) == 1 and att(pool(), scale=-1.0) == 1
    assert att(pool(), H=100) == 2 and att(pool(), dt=0) == 2 and att(pool(), q=P + 8) == 3 and att(pool(), nws=0) == 4 and att(pool(), ws=0) == 4

    def pages(release=(), fork=(), move=(), set_=()):
        flat = []
        for x, w in ((release, 1), (fork, 5), (move, 2), (set_, 2)):
            a = np.array(x, np.int32).reshape(-1, w)
            keep.append(a)
            flat += [a.ctypes.data, a.shape[0]]
        return _code("bf_paged_pages", pool(), *flat, 0)
    assert pages(release=[3]) == 1 and pages(release=[-1]) == 1 and pages(fork=[0, 3, 1, 0, 1]) == 1 and pages(fork=[0, 1, 300, 0, 1]) == 1
    assert pages(fork=[0, 1, 5, 8, 1]) == 1 and pages(fork=[0, 1, 5, 1, 1]) == 1 and pages(move=[8, 1]) == 1 and pages(move=[5, 1, 4, 0]) == 1
    assert pages(set_=[15, 0]) == 1 and pages(set_=[-1, 0]) == 1


def test_a_layers_progress_follows_the_page_table():
    """What teacher has written of each slot, as the sequences are forked, cut and ended, and where the host cannot tell."""
    from heimdall_b200.paged import _Progress

    class Cache:
        layers, host, _appended = 3, PageTable(40, 4, 16, 6), {1}
    host, no = Cache.host, _Progress.UNKNOWN
    host.reserve([3], 5)                                    # written directly in layer 1 before the first layer()
    p = _Progress(Cache)
    assert p.n.tolist() == [[0] * 4, [0, 0, 0, no], [0] * 4]

    def teacher(layer, B, t):
        if (host.lens[:B] == p.n[layer, :B]).all():
            host.reserve(range(B), t)
            p.room[:B] = host.lens[:B]
        assert (host.lens[:B] == p.n[layer, :B] + t).all()
        p.n[layer, :B] = host.lens[:B]
    for layer in (0, 1, 2):
        teacher(layer, 2, 20)
    host.truncate([0, 1], [18, 0])
    p.truncate([0, 1], [18, 0])
    assert p.n[:, :2].tolist() == [[18, 0]] * 3
    host.fork([0, 3], [1, 2])
    p.fork([0, 3], [1, 2])
    assert p.n.tolist() == [[18, 18, 0, 0], [18, 18, no, no], [18, 18, 0, 0]]
    teacher(0, 2, 1)
    p.appended(1, torch.tensor([2, 3]), 2)                  # teacher's own room is not in doubt
    p.appended(1, None, 4)
    assert p.n[1].tolist() == [18, 18, no, no]
    teacher(1, 2, 1), teacher(2, 2, 1)
    host.reserve([0, 1], 2)                                 # the caller's is
    p.appended(0, torch.tensor([1, 9, -1]), 3)
    assert p.n[0].tolist() == [19, no, 0, 0]
    p.appended(2, None, 1)
    assert p.n[2].tolist() == [no, 19, 0, 0]
    host.truncate([1], 0)
    p.truncate([1], 0)
    host.free([0, 3])
    p.free([0, 3])
    assert p.n[:, [0, 1, 3]].tolist() == [[0] * 3] * 3
