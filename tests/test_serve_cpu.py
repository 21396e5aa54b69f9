"""The operators of include/lg_serve.h without a GPU: exported symbols, refusals on the host, and the plain step's own invariants."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from tests.conftest import ROOT
from tests.serve_oracle import Pages, draw


def test_library_exports_every_declared_serving_symbol(lg):
    text = open(os.path.join(ROOT, "include", "lg_serve.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(lg_\w+)\s*\(", text))
    assert declared == set(lg.SERVE_SYMBOLS)
    assert all(hasattr(lg.load(), name) for name in declared)


def _desc(lg, **kw):
    """A description that passes every check on its own numbers (its addresses are no device memory)."""
    d = dict(k=4096, v=8192, page_stride=16 * 2 * 64, row_stride=2 * 64, head_stride=64, type=1, n_pages=10, page_size=16, n_kv_heads=2, head_dim=64,
             max_req=4, max_pages=5, table_stride=5, table=256, len=512, free_pages=1024, n_free=2048, status=None)
    d.update(kw)
    return lg.PagedDesc(*[d[n] for n, _ in lg.PagedDesc._fields_])


BAD = [dict(k=None), dict(v=None), dict(table=None), dict(len=None), dict(type=2), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0), dict(n_kv_heads=65536), dict(max_req=0),
       dict(max_pages=0), dict(table_stride=4), dict(head_dim=0), dict(head_dim=12), dict(head_dim=520), dict(n_pages=1 << 28, page_size=16),
       dict(max_pages=1 << 28, table_stride=1 << 28), dict(n_pages=1, max_pages=(1 << 26) + 1, table_stride=1 << 27), dict(page_stride=-8), dict(row_stride=4), dict(head_stride=65), dict(k=4104), dict(v=8194), dict(len=513)]


@pytest.mark.parametrize("bad", BAD, ids=lambda b: ",".join(b))
def test_bad_caches_are_refused(lg, bad, capfd):
    L, c = lg.load(), _desc(lg, **bad)
    assert L.lg_paged_step(C.byref(c), 1, None, 64, 0, 64, None, None, None, None) == -1
    assert L.lg_paged_append(C.byref(c), 64, 64, 1, 128, 128, 1, 64, None) == -1
    assert L.lg_paged_attn_work(C.byref(c), 1, 1, 2) == -1
    assert L.lg_paged_attn(C.byref(c), 64, 1, 128, 1, 1, 1, None, 2, 0.0, 0, 64, 128, 64, 1 << 30, None) == -1
    assert "lg_paged" in capfd.readouterr().err
    assert L.lg_paged_attn_work(None, 1, 1, 2) == -1


@pytest.mark.parametrize("pages,page,heads,dim,order", [(7, 16, 2, 64, "rows"), (5, 24, 3, 80, "heads"), (1, 1, 1, 8, "rows"), (60000, 128, 8, 128, "rows")])
def test_places_stay_in_the_cache_and_bad_pages_have_none(lg, pages, page, heads, dim, order):
    rs, hs = (heads * dim, dim) if order == "rows" else (dim, page * dim)
    c = _desc(lg, n_pages=pages, page_size=page, n_kv_heads=heads, head_dim=dim, page_stride=page * heads * dim, row_stride=rs, head_stride=hs)
    place = lambda *at: lg.load().lg_debug_paged_place(C.byref(c), *at)  # noqa: E731
    rng = np.random.default_rng(pages)
    for p, r, h in [(0, 0, 0), (pages - 1, page - 1, heads - 1)] + [tuple(rng.integers(0, (pages, page, heads))) for _ in range(200)]:
        at = place(int(p), int(r), int(h))
        assert at == int(p) * page * heads * dim + int(r) * rs + int(h) * hs and 0 <= at <= pages * page * heads * dim - dim      # past 2^31 in the last case
    for bad in ((-1, 0, 0), (pages, 0, 0), (1 << 30, 0, 0), (-(1 << 31), 0, 0), (0, -1, 0), (0, page, 0), (0, 0, heads), (0, 0, -1)):
        assert place(*bad) == -1


def test_bad_steps_are_refused(lg):
    L, c, r = lg.load(), _desc(lg), C.byref
    call = lambda desc=c, n=1, keep=None, new=64, cap=0, start=64, pos=None: L.lg_paged_step(r(desc), n, keep, new, cap, start, pos, None, None, None)  # noqa: E731
    for kw in (dict(n=0), dict(n=5), dict(new=None), dict(start=None), dict(cap=-1), dict(keep=66), dict(pos=1), dict(desc=_desc(lg, free_pages=None)),
               dict(desc=_desc(lg, n_free=None))):
        assert call(**kw) == -1, kw
    assert call(desc=_desc(lg, max_req=9000), n=8193) == -2
    assert call() == -1                                        # addresses that are no device memory


def test_bad_appends_are_refused(lg):
    L, c = lg.load(), _desc(lg)
    call = lambda k=64, v=64, type=1, ld_k=128, ld_v=128, n=1, slot=64: L.lg_paged_append(C.byref(c), k, v, type, ld_k, ld_v, n, slot, None)  # noqa: E731
    for kw in (dict(k=None), dict(v=None), dict(slot=None), dict(n=-1), dict(type=30), dict(type=7), dict(ld_k=127), dict(ld_v=0), dict(k=65), dict(type=0, v=66), dict(slot=2)):
        assert call(**kw) == -1, kw
    assert call() == -1


def test_bad_attention_calls_are_refused(lg):
    L, c = lg.load(), _desc(lg)
    nan, inf = float("nan"), float("inf")

    def call(q=64, type=1, ld_q=256, n_req=2, n_new=3, n_rows=6, start=None, heads=4, scale=0.0, window=0, out=64, ld_out=256, work=64, size=1 << 30):
        return L.lg_paged_attn(C.byref(c), q, type, ld_q, n_req, n_new, n_rows, start, heads, scale, window, out, ld_out, work, size, None)

    for kw in (dict(q=None), dict(out=None), dict(work=None), dict(type=30), dict(ld_q=255), dict(ld_out=8), dict(n_req=0), dict(n_req=5), dict(n_new=0), dict(n_new=9, n_rows=18),
               dict(n_rows=5), dict(n_rows=-1, start=64), dict(start=66), dict(heads=3), dict(heads=0), dict(scale=-1.0), dict(scale=nan), dict(scale=inf), dict(window=-1),
               dict(q=65), dict(out=63), dict(work=72)):
        assert call(**kw) == -1, kw
    assert call(size=L.lg_paged_attn_work(C.byref(c), 2, 3, 4) - 1) == -3
    assert call() == -1
    for n_req, n_new, heads in ((0, 1, 2), (5, 1, 2), (1, 0, 2), (1, 9, 2), (1, 1, 3), (1, 1, 0)):
        assert L.lg_paged_attn_work(C.byref(c), n_req, n_new, heads) == -1
    assert L.lg_paged_attn_work(C.byref(c), 1, 1, 2) > 0


def test_bad_samples_are_refused(lg):
    L = lg.load()
    call = lambda x=64, type=0, ld=100, rows=1, vocab=100, t=None, k=None, u=64, token=64, prob=None: L.lg_sample(x, type, ld, rows, vocab, t, k, None, None, u, token, prob, None)  # noqa: E731
    for kw in (dict(x=None), dict(type=8), dict(ld=99), dict(rows=-1), dict(vocab=0), dict(u=None), dict(token=None), dict(x=66), dict(type=1, x=65), dict(t=2), dict(k=3), dict(prob=5)):
        assert call(**kw) == -1, kw
    assert call(vocab=(1 << 20) + 1, ld=1 << 21) == -2
    assert call() == -1


class _Tensor:
    """What the binding asks of a tensor, without one."""

    def __init__(self, shape, dtype, stride=None):
        self.shape, self.dtype = tuple(shape), f"torch.{dtype}"
        step, self._stride = 1, []
        for n in reversed(self.shape):
            self._stride.insert(0, step)
            step *= n
        self._dense = stride is None
        self._stride = tuple(stride or self._stride)

    def dim(self): return len(self.shape)
    def stride(self, i=None): return self._stride if i is None else self._stride[i]
    def numel(self): return int(np.prod(self.shape))
    def is_contiguous(self): return self._dense
    def element_size(self): return 4
    def data_ptr(self): return 4096


def test_binding_checks_types_shapes_and_strides(lg):
    T = _Tensor
    kv, table, length = T((9, 16, 2, 64), "float16"), T((4, 5), "int32"), T((4,), "int32")
    for k, v in ((kv, T((9, 16, 2, 64), "bfloat16")), (T((9, 16, 2, 64), "int8"),) * 2, (kv, T((9, 16, 1, 64), "float16")), (kv, T((9, 16, 2, 64), "float16", (1, 9, 8, 2))),
                 (T((9, 16, 128), "float16"),) * 2):
        with pytest.raises(ValueError):
            lg.PagedCache(k, v, table, length)
    for bad in (dict(table=T((4, 5), "int64")), dict(table=T((5,), "int32")), dict(length=T((3,), "int32")), dict(length=T((4,), "float32")), dict(free=T((9,), "int32")),
                dict(free=T((8,), "int32"), n_free=T((1,), "int32"))):
        with pytest.raises(ValueError):
            lg.PagedCache(kv, kv, **{**dict(table=table, length=length), **bad})
    c = lg.PagedCache(kv, kv, table, length, T((9,), "int32"), T((1,), "int32"))
    i = lambda n, t="int32": T((n,), t)  # noqa: E731
    for args in ((i(4), i(4)), (i(4, "int64"), i(5)), (i(4), i(5), i(7, "float32")), (i(4), i(5), i(7), i(7), i(7), i(3))):
        with pytest.raises(ValueError):
            c.step(*args)
    for args in ((T((3, 2, 32), "float16"), T((3, 2, 64), "float16"), i(3)), (T((3, 128), "float16"), T((3, 128), "float32"), i(3)), (T((3, 128), "float16"), T((3, 128), "float16"), i(2)),
                 (T((3, 128), "float16"), T((2, 128), "float16"), i(3))):
        with pytest.raises(ValueError):
            c.append(*args)
    q = T((4, 4, 64), "float32")
    for q_, out in ((q, T((4, 4, 64), "float16")), (T((4, 256), "float32"),) * 2, (T((4, 4, 32), "float32"),) * 2, (q, T((4, 4, 64), "float32", (256, 1, 4)))):
        with pytest.raises(ValueError):
            c.attn(q_, out, T((1 << 20,), "uint8"))
    for args, kw in (((T((4, 100), "int32"), i(4, "float32"), i(4)), {}), ((T((4, 100), "float32"), i(3, "float32"), i(4)), {}), ((T((4, 100), "float32", (1, 4)), i(4, "float32"), i(4)), {}),
                     ((T((4, 100), "float32"), i(4, "float32"), i(4)), dict(top_k=i(4, "float32")))):
        with pytest.raises(ValueError):
            lg.sample(*args, **kw)


def test_plain_step_keeps_every_page_once():
    """The oracle itself: whatever happens, the pages of tables and stack are all pages, each once."""
    rng = np.random.default_rng(1)
    p = Pages(np.full((20, 9), -1), np.zeros(20, int), rng.permutation(70), 70, 4)
    for _ in range(60):
        keep = np.maximum(0, p.len - rng.integers(0, 6, 20)) * (rng.random(20) < 0.9)
        start, pos, slot, req, _ = p.step(rng.integers(0, 7, 20), 200, keep.astype(int))
        held = [int(x) for r in range(20) for x in p.table[r, : -(-int(p.len[r]) // 4)]]
        assert sorted(held + [int(x) for x in p.free[:p.n_free]]) == list(range(70))
        live = [s for s in slot if s >= 0]
        assert len(set(live)) == len(live) == start[-1]


def test_plain_draw_on_hand_made_rows():
    x = [0.0, 1.0, -np.inf, 1.0, np.nan, -1.0]                 # order 1, 3, 0, 5
    e = np.exp(-1.0)
    assert draw(x, 0.0) == (0, pytest.approx(e / (2 + e + e * e)))
    assert draw(x, 0.9999)[0] == 5 and draw(x, 0.5, top_k=1) == (1, 1.0) and draw(x, 0.5, top_k=2) == (3, 0.5)
    # 1 / (2 + e + e^2) = 0.3995 < 0.4: the first of the order is not enough
    assert draw(x, 0.0, min_p=0.5) == (1, 0.5) and draw(x, 0.99, top_p=0.4)[0] == 3 and draw(x, 0.3, temperature=0.0) == (1, 1.0)
    assert draw([np.nan, -np.inf], 0.5) == (-1, 0.0) and draw([np.inf, 0.0, np.inf], 0.6) == (2, 0.5)


def test_room_of_a_step(lg):
    """cap: the smallest output's size, 0 without outputs, or what the caller says -- which the outputs have to hold."""
    i = lambda n: _Tensor((n,), "int32")  # noqa: E731
    kv = _Tensor((9, 16, 2, 64), "float16")
    c = lg.PagedCache(kv, kv, _Tensor((4, 5), "int32"), i(4), i(9), i(1))
    caps = []

    class Lib:
        @staticmethod
        def lg_paged_step(ref, n, keep, new, cap, *rest):
            caps.append(cap)
            return 0

    c.L = Lib
    c.step(i(4), i(5))
    c.step(i(4), i(5), i(7), i(6))
    c.step(i(4), i(5), cap=100)
    c.step(i(4), i(5), i(7), i(6), cap=5)
    assert caps == [0, 6, 100, 5]
    for args, cap in (((i(7), i(6)), 7), ((), -1), ((), 1 << 32)):
        with pytest.raises(ValueError):
            c.step(i(4), i(5), *args, cap=cap)


# (lengths, new tokens, free pages, cap): who is served, and the status -- pages of 16 rows, 4 columns, by the rules of include/lg_serve.h
SERVED = [
    (([16, 16], [17, 1], 2, 1), ([0, 0], Pages.NO_ROWS | Pages.NO_PAGES)),       # pages first: both are request 0's, which then has no rows; they are not offered again
    (([16, 16, 16, 3], [17, 33, 1, 2], 3, 100), ([1, 0, 0, 1], Pages.NO_PAGES)),  # one page would do for request 2, behind one that had too few
    (([1, 1, 1, 16], [5, 6, 2, 0], 0, 9), ([1, 0, 0, 1], Pages.NO_ROWS)),         # two rows would do for request 2, behind one that had too few
    (([60, 16, 0], [5, 1, 0], 1, 9), ([0, 1, 1], Pages.TOO_LONG)),
]


@pytest.mark.parametrize("case,want", SERVED)
def test_who_is_served(case, want):
    lens, new, free, cap = case
    table = np.full((len(lens), 4), -1)
    at = free
    for r, n in enumerate(lens):
        k = -(-n // 16)
        table[r, :k] = range(at, at + k)
        at += k
    p = Pages(table, lens, list(range(at)), free, 16)
    *_, status = p.step(new, cap)
    assert p.len.tolist() == [n + m * s for n, m, s in zip(lens, new, want[0])] and status == want[1]


def test_a_workspace_in_pieces_is_refused(lg):
    """One element expanded to the size that is asked for is not that many bytes."""
    kv, q = _Tensor((9, 16, 2, 64), "float16"), _Tensor((4, 4, 64), "float16")
    c = lg.PagedCache(kv, kv, _Tensor((4, 5), "int32"), _Tensor((4,), "int32"))

    class Lib:
        @staticmethod
        def lg_paged_attn(*args):
            raise AssertionError("called")

    c.L = Lib
    for stride in ((0,), (2,)):
        with pytest.raises(ValueError, match="work"):
            c.attn(q, q, _Tensor((1 << 24,), "uint8", stride))
