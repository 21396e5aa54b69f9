"""Paged cache on the GPU -- step, append, attention -- against plain 64-bit forms and the contiguous-cache attention."""
import numpy as np
import pytest

from tests.serve_oracle import Pages, attention

pytestmark = pytest.mark.gpu

F32, F16, BF16 = "float32", "float16", "bfloat16"


def _i32(a):
    import torch
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _pool(rng, lens, page, columns, spare, extra_pages=0):
    """(table, free, n_free, pages): requests of these lengths on pages in random order, `spare` free ones behind them."""
    held = [-(-n // page) for n in lens]
    order = rng.permutation(sum(held) + spare + extra_pages)
    table, at = np.full((len(lens), columns), -1), 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    free = np.zeros(len(order), dtype=np.int64)
    free[:spare] = order[at:at + spare]
    return table, free, spare, len(order)


class _Cache:
    """A PagedCache on fresh tensors with the oracle's state beside it."""

    def __init__(self, lg, rng, lens, page, columns, spare, kv_heads=1, dim=8, dtype=F16, layout="rows"):
        import torch
        table, free, n_free, pages = _pool(rng, lens, page, columns, spare)
        self.oracle = Pages(table, lens, free, n_free, page)
        self.table, self.len, self.free, self.n_free, self.status = _i32(table), _i32(lens), _i32(free), _i32([n_free]), _i32([0])
        dt = getattr(torch, dtype)
        if layout == "rows":                                   # [pages][rows][heads][dim]
            self.k, self.v = (torch.full((pages, page, kv_heads, dim), float("nan"), dtype=dt, device="cuda") for _ in range(2))
        elif layout == "heads":                                # [pages][heads][rows][dim]
            self.k, self.v = (torch.full((pages, kv_heads, page, dim), float("nan"), dtype=dt, device="cuda").transpose(1, 2) for _ in range(2))
        else:                                                  # K and V of a page side by side, rows wider than the heads
            both = torch.full((pages, 2, page, kv_heads + 1, dim), float("nan"), dtype=dt, device="cuda")
            self.k, self.v = both[:, 0, :, :kv_heads], both[:, 1, :, :kv_heads]
        self.c = lg.PagedCache(self.k, self.v, self.table, self.len, self.free, self.n_free, self.status)

    def step(self, new, cap, keep=None, stream=0):
        import torch
        n = len(new)
        start = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
        pos, slot, req = (torch.full((cap,), -7, dtype=torch.int32, device="cuda") for _ in range(3))
        self.c.step(_i32(new), start, pos if cap else None, slot if cap else None, req if cap else None, None if keep is None else _i32(keep), stream=stream)
        return start, pos, slot, req

    def check(self, got, want):
        for name, g, w in zip(("start", "pos", "slot", "req"), got, want):
            assert np.array_equal(g.cpu().numpy(), w), name
        assert self.status.item() == want[4]
        assert np.array_equal(self.len.cpu().numpy(), self.oracle.len)
        assert self.n_free.item() == self.oracle.n_free
        assert np.array_equal(self.free.cpu().numpy()[: self.oracle.n_free], self.oracle.free[: self.oracle.n_free])
        assert np.array_equal(self.table.cpu().numpy(), self.oracle.table)


# ------------------------------------------------------------------------------------------------------------------------
# step
# ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,page,top,spare", [(1, 1, 5, 9), (3, 16, 40, 6), (48, 16, 300, 60), (1025, 7, 60, 1500), (8192, 4, 9, 20000)])
def test_step_follows_the_plain_form_over_many_steps(lg, n, page, top, spare):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, top + 1, n)
    lens[0] = 0
    c = _Cache(lg, rng, lens, page, -(-top // page) + 3, spare)
    for kind in ("grow", "verify", "roll back", "chunk", "release", "grow", "nothing"):
        new, keep = rng.integers(0, 3, n), None
        if kind == "verify":
            new = np.full(n, 4)
        if kind == "roll back":
            keep, new = np.maximum(c.oracle.len - rng.integers(0, 5, n), -1), np.zeros(n, dtype=int)
        if kind == "chunk":
            new[::5] = page * 2 + 1
        if kind == "release":
            keep, new = np.where(rng.random(n) < 0.5, 0, 1 << 30), rng.integers(0, 2, n)
        if kind == "nothing":
            new[:] = 0
        cap = int(new.sum()) + 3
        got = c.step(new, cap, keep)
        c.check(got, c.oracle.step(new, cap, keep))
        c.status.zero_()


@pytest.mark.parametrize("spare,cap,columns", [(2, 100, 8), (100, 11, 8), (100, 100, 3), (0, 0, 4), (3, 9, 3)])
def test_step_serves_in_order_while_pages_rows_and_columns_last(lg, spare, cap, columns):
    rng = np.random.default_rng(5)
    lens = [7, 8, 0, 3, 16, 9, 0, 12]
    c = _Cache(lg, rng, lens, 8, max(columns, 2), spare)
    for new in ([1, 1, 9, 0, 4, 2, 30, 3], [2, 2, 2, 2, 2, 2, 2, 2], [0, 0, 1, 0, 0, 0, 0, 1]):
        c.check(c.step(new, cap), c.oracle.step(new, cap))
        c.status.zero_()


def test_roll_back_leaves_tables_and_stack_as_they_were(lg):
    rng = np.random.default_rng(9)
    c = _Cache(lg, rng, rng.integers(1, 90, 300), 8, 16, 900)
    before = [t.clone() for t in (c.table, c.len, c.free, c.n_free)]
    keep = c.len.cpu().numpy()
    c.step(np.full(300, 8), 2400)
    assert c.n_free.item() < 900
    c.step(np.zeros(300, dtype=int), 0, keep)
    assert all(bool((a == b).all()) for a, b in zip(before, (c.table, c.len, c.free, c.n_free)))
    assert c.status.item() == 0


def test_step_marks_bad_pages_of_the_stack_and_of_the_table(lg):
    rng = np.random.default_rng(3)
    c = _Cache(lg, rng, [4, 3], 4, 3, 2)
    c.free[1] = 1 << 20                                        # the top of the stack: the first page to be taken
    c.table[1, 0] = -5
    _, pos, slot, req = c.step([1, 1], 2)
    assert slot.tolist() == [-1, -1] and pos.tolist() == [4, 3] and req.tolist() == [0, 1]
    assert c.status.item() == Pages.BAD_PAGE
    c.status.zero_()
    c.step([0, 0], 0, [0, 0])                                  # what is no page does not come back as one
    assert c.status.item() == Pages.BAD_PAGE and c.len.tolist() == [0, 0] and (c.table.cpu().numpy() == -1)[0, :2].all()


# ------------------------------------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,cache", [(F32, F16), (F32, BF16), (F32, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("n,kv_heads,dim,page,layout", [(1, 1, 8, 1, "rows"), (37, 3, 80, 24, "heads"), (513, 2, 256, 16, "pairs")])
def test_append_rounds_rows_into_their_slots_and_nothing_else(lg, dtype, cache, n, kv_heads, dim, page, layout):
    import torch
    rng = np.random.default_rng(n)
    pages = -(-n // page) + 2
    c = _Cache(lg, rng, [1], page, pages, pages - 1, kv_heads, dim, cache, layout)
    slot = rng.permutation(pages * page)[:n]
    slot[::7] = -1
    wide = torch.randn(n, 2 * kv_heads * dim + 3, device="cuda").to(getattr(torch, dtype))      # rows at odd addresses
    k, v = wide[:, 1:1 + kv_heads * dim], wide[:, 2 + kv_heads * dim:2 + 2 * kv_heads * dim]
    want_k, want_v = c.k.clone(), c.v.clone()
    for i, s in enumerate(slot):
        if s >= 0:
            want_k[s // page, s % page] = k[i].view(kv_heads, dim).to(want_k.dtype)
            want_v[s // page, s % page] = v[i].view(kv_heads, dim).to(want_v.dtype)
    c.c.append(k, v, _i32(slot))
    assert torch.equal(c.k.nan_to_num(77.0), want_k.nan_to_num(77.0)) and torch.equal(c.v.nan_to_num(77.0), want_v.nan_to_num(77.0))
    assert c.status.item() == 0
    c.c.append(k.contiguous(), v.contiguous(), _i32(np.where(slot < 0, pages * page, -2)))       # outside the cache: left out
    assert torch.equal(c.k.nan_to_num(77.0), want_k.nan_to_num(77.0)) and c.status.item() == 16


def test_append_of_no_rows(lg):
    import torch
    c = _Cache(lg, np.random.default_rng(0), [1], 4, 1, 0)
    c.c.append(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 8, device="cuda"), _i32([0]))
    assert bool(c.k.isnan().all())


# ------------------------------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------------------------------

HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _tolerance(want, q, k, v, scale, dtype, cache):
    """Bound on |got - want|: f32 sums of dim / 16 tensor-core steps and the splits of q put an error of at most e on a score, which scales
    its weight by e either way, the numerator's and the denominator's; weights are kept to 2^-16 (two bf16 halves of a
    bf16 answer) or 2^-20; then half a step of the output's type."""
    bound = scale * np.linalg.norm(q, axis=-1).max() * np.linalg.norm(k, axis=-1).max()
    e = (q.shape[-1] / 16 + 8) * 2.0 ** -23 * bound
    weights = 2.0 ** -16 if dtype == BF16 else 2.0 ** -20
    return np.abs(v).max() * (2 * e + weights + 16 * 2.0 ** -23) + HALF_STEP[dtype] * np.abs(want)


def _fill(c, rng, lens, q, m, page, kv_heads, dim, window):
    """K and V of the rows that some query sees; what none sees stays NaN.  The outermost visible rows lean towards a query, so that leaving one
    out shows.  Returns the cache's values, one array per request."""
    import torch
    heads, out = q.shape[1], []
    table = c.oracle.table
    for r, n in enumerate(lens):
        k, v = (torch.randn((n, kv_heads, dim), device="cuda") for _ in range(2))
        group = heads // kv_heads
        for t in range(m[r]):
            at = n - m[r] + t
            first = max(0, at - window + 1) if window else 0
            row = sum(m[:r]) + t
            if at >= 0:
                k[at] += 0.4 * q[row].float().view(kv_heads, group, dim)[:, 0]
                k[first] += 0.4 * q[row].float().view(kv_heads, group, dim)[:, -1]
        k, v = k.to(c.k.dtype), v.to(c.v.dtype)
        lowest = max(0, n - m[r] - window + 1) if window else 0
        for i in range(lowest, n):
            c.k[table[r, i // page], i % page] = k[i]
            c.v[table[r, i // page], i % page] = v[i]
        out.append((k.double().cpu().numpy(), v.double().cpu().numpy()))
    return out


def _attn_case(lg, seed, lens, m, heads, kv_heads, dim, page, dtype, cache, window=0, layout="rows", ragged=False, scale=0.0, q_gain=1.0):
    import torch
    rng = np.random.default_rng(seed)
    torch.manual_seed(seed)
    columns = max(1, max(-(-n // page) for n in lens))
    c = _Cache(lg, rng, lens, page, columns, 3, kv_heads, dim, cache, layout)
    rows, behind = sum(m), 3 if ragged else 0
    q = (q_gain * torch.randn((rows + behind, heads, dim), device="cuda")).to(getattr(torch, dtype))
    data = _fill(c, rng, lens, q, m, page, kv_heads, dim, window)
    out = torch.full_like(q, 99.0)
    n_new = max(1, max(m))
    start = _i32(np.concatenate([[0], np.cumsum(m)])) if ragged else None
    work = torch.full((c.c.attn_work(len(lens), n_new, heads),), 255, dtype=torch.uint8, device="cuda")   # NaN in what is read before it is written
    c.c.attn(q, out, work, n_new=n_new, start=start, window=window, scale=scale)
    got = out.double().cpu().numpy()
    qd, at, s = q.double().cpu().numpy(), 0, scale or dim ** -0.5
    for r, n in enumerate(lens):
        k, v = data[r]
        want = attention(qd[at:at + m[r]], k, v, s, [n - m[r] + t for t in range(m[r])], window)
        if m[r]:
            tol = _tolerance(want, qd[at:at + m[r]], k, v, s, dtype, cache) if n else 0.0
            err = np.abs(got[at:at + m[r]] - want)
            assert np.isfinite(got[at:at + m[r]]).all(), r
            assert (err <= tol).all(), (r, n, float(err.max()), float(np.max(err - tol)))
        at += m[r]
    assert (got[rows:] == 99.0).all()                          # rows behind the last request
    assert c.status.item() == 0
    return c, q, out, work


TYPES = [(F32, F16), (F16, F16), (BF16, BF16), (F32, BF16), (F32, F32)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page,layout", [(4, 4, 64, 16, "rows"), (8, 2, 256, 16, "heads"), (7, 1, 80, 24, "pairs"), (16, 2, 128, 1, "rows"),
                                                             (2, 1, 512, 64, "rows"), (24, 2, 8, 128, "heads")])
def test_attention_of_single_tokens(lg, dtype, cache, heads, kv_heads, dim, page, layout):
    lens = [1, 0, 15, 16, 17, 129, 700, 64, 2]
    _attn_case(lg, dim, lens, [1] * len(lens), heads, kv_heads, dim, page, dtype, cache, layout=layout)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("new,heads,kv_heads,dim", [(2, 4, 2, 64), (4, 16, 8, 256), (8, 8, 1, 128), (5, 7, 1, 96), (3, 2, 2, 512), (8, 12, 1, 512), (8, 16, 1, 256)])
def test_attention_of_verify_blocks(lg, dtype, cache, new, heads, kv_heads, dim):
    lens = [new, new - 1, 1, 0, 33, 500, 128 + new]            # shorter than the block: its first rows see nothing
    _attn_case(lg, new, lens, [new] * len(lens), heads, kv_heads, dim, 16, dtype, cache)


@pytest.mark.parametrize("dtype,cache", [(F32, F16), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("window,new", [(1, 1), (16, 1), (100, 4), (257, 8), (5000, 2)])
def test_attention_of_sliding_windows(lg, dtype, cache, window, new):
    lens = [3 + new, 16, 100, 257, 1000, 1]
    _attn_case(lg, window, lens, [new] * len(lens), 8, 2, 128, 16, dtype, cache, window=window)


@pytest.mark.parametrize("dtype,cache", [(F32, F16), (BF16, BF16), (F32, F32)])
def test_attention_of_ragged_blocks(lg, dtype, cache):
    m = [1, 0, 4, 2, 8, 0, 1, 3]
    lens = [5, 40, 4, 300, 8, 0, 2000, 129]
    _attn_case(lg, 1, lens, m, 8, 2, 128, 16, dtype, cache, ragged=True)


@pytest.mark.parametrize("dtype,cache", [(F32, F16), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("kv_heads,length", [(1, 20011), (8, 9000)])
def test_attention_split_over_long_caches(lg, dtype, cache, kv_heads, length):
    _attn_case(lg, length, [length, 100], [1, 1], 4 * kv_heads, kv_heads, 128, 64, dtype, cache)


@pytest.mark.parametrize("dtype,cache,gain", [(F32, F16, 300.0), (F32, F16, 1e-4), (F32, BF16, 1e5), (F32, F32, 1e5)])
def test_attention_of_queries_far_from_one(lg, dtype, cache, gain):
    """Queries outside of what 16 bits hold well, with a scale that brings the scores back."""
    _attn_case(lg, 4, [300, 20], [1, 1], 4, 2, 128, 16, dtype, cache, scale=128 ** -0.5 / gain, q_gain=gain)


@pytest.mark.parametrize("dtype,cache", [(F32, F16), (BF16, BF16), (F32, F32)])
def test_the_same_call_gives_the_same_bits(lg, dtype, cache):
    """Whatever the workspace holds; a request alone agrees with itself in the batch to the tolerance of both (_attn_case)."""
    import torch
    lens, m = [900, 17, 25000, 300], [2, 2, 2, 2]
    c, q, out, work = _attn_case(lg, 2, lens, m, 8, 2, 128, 16, dtype, cache)
    again = torch.empty_like(out)
    work.fill_(17)
    c.c.attn(q, again, work, n_new=2)
    assert torch.equal(again, out)
    for r in range(4):
        alone = torch.empty_like(out[:2])
        one = lg.PagedCache(c.k, c.v, c.table[r:r + 1], c.len[r:r + 1])
        one.attn(q[2 * r:2 * r + 2], alone, work, n_new=2)
        step = 2 * HALF_STEP[dtype] * out[2 * r:2 * r + 2].abs().float() + (2.0 ** -16 if dtype != F32 else 2e-4)
        assert bool(((alone - out[2 * r:2 * r + 2]).abs().float() <= step).all()), r


@pytest.mark.parametrize("dtype,cache", [(F32, F16), (BF16, BF16), (F32, F32)])
def test_attention_leaves_out_bad_pages(lg, dtype, cache):
    """Pages outside the cache count as rows that no query sees; a request of nothing else gives zeros."""
    import torch
    c, q, out, work = _attn_case(lg, 6, [64, 48, 40], [1, 1, 1], 4, 2, 64, 16, dtype, cache)
    good = out.clone()
    c.table[1, 1] = c.k.shape[0]
    c.table[2, :3] = torch.tensor([-1, 1 << 30, -(1 << 31)], dtype=torch.int32, device="cuda")
    c.c.attn(q, out, work)
    assert c.status.item() == 8
    assert torch.equal(out[0], good[0]) and bool((out[2] == 0).all())
    table = c.oracle.table
    k, v = (torch.cat([x[table[1, 0]], x[table[1, 2]]]).double().cpu().numpy() for x in (c.k, c.v))
    want = attention(q[1:2].double().cpu().numpy(), k, v, 64 ** -0.5, [31])
    err = np.abs(out[1:2].double().cpu().numpy() - want)
    assert (err <= _tolerance(want, q[1:2].double().cpu().numpy(), k, v, 64 ** -0.5, dtype, cache)).all()
    c.status.zero_()
    c.len[0], c.len[1] = 1 << 30, -3                           # lengths outside the table's columns
    c.c.attn(q, out, work)
    assert c.status.item() == 8 and bool((out[1] == 0).all())


def test_attention_refuses_rows_that_it_does_not_cover(lg):
    import torch
    c, q, out, work = _attn_case(lg, 8, [40, 50, 60], [2, 1, 3], 4, 2, 64, 16, F32, F16, ragged=True)
    full = out.clone()
    out.fill_(99.0)
    c.c.attn(q, out, work, n_new=2, start=_i32([0, 2, 3, 6]))   # the last request has three rows: its third is left as it is
    assert c.status.item() == 32 and torch.equal(out[:5], full[:5]) and bool((out[5:] == 99.0).all())
    c.status.zero_()
    out.fill_(99.0)
    c.c.attn(q, out, work, n_new=3, start=_i32([0, 2, 1, 1 << 30]))   # falling starts, rows behind q: nothing of those
    assert c.status.item() == 32 and torch.equal(out[:2], full[:2]) and bool((out[2:] == 99.0).all())


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_infinities_and_nan_in_visible_rows(lg, dtype, cache):
    """As the formula: a score of -inf has no weight, NaN spreads to its own request and head only."""
    import torch
    c, q, out, work = _attn_case(lg, 12, [40, 40], [1, 1], 2, 2, 64, 16, dtype, cache)
    good = out.clone()
    table = c.oracle.table
    c.v[table[1, 0], 3, 1, 5] = float("nan")
    c.c.attn(q, out, work)
    assert torch.equal(out[0], good[0]) and torch.equal(out[1, 0], good[1, 0])
    assert bool(out[1, 1, 5].isnan()) and not bool(out[1, 1, :5].isnan().any())
    if dtype != cache or cache == F32:
        return                                                 # computed in parts: inf times parts of either sign
    c.k[table[0, 0], 0, 0] = torch.where(q[0, 0] > 0, float("-inf"), float("inf")).to(c.k.dtype)
    c.c.attn(q, out, work)
    k, v = (torch.cat([x[table[0, j]] for j in range(3)]).double().cpu().numpy()[1:40, :1] for x in (c.k, c.v))
    want = attention(q[:1, :1].double().cpu().numpy(), k, v, 64 ** -0.5, [38])
    err = np.abs(out[:1, :1].double().cpu().numpy() - want)
    assert (err <= _tolerance(want, q[:1, :1].double().cpu().numpy(), k, v, 64 ** -0.5, dtype, cache)).all()
    assert torch.equal(out[0, 1], good[0, 1])


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,window", [(2, 1, 64, 0), (8, 1, 128, 0), (4, 2, 256, 20), (2, 2, 512, 3)])
def test_a_bad_row_reaches_only_the_queries_that_see_it(lg, dtype, cache, heads, kv_heads, dim, window):
    """V rows of inf and NaN at the end of a verify block and at the beginning of its windows: the block's other queries are as without them."""
    import torch
    lens, m = [100, 21, 4], [4, 4, 4]
    c, q, out, work = _attn_case(lg, 21, lens, m, heads, kv_heads, dim, 16, dtype, cache, window=window)
    good, table = out.clone(), c.oracle.table
    for r, n in enumerate(lens):
        c.v[table[r, (n - 2) // 16], (n - 2) % 16] = float("nan")                 # rows 2 and 3 of the block see it
        if window:
            first = max(0, n - 4 - window + 1)
            if first + window <= n - 4 + 1:
                c.v[table[r, first // 16], first % 16] = float("inf")             # row 0 alone sees it
    c.c.attn(q, out, work, n_new=4, window=window)
    for r, n in enumerate(lens):
        spoilt = window and max(0, n - 4 - window + 1) + window <= n - 4 + 1
        for t in range(4):
            got, want = out[4 * r + t].float(), good[4 * r + t].float()
            if t >= 2:
                assert bool(got.isnan().all())
            elif t == 0 and spoilt:
                assert not bool(got.isfinite().any())
            else:
                # another order of the same sums: f32 rounding of up to 104 terms, then the type's
                assert bool(((got - want).abs() <= 2.0 ** -15 * c.v.float().nan_to_num(0, 0, 0).abs().max() + 2 * HALF_STEP[dtype] * want.abs()).all()), (r, t)


@pytest.mark.parametrize("dtype,page", [(F16, 16), (BF16, 10)])
def test_rows_past_two_to_the_31_elements(lg, dtype, page):
    """A cache of 2.4 G elements: append and attention at its end."""
    import torch
    dt, heads, dim = getattr(torch, dtype), 2, 128
    pages = 2_400_000_000 // (page * heads * dim)
    k, v = (torch.empty((pages, page, heads, dim), dtype=dt, device="cuda") for _ in range(2))
    n = 3 * page - 4
    table = _i32([[pages - 1, pages // 2, pages - 2]])
    slot = np.concatenate([p * page + np.arange(page) for p in table.cpu().numpy()[0]])[:n]
    torch.manual_seed(1)
    rows = [torch.randn((n, heads, dim), device="cuda").to(dt) for _ in range(2)]
    status = _i32([0])
    c = lg.PagedCache(k, v, table, _i32([n]), status=status)
    c.append(rows[0], rows[1], _i32(slot))
    assert all(torch.equal(x.view(-1, heads, dim)[_i32(slot).long()], r) for x, r in zip((k, v), rows))
    q = torch.randn((1, 4, dim), device="cuda")
    out = torch.empty_like(q)
    c.attn(q, out, torch.empty(c.attn_work(1, 1, 4), dtype=torch.uint8, device="cuda"))
    kk, vv, qd = rows[0].double().cpu().numpy(), rows[1].double().cpu().numpy(), q.double().cpu().numpy()
    want = attention(qd, kk, vv, dim ** -0.5, [n - 1])
    assert (np.abs(out.double().cpu().numpy() - want) <= _tolerance(want, qd, kk, vv, dim ** -0.5, F32, dtype)).all() and status.item() == 0
    del k, v, c
    torch.cuda.empty_cache()


def test_a_window_of_everything(lg):
    for window in (1 << 20, (1 << 31) - 1):
        _attn_case(lg, 3, [40, 7], [2, 2], 4, 2, 64, 16, F16, F16, window=window)


def test_calls_on_two_streams_with_workspaces_of_their_own(lg):
    import torch
    cases = [_attn_case(lg, s, [5000, 900, 64], [1, 1, 1], 8, 2, 128, 16, F32, F16) for s in (31, 32)]
    want = [x[2].clone() for x in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for (c, q, out, work), st in zip(cases, streams):
            c.c.attn(q, out, work, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(x[2], w) for x, w in zip(cases, want))


# ------------------------------------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------------------------------------

def test_steps_appends_and_attention_as_a_server_runs_them(lg):
    """Requests that come, grow, are cut back and leave; each step's rows go through step, append and attention on one stream, and the answers equal
    the contiguous-cache attention of this library over the same rows (both within its own tolerance of 2e-4)."""
    import torch
    rng = np.random.default_rng(11)
    torch.manual_seed(11)
    R, heads, kv_heads, dim, page = 6, 8, 2, 64, 16
    c = _Cache(lg, rng, [0] * R, page, 12, 40, kv_heads, dim, F16)
    kept = [[np.zeros((0, kv_heads * dim), np.float32)] * 2 for _ in range(R)]
    work = torch.empty(c.c.attn_work(R, 8, heads), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for kind in ("prompt", "one", "verify", "cut", "one", "leave", "verify", "one"):
        lens = c.oracle.len.copy()
        new = {"prompt": rng.integers(1, 8, R), "one": np.ones(R, int), "verify": np.full(R, 4), "cut": np.full(R, 4), "leave": rng.integers(0, 3, R)}[kind]
        keep = None
        if kind == "cut":
            keep = lens - rng.integers(0, 4, R)
        if kind == "leave":
            keep = np.where(np.arange(R) % 3 == 0, 0, lens)
        rows = int(new.sum())
        with torch.cuda.stream(side):
            got = c.step(new, rows + 2, keep, side.cuda_stream)
            k, v = (torch.randn((rows + 2, kv_heads, dim), device="cuda") for _ in range(2))
            q = torch.randn((rows + 2, heads, dim), device="cuda")
            out = torch.zeros_like(q)
            c.c.append(k, v, got[2], stream=side.cuda_stream)
            c.c.attn(q, out, work, n_new=8, start=got[0], scale=1.0, stream=side.cuda_stream)       # the other attention's scale
            side.synchronize()
        c.check(got, c.oracle.step(new, rows + 2, keep))
        at = 0
        for r in range(R):
            n = int(new[r])
            for j, x in enumerate((k, v)):
                old = kept[r][j][: lens[r] if keep is None else keep[r]]
                kept[r][j] = np.concatenate([old, x[at:at + n].reshape(n, kv_heads * dim).cpu().numpy()])
            if n:
                want = lg.flash_decode(q[at:at + n].cpu().numpy(), kept[r][0], kept[r][1], kv_heads, 0, len(kept[r][0]) - n)
                assert np.abs(out[at:at + n].cpu().numpy() - want).max() < 2e-4
            at += n
        assert bool((out[at:] == 0).all())


def test_captured_calls_follow_lengths_and_tables(lg):
    """Two graphs of a whole step, each with a workspace of its own, replayed while lengths change on the device."""
    import torch
    rng = np.random.default_rng(13)
    torch.manual_seed(13)
    R, heads, kv_heads, dim = 5, 4, 2, 128
    made = []
    for _ in range(2):
        c = _Cache(lg, rng, [300, 0, 20, 77, 1], 16, 40, 60, kv_heads, dim, BF16)
        c.k.normal_()
        c.v.normal_()
        new, start = _i32([1] * R), _i32([0] * (R + 1))
        pos, slot, req = (_i32([0] * R) for _ in range(3))
        k, v, q = (torch.randn((R, h, dim), device="cuda").to(torch.bfloat16) for h in (kv_heads, kv_heads, heads))
        out, work = torch.zeros_like(q), torch.empty(c.c.attn_work(R, 1, heads), dtype=torch.uint8, device="cuda")

        def go():
            st = torch.cuda.current_stream().cuda_stream
            c.c.step(new, start, pos, slot, req, stream=st)
            c.c.append(k, v, slot, stream=st)
            c.c.attn(q, out, work, start=start, stream=st)

        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            go()
        made.append((c, g, q, k, v, out, (new, start, pos, slot, req, work)))     # what a graph reads stays
    for _ in range(20):
        for c, g, *_ in made:
            g.replay()
    torch.cuda.synchronize()
    for c, g, q, k, v, out, _ in made:
        assert c.len.tolist() == [320, 20, 40, 97, 21] and c.status.item() == 0
        table = c.table.cpu().numpy()
        for r, n in enumerate(c.len.tolist()):
            kk, vv = (torch.cat([x[p] for p in table[r, : -(-n // 16)]])[:n].double().cpu().numpy() for x in (c.k, c.v))
            qd = q[r:r + 1].double().cpu().numpy()
            want = attention(qd, kk, vv, dim ** -0.5, [n - 1])
            err = np.abs(out[r:r + 1].double().cpu().numpy() - want)
            assert (err <= _tolerance(want, qd, kk, vv, dim ** -0.5, BF16, BF16)).all()


FIRST_CALLS = """
import importlib, torch
lg = importlib.import_module("little-gemma_b200")
i32 = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")
x, u, token, p = torch.randn(5, 40000, device="cuda"), torch.rand(5, device="cuda"), i32(5), torch.full((5,), 0.9, device="cuda")
k, q = torch.randn(20, 16, 2, 128, device="cuda").half(), torch.randn(2, 4, 128, device="cuda")
c = lg.PagedCache(k, k, torch.arange(20, device="cuda").int().view(2, 10), i32(2) + 100, i32(20), i32(1))
many = lg.PagedCache(k, k, i32(8192, 1), i32(8192), i32(20), i32(1))
out, work, start, start2 = torch.empty_like(q), torch.empty(c.attn_work(2, 1, 4), dtype=torch.uint8, device="cuda"), i32(3), i32(8193)
none, none2, g = i32(2), i32(8192), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream().cuda_stream
    c.step(none, start, stream=s)
    many.step(none2, start2, stream=s)
    c.attn(q, out, work, stream=s)
    lg.sample(x, u, token, top_p=p, stream=s)
g.replay()
torch.cuda.synchronize()
want, got = out.clone(), token.clone()
c.attn(q, out, work)
lg.sample(x, u, token, top_p=p)
assert torch.equal(out, want) and torch.equal(token, got) and bool(out.isfinite().all())
print("the same")
"""


def test_first_calls_of_a_process_may_be_captured():
    import subprocess
    import sys
    from tests.conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]


def test_host_memory_is_refused(lg):
    """Pointers that are no device memory: nothing is launched."""
    import torch
    c, q, out, work = _attn_case(lg, 1, [20], [1], 2, 1, 64, 16, F16, F16)
    for bad in ((q.cpu(), out, work), (q, out.cpu(), work), (q, out, work.cpu())):
        with pytest.raises(ValueError):
            c.c.attn(*bad)
    with pytest.raises(ValueError):
        c.c.append(torch.zeros(1, 64), torch.zeros(1, 64, device="cuda"), _i32([0]))
    with pytest.raises(ValueError):
        c.c.step(torch.zeros(1, dtype=torch.int32), _i32([0, 0]))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv_heads,dim", [(8, 128), (4, 256), (2, 512)])
def test_long_sums_of_one_sign_have_no_bias(lg, dtype, kv_heads, dim):
    """16 requests that share one document of 131072 rows, V between 1 and 2.5: answers may differ from the rounded 64-bit ones both ways alike.  A warp adds up
    at most 131072 / 16 / 2 slices; roundings to nearest of either sign, at most 2^-24 of the sum each, leave sqrt(4096) 2^-24 in the mean where all outputs
    had them in common (they do not): four times that."""
    import torch
    dt, n, R, page, gqa = getattr(torch, dtype), 131072, 16, 64, 4
    torch.manual_seed(dim)
    k = torch.randn((n // page, page, kv_heads, dim), device="cuda").to(dt)
    v = (1 + torch.rand((kv_heads, dim), device="cuda") + 0.5 * torch.rand((n // page, page, kv_heads, dim), device="cuda")).to(dt)
    c = lg.PagedCache(k, v, _i32(np.tile(np.arange(n // page), (R, 1))), _i32([n] * R))
    q = (0.3 * torch.randn((R, kv_heads * gqa, dim), device="cuda")).to(dt)
    out = torch.empty_like(q)
    c.attn(q, out, torch.empty(c.attn_work(R, 1, kv_heads * gqa), dtype=torch.uint8, device="cuda"))
    off = []
    for h in range(kv_heads):
        p = torch.softmax(q[:, h * gqa:(h + 1) * gqa].double().reshape(-1, dim) @ k[:, :, h].reshape(n, dim).double().T * dim ** -0.5, -1)
        want = p @ v[:, :, h].reshape(n, dim).double()
        got = out[:, h * gqa:(h + 1) * gqa].reshape(-1, dim).double()
        assert bool(((got - want).abs() <= (HALF_STEP[dtype] + 2.0 ** -14) * want).all())      # a tenth of half an f16 step beside the rounding
        off.append(((got - want.to(dt).double()) / want).mean().item())
    assert abs(np.mean(off)) <= 4 * 4096 ** 0.5 * 2.0 ** -24, off


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,new", [(8, 1, 512, 4), (7, 1, 512, 3), (8, 2, 512, 5), (16, 1, 256, 4), (8, 2, 256, 5), (32, 1, 128, 2), (64, 2, 64, 8), (40, 1, 80, 3)])
@pytest.mark.parametrize("window", [0, 20])
def test_a_bad_row_stays_with_the_tokens_that_see_it_where_a_block_is_several_groups(lg, dtype, cache, heads, kv_heads, dim, new, window):
    """More query rows a KV head than one tile has: groups of one token and groups across tokens."""
    import torch
    lens, m = [100, 33, new + 2], [new] * 3
    c, q, out, work = _attn_case(lg, 22, lens, m, heads, kv_heads, dim, 16, dtype, cache, window=window)
    good, table = out.clone(), c.oracle.table
    top = c.v.float().nan_to_num(0, 0, 0).abs().max()
    first = [max(0, n - new - window + 1) for n in lens]
    alone = [window > 0 and f + window <= n - new + 1 for f, n in zip(first, lens)]            # the first token alone sees that row
    for r, n in enumerate(lens):
        c.v[table[r, (n - 1) // 16], (n - 1) % 16] = float("nan")                 # the last token alone sees it
        if alone[r]:
            c.v[table[r, first[r] // 16], first[r] % 16] = float("inf")
    c.c.attn(q, out, work, n_new=new, window=window)
    for r in range(3):
        for t in range(new):
            got, want = out[r * new + t].float(), good[r * new + t].float()
            if t == new - 1:
                assert bool(got.isnan().all())
            elif t == 0 and alone[r]:
                assert not bool(got.isfinite().any())
            else:
                # another order of the same sums: f32 rounding of up to 104 terms, then the type's
                assert bool(((got - want).abs() <= 2.0 ** -15 * top + 2 * HALF_STEP[dtype] * want.abs()).all()), (r, t)


def _again(c, q, out, work, lens, m, kv_heads, window, dtype, cache, top=None):
    """The call on changed V rows against the 64-bit form: inf, NaN and finite numbers in the same places, the finite ones within _tolerance()."""
    c.c.attn(q, out, work, n_new=max(m), window=window)
    got, qd, table, at = out.double().cpu().numpy(), q.double().cpu().numpy(), c.oracle.table, 0
    for r, n in enumerate(lens):
        k, v = ((x[table[r, : -(-n // 16)]].double().flatten(0, 1)[:n]).cpu().numpy() for x in (c.k, c.v))
        positions = [n - m[r] + t for t in range(m[r])]
        lowest = max(0, positions[0] - window + 1) if window else 0
        k, v = k[lowest:], v[lowest:]
        with np.errstate(invalid="ignore"):
            want = attention(qd[at:at + m[r]], k, v, q.shape[-1] ** -0.5, [p - lowest for p in positions], window)
        g = got[at:at + m[r]]
        assert np.array_equal(np.isnan(g), np.isnan(want)), r
        fine = np.isfinite(want)
        assert np.array_equal(g[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), r
        flat = np.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
        tol = _tolerance(np.where(fine, want, 0.0), qd[at:at + m[r]], k, flat, q.shape[-1] ** -0.5, dtype, cache)
        assert (np.abs(g - want)[fine] <= tol[fine]).all(), r
        at += m[r]
    assert c.status.item() == 0


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,new,window", [(2, 1, 64, 1, 0), (8, 2, 128, 1, 100), (32, 1, 128, 2, 0), (16, 2, 256, 4, 20), (3, 1, 80, 3, 0), (8, 1, 512, 2, 0), (2, 2, 512, 1, 40)])
def test_infinities_in_v_as_the_formula(lg, dtype, cache, heads, kv_heads, dim, new, window):
    """inf times a weight, however small, is inf; two of either sign are NaN; the other dims are as ever."""
    inf, lens, m = float("inf"), [300, 40, 17 + new, 6000], [new] * 4
    c, q, out, work = _attn_case(lg, 41, lens, m, heads, kv_heads, dim, 16, dtype, cache, window=window)
    table = c.oracle.table
    for r, n in enumerate(lens):
        for back, d, x in ((1, 3, inf), (9, 4, -inf), (10, 4, -inf), (11, 5, inf), (12, 5, -inf), (12, 6, float("nan")), (13, 7, inf)):
            c.v[table[r, (n - back) // 16], (n - back) % 16, kv_heads - 1, d] = x
        if not window:
            c.v[table[r, 0], 0, 0, 1] = inf                    # far from the last row: other warps and CTAs join it
    _again(c, q, out, work, lens, m, kv_heads, window, dtype, cache)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_infinities_in_v_behind_weights_near_zero(lg, dtype, cache):
    """Weights of 1e-43 to 1e-130 of the largest: 0 in 32 bits, not in the formula."""
    lens = [100, 3000]
    c, q, out, work = _attn_case(lg, 42, lens, [1, 1], 2, 1, 64, 16, dtype, cache)
    table = c.oracle.table
    for r, n in enumerate(lens):
        # the last row leans towards head 0's query: its score is 100 to 300 above all others
        c.k[table[r, (n - 1) // 16], (n - 1) % 16] = (q[r, 0].float() * (200.0 * 8 / q[r, 0].float().square().sum())).to(c.k.dtype)
        for i in (0, 20, n - 2):
            c.v[table[r, i // 16], i % 16, 0, i % 7] = float("-inf")
    c.c.attn(q, out, work)
    for r, n in enumerate(lens):
        bad = {i % 7 for i in (0, 20, n - 2)}
        got = out[r, 0]
        assert all(got[d].item() == float("-inf") for d in bad), r
        last = c.v[table[r, (n - 1) // 16], (n - 1) % 16, 0].float()
        rest = [d for d in range(64) if d not in bad]
        assert bool(((got[rest].float() - last[rest]).abs() <= 2.0 ** -16 * last.abs().max() + HALF_STEP[dtype] * last[rest].abs()).all()), r


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,new", [(2, 1, 64, 1), (16, 2, 128, 4), (4, 1, 256, 1), (8, 1, 512, 2)])
def test_v_near_the_largest_number_of_its_type(lg, dtype, cache, heads, kv_heads, dim, new):
    """A mean of numbers is none larger, wherever it is added up: in a warp, over warps, over CTAs."""
    import torch
    lens, m = [1 + new, 7, 90, 20011], [new] * 4
    c, q, out, work = _attn_case(lg, 43, lens, m, heads, kv_heads, dim, 16, dtype, cache)
    most = torch.finfo(c.v.dtype).max
    for share in (1.0, 0.6):
        c.v.fill_(most * share)
        c.v[..., 1::2] = -most * share
        c.c.attn(q, out, work, n_new=new)
        want = c.v[0, 0, 0].double()                           # as the cache holds it
        # equal numbers: the sum of the weights over itself, 16 f32 roundings, then the type's; at the very top one of them may go over it
        near = (out.double() - want).abs() <= (2.0 ** -16 + HALF_STEP[dtype]) * most * share
        assert bool((near | ((share == 1.0) & (out.double() == want.sign() * float("inf")))).all()) and not bool(out.isnan().any()), share


@pytest.mark.parametrize("n", [2, 2000])
def test_an_entry_that_is_no_page_brings_none_back(lg, n):
    """Released with a bad entry in its table: the stack must not show again what another request took from that place."""
    rng = np.random.default_rng(n)
    c = _Cache(lg, rng, [8, 4] + [5] * (n - 2), 4, 6, 3 + 2 * n)
    c.step([8, 0] + [1] * (n - 2), 9 + n)                      # request 0 takes the two pages at the top
    c.table[1, 0] = -5
    c.table[n - 1, 0] = c.k.shape[0]
    c.step([0] * n, 0, [1 << 30, 0] + [0] * (n - 2))
    assert c.status.item() == Pages.BAD_PAGE

    def pages():
        table, lens, n_free = c.table.cpu().numpy(), c.len.cpu().numpy(), c.n_free.item()
        held = [int(x) for r in range(n) for x in table[r, : -(-int(lens[r]) // 4)]] + [int(x) for x in c.free.cpu().numpy()[:n_free]]
        return [p for p in held if 0 <= p < c.k.shape[0]]

    assert len(set(pages())) == len(pages()) == c.k.shape[0] - (1 if n == 2 else 2)          # a bad entry's own page is lost
    c.status.zero_()
    start, _, slot, req = c.step([0] + [9] * (n - 1), 9 * n)
    live = [int(s) for s in slot.tolist() if s >= 0]
    assert len(set(pages())) == len(pages()) and len(set(live)) == len(live)
    assert c.status.item() == Pages.BAD_PAGE and req.tolist().count(1) == 9 and slot.tolist().count(-1) > 9
    taken = set(c.table.cpu().numpy()[0, :4].tolist())
    assert not taken & {s // 4 for s in live}


def test_a_step_without_outputs_for_tokens_has_no_limit_of_rows(lg):
    """The largest cap there is, with pos, slot and req NULL: the loop over rows ends at the step's own."""
    import ctypes
    rng = np.random.default_rng(15)
    c = _Cache(lg, rng, [5, 0, 16, 3000], 16, 200, 20)
    for new, keep in (([3, 1, 0, 90], None), ([0, 0, 0, 0], [5, 0, 9, 3000]), ([1, 0, 1 << 30, 2], None)):
        start, d_new, d_keep = _i32([-7] * 5), _i32(new), None if keep is None else _i32(keep)
        assert lg.load().lg_paged_step(ctypes.byref(c.c.desc), 4, d_keep.data_ptr() if keep else None, d_new.data_ptr(), (1 << 31) - 1, start.data_ptr(), None, None, None, None) == 0
        want = c.oracle.step(new, 200, keep)
        assert start.tolist() == want[0] and c.status.item() == want[4]
        assert c.len.tolist() == c.oracle.len.tolist() and np.array_equal(c.table.cpu().numpy(), c.oracle.table) and c.n_free.item() == c.oracle.n_free
        c.status.zero_()


def test_a_step_without_outputs_serves_what_its_cap_allows(lg):
    rng = np.random.default_rng(16)
    c = _Cache(lg, rng, [5, 0, 16], 16, 8, 9)
    start = _i32([-7] * 4)
    c.c.step(_i32([3, 1, 0]), start)                           # no room given: nobody with new rows
    assert start.tolist() == [0, 0, 0, 0] and c.len.tolist() == [5, 0, 16] and c.status.item() == Pages.NO_ROWS
    c.status.zero_()
    c.c.step(_i32([3, 1, 20]), start, cap=24)
    want = c.oracle.step([3, 1, 20], 24)
    assert start.tolist() == want[0] == [0, 3, 4, 24] and c.len.tolist() == [8, 1, 36] and c.status.item() == 0
    assert np.array_equal(c.table.cpu().numpy(), c.oracle.table)


def test_who_is_served_goes_by_the_declared_rule(lg):
    from tests.test_serve_cpu import SERVED
    for (lens, new, free, cap), (served, status) in SERVED:
        c = _Cache(lg, np.random.default_rng(1), lens, 16, 4, free)
        start, *_ = c.step(new, cap)
        assert c.len.tolist() == [n + m * s for n, m, s in zip(lens, new, served)] and c.status.item() == status
        assert start.tolist() == [sum(m * s for m, s in zip(new[:i], served[:i])) for i in range(len(new) + 1)]


@pytest.mark.parametrize("cache", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (6, 3, 128), (4, 2, 256), (8, 1, 512)])
def test_f32_answers_are_as_exact_as_f32_sums(lg, cache, heads, kv_heads, dim):
    """The error in the norm.  A score (1.5 on average) is a sum in 8 steps per 128 dims, each of which cuts off half of 2^-23 of a partial sum, half the score, on
    average: 3 2^-23; as much for the sums over 128 dims, the lower parts, scale and maximum together; 2^-22 for the exponential: an error of a weight of
    8 2^-23, which is the answer's."""
    import torch
    torch.manual_seed(dim)
    n, page = 4000, 16
    k, v = (torch.randn((n // page, page, kv_heads, dim), device="cuda").to(getattr(torch, cache)) for _ in range(2))
    c = lg.PagedCache(k, v, _i32(np.arange(n // page)[None]), _i32([n]))
    q = 1.5 * torch.randn((1, heads, dim), device="cuda")
    out = torch.empty_like(q)
    c.attn(q, out, torch.empty(c.attn_work(1, 1, heads), dtype=torch.uint8, device="cuda"))
    want = attention(q.double().cpu().numpy(), k.flatten(0, 1).double().cpu().numpy(), v.flatten(0, 1).double().cpu().numpy(), dim ** -0.5, [n - 1])
    assert np.linalg.norm(out.double().cpu().numpy() - want) <= 2.0 ** -20 * np.linalg.norm(want)
