"""The operators of the 4-bit cache on the GPU against plain ones in 64 bits (plain_cache4.py)."""
import numpy as np
import pytest
import torch

import plain_cache4 as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from kvcm_amd import ops as _ops
    _ops.lib()
    return _ops


def ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device=DEV)


def garbage(ops, pages, nkv, hd, page, gen):
    """A cache whose every byte is anything: what reused pages hold beyond their owner's tokens (NaN and Inf steps among it)."""
    return torch.randint(0, 256, ops.cache4_shape(pages, nkv, hd, page), generator=gen, dtype=torch.uint8).to(DEV)


def filled(ops, pages, nkv, hd, page, gen, slots, dtype=BF):
    """Garbage, with sound tokens at ``slots``."""
    cache = garbage(ops, pages, nkv, hd, page, gen)
    x = torch.randn(len(slots), 3 * nkv * hd, generator=gen) + 2 * (torch.rand(3 * nkv * hd, generator=gen) < 0.1)
    ops.rope_cache4(x.to(dtype).to(DEV), nkv, nkv, hd, cache, ints(slots))
    return cache


# ----------------------------------------------------------------------------------- writing and reading
def rotated(x, cos_sin, dtype):
    """[rows, heads, hd] rotated as the rows' type has it: bfloat16 in 32 bits (one product rounded, the other kept whole), float32 in 64."""
    a, b = np.split(x, 2, -1)
    cs, sn = (cos_sin[:, None, :, i].astype(np.float64) for i in (0, 1))
    if dtype == F32:
        return np.concatenate([(a * cs - b * sn).astype(np.float32), (b * cs + a * sn).astype(np.float32)], -1).astype(np.float64)
    r32 = lambda v: v.astype(np.float32).astype(np.float64)
    return plain.bf16(np.concatenate([r32(a * cs - r32(b * sn)), r32(b * cs + r32(a * sn))], -1))


@pytest.mark.parametrize("dtype", (BF, F32))
@pytest.mark.parametrize("nh, nkv, hd, page, rotate", ((3, 1, 32, 16, True), (8, 2, 64, 32, True), (4, 4, 128, 16, True), (2, 1, 256, 48, True), (8, 2, 64, 16, False),
                                                       (2, 2, 32, 64, False)))
def test_store_writes_the_format_and_nothing_else(ops, nh, nkv, hd, page, rotate, dtype):
    gen = torch.Generator().manual_seed(nh * hd + page)
    T, pages, width = 23, 7, (nh + 2 * nkv) * hd
    rows = torch.randn(T, width, generator=gen) * torch.exp(2 * torch.randn(T, 1, generator=gen))
    rows[3] = 0.0
    rows[4] = 1.5                                        # no range: step 0
    rows[5, ::3] = 2.0 ** -130                           # ranges of denormal steps
    rows[6] *= 1e30
    rows[15] = 1.005                                     # float rows: no range, and low is rounded above it
    rows[16] = 1.001                                     # and below it
    if not rotate:
        rows[17, nh * hd] = 3e38                         # a range that passes the largest float
        rows[17, nh * hd + 1] = -3e38
        rows[7, nh * hd + 1] = float("inf")
        rows[8, -1] = float("nan")
        rows[9, -hd:] = float("-inf")
        rows[10, nh * hd] = -3.3e38
        rows[11, nh * hd] = 3e-39
    wide = torch.full((T, width + 24), 7.0).to(dtype)
    wide[:, 8:8 + width] = rows.to(dtype)
    held = wide.to(DEV)
    qkv = held[:, 8:8 + width] if dtype == F32 else held[:, 8:8 + width]
    slots = torch.randperm(pages * page, generator=gen)[:T].tolist()
    slots[12], slots[13], slots[14] = -1, pages * page, -2 ** 31
    before = garbage(ops, pages, nkv, hd, page, gen)
    cache = before.clone()
    table = None
    if rotate:
        angles = torch.rand(T, hd // 2, generator=gen) * 40
        table = torch.stack([angles.cos(), angles.sin()], -1).contiguous()
    ops.rope_cache4(qkv, nh, nkv, hd, cache, ints(slots), cos_sin=None if table is None else table.to(DEV))
    x = rows.to(dtype).double().numpy().reshape(T, nh + 2 * nkv, hd)
    if rotate:
        x[:, :nh + nkv] = rotated(x[:, :nh + nkv], table.numpy(), dtype)
    want = before.cpu().numpy()
    for r, s in enumerate(slots):
        if 0 <= s < pages * page:
            for g in range(nkv):
                plain.write(want, s, g, x[r, nh + g], x[r, nh + nkv + g])
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    after = held.cpu()
    assert torch.equal(after[:, :8], wide[:, :8]) and torch.equal(after[:, 8 + width:], wide[:, 8 + width:])
    assert torch.equal(after[:, 8 + nh * hd:8 + width].nan_to_num(5.0), wide[:, 8 + nh * hd:8 + width].nan_to_num(5.0))
    assert torch.equal(after[:, 8:8 + nh * hd].double(), torch.as_tensor(x[:, :nh]).reshape(T, -1))


def test_store_takes_one_row_many_rows_none_and_a_place_for_the_queries(ops):
    gen = torch.Generator().manual_seed(5)
    nh, nkv, hd, page, pages = 4, 2, 64, 16, 90
    for T in (0, 1, 1300):
        qkv = torch.randn(max(T, 2), (nh + 2 * nkv) * hd, generator=gen).to(BF).to(DEV)
        angles = torch.rand(max(T, 2), hd // 2, generator=gen)
        table = torch.stack([angles.cos(), angles.sin()], -1).to(DEV)
        slots = torch.randperm(pages * page, generator=gen)[:max(T, 2)].to(torch.int32).to(DEV)
        one, two = (torch.zeros(ops.cache4_shape(pages, nkv, hd, page), dtype=torch.uint8, device=DEV) for _ in range(2))
        kept, q = qkv.clone(), torch.full((max(T, 2), nh * hd + 3), 9.0, dtype=BF, device=DEV)
        ops.rope_cache4(qkv, nh, nkv, hd, one, slots, cos_sin=table, q_out=q, rows=T)
        assert torch.equal(qkv, kept)
        ops.rope_cache4(qkv, nh, nkv, hd, two, slots, cos_sin=table, rows=T)
        assert torch.equal(one, two) and torch.equal(q[:T, :nh * hd], qkv[:T, :nh * hd]) and torch.equal(qkv[T:], kept[T:])
        assert bool((q[:, nh * hd:] == 9).all()) and bool((q[T:] == 9).all())
        assert T > 0 or not one.any()


@pytest.mark.parametrize("dtype", (BF, F32))
@pytest.mark.parametrize("nkv, hd, page", ((1, 32, 16), (3, 64, 32), (2, 128, 16), (2, 256, 16)))
def test_read_gives_what_the_bytes_stand_for(ops, nkv, hd, page, dtype):
    gen = torch.Generator().manual_seed(hd)
    pages = 5
    slots = list(range(pages * page))
    cache = filled(ops, pages, nkv, hd, page, gen, slots)
    order = torch.randperm(len(slots), generator=gen)[:57].tolist() + [-1, pages * page, 3, 3]      # one twice, two of none
    k, v = (torch.full((len(order) + 1, nkv * hd + 5), 9.0, dtype=dtype, device=DEV) for _ in range(2))
    ops.cache4_rows(cache, ints(order), k, v)
    kc, ks, kl, vc, vs, vl = plain.parts(cache, nkv, hd)
    valid = torch.tensor([0 <= s < pages * page for s in order], device=DEV)
    at = ints(order).long().clamp(0, pages * page - 1)
    for got, want in ((k, kl + ks * kc), (v, vl + vs * vc)):
        want = torch.where(valid.view(-1, 1), want[at].flatten(1), torch.zeros((), dtype=torch.float64, device=DEV))
        assert torch.equal(got[:-1, :nkv * hd], want.to(dtype))
        assert bool((got[:, nkv * hd:] == 9).all()) and bool((got[-1] == 9).all())


def test_a_token_is_within_half_a_step(ops):
    """|x - value| <= step / 2 + 15 * 2^-9 step at the top (a step rounded down) for bfloat16 vectors, whose low is exact."""
    gen = torch.Generator().manual_seed(2)
    nkv, hd, T = 4, 128, 256
    x = torch.randn(T, 3 * nkv * hd, generator=gen).to(BF).to(DEV)
    cache = torch.zeros(ops.cache4_shape(16, nkv, hd, 16), dtype=torch.uint8, device=DEV)
    ops.rope_cache4(x, nkv, nkv, hd, cache, ints(range(T)))
    k, v = (torch.empty(T, nkv * hd, device=DEV) for _ in range(2))
    ops.cache4_rows(cache, ints(range(T)), k, v)
    for got, want in ((k, x[:, nkv * hd:2 * nkv * hd]), (v, x[:, 2 * nkv * hd:])):
        a, b = got.view(T, nkv, hd), want.float().view(T, nkv, hd)
        step = (b.amax(-1, keepdim=True) - b.amin(-1, keepdim=True)) / 15
        assert bool(((a - b).abs() <= step * (0.5 * (1 + 2.0 ** -8) + 15 * 2.0 ** -9 + 1e-5)).all())


# ----------------------------------------------------------------------------------- attention
SIZES = ((4, 4, 32, 16), (8, 1, 64, 16), (6, 2, 64, 32), (8, 8, 128, 16), (8, 2, 128, 64), (34, 2, 64, 16), (4, 2, 256, 16))


class Sequences:
    """Page tables of sequences of given lengths over a shuffled pool with garbage in every other place."""

    def __init__(self, ops, nh, nkv, hd, page, lengths, gen, dtype, spare=2):
        self.nh, self.nkv, self.hd, self.page, self.dtype = nh, nkv, hd, page, dtype
        need = [-(-n // page) for n in lengths]
        self.pages, self.stride = sum(need) + spare, max(max(need), 1) + 1
        order = torch.randperm(self.pages, generator=gen).tolist()
        self.tables = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(lengths), self.stride), generator=gen).to(torch.int32)      # beyond a length: anything
        self.slots = []
        for i, n in enumerate(lengths):
            mine = [order.pop() for _ in range(need[i])]
            self.tables[i, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            self.slots.append(torch.tensor([mine[t // page] * page + t % page for t in range(n)], dtype=torch.long, device=DEV))
        self.cache = filled(ops, self.pages, nkv, hd, page, gen, torch.cat(self.slots).tolist(), dtype)
        self.held = plain.parts(self.cache, nkv, hd)
        self.dev_tables = self.tables.to(DEV).view(-1)

    def expect(self, q, seqs, visible, scale):
        none = torch.zeros(0, dtype=torch.long, device=DEV)
        return plain.attend(q.double().view(q.shape[0], self.nh, self.hd), self.held, [self.slots[s] if s >= 0 else none for s in seqs], visible,
                            self.nh, self.nkv, scale, self.dtype)


def near(out, want, tol):
    got = out.double().view(want.shape)
    assert not bool(got.isnan().any())
    worst = ((got - want).abs() / tol.clamp_min(1e-30)).max()
    assert bool(((got - want).abs() <= tol).all()), f"{float(worst):.3f} of the tolerance"


def queries(rows, width, dtype, gen, extra=0):
    return torch.randn(rows, width + extra, generator=gen).to(dtype).to(DEV)


LENGTHS = (1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 300)


@pytest.mark.parametrize("window", (0, 1, 40))
@pytest.mark.parametrize("dtype", (BF, F32))
@pytest.mark.parametrize("nh, nkv, hd, page", SIZES)
def test_decode(ops, nh, nkv, hd, page, dtype, window):
    gen = torch.Generator().manual_seed(nh * hd + page)
    s = Sequences(ops, nh, nkv, hd, page, LENGTHS, gen, dtype)
    # every sequence twice, the second time not to its end; padding rows between; sequences that have no table
    seqs = list(range(len(LENGTHS))) + list(range(len(LENGTHS))) + [0, 3, -1, len(LENGTHS)]
    ctx = list(LENGTHS) + [max(1, n // 2) for n in LENGTHS] + [0, -7, 20, 20]
    order = torch.randperm(len(seqs), generator=gen).tolist()
    seqs, ctx = [seqs[i] for i in order], [ctx[i] for i in order]
    T = len(seqs)
    q = queries(T + 2, nh * hd, dtype, gen, extra=2 * nkv * hd)
    out = torch.full((T + 2, nh * hd + 8), 9.0, dtype=dtype, device=DEV)
    scale = hd ** -0.5
    ops.attention_decode4(q, out, s.cache, s.dev_tables, s.stride, ints(seqs), ints(ctx), nh, nkv, hd, scale, max(LENGTHS), window=window, rows=T)
    sound = [0 <= n < len(LENGTHS) for n in seqs]
    visible = [(max(0, c - window) if window else 0, c) if ok else (0, 0) for c, ok in zip(ctx, sound)]
    want, tol = s.expect(q[:T, :nh * hd], [n if ok else -1 for n, ok in zip(seqs, sound)], visible, scale)
    near(out[:T, :nh * hd], want, tol)
    assert bool((out[:, nh * hd:] == 9).all()) and bool((out[T:] == 9).all())


@pytest.mark.parametrize("rows, ctx, window", ((1, 5000, 0), (3, 4097, 0), (1, 5000, 4000), (2, 1500, 0), (40, 700, 0)))
@pytest.mark.parametrize("nh, nkv, hd, dtype", ((8, 1, 64, BF), (4, 2, 128, BF), (4, 2, 64, F32)))
def test_decode_over_contexts_cut_into_parts(ops, nh, nkv, hd, dtype, rows, ctx, window):
    gen = torch.Generator().manual_seed(rows + ctx)
    lengths = [ctx] + [max(1, ctx // (i + 1) - i) for i in range(1, rows)]
    s = Sequences(ops, nh, nkv, hd, 16, lengths, gen, dtype)
    q, out = queries(rows, nh * hd, dtype, gen), torch.empty(rows, nh * hd, dtype=dtype, device=DEV)
    args = (q, out, s.cache, s.dev_tables, s.stride, ints(range(rows)), ints(lengths), nh, nkv, hd, hd ** -0.5)
    visible = [(max(0, n - window) if window else 0, n) for n in lengths]
    want, tol = s.expect(q, range(rows), visible, hd ** -0.5)
    for bound in (ctx, 4 * ctx):
        ops.attention_decode4(*args, bound, window=window)
        near(out, want, tol)
    first = out.clone()
    ops.attention_decode4(*args, 4 * ctx, window=window)
    assert torch.equal(first, out)


@pytest.mark.parametrize("window", (0, 1, 29))
@pytest.mark.parametrize("dtype", (BF, F32))
@pytest.mark.parametrize("nh, nkv, hd, page", SIZES)
def test_prefill(ops, nh, nkv, hd, page, dtype, window):
    gen = torch.Generator().manual_seed(nh + hd + page)
    runs = (1, 70, 2, 0, 17, 33, 1, 16, 5)
    starts = (0, 0, 15, 7, 16, 100, 63, 1, 290)
    s = Sequences(ops, nh, nkv, hd, page, [r + p for r, p in zip(runs, starts)], gen, dtype)
    first = np.concatenate([[3], 3 + np.cumsum(runs)])      # rows before the first run and behind the last belong to nobody
    T = int(first[-1]) + 4
    q = queries(T, nh * hd, dtype, gen, extra=2 * nkv * hd)
    out = torch.full((T, nh * hd), 9.0, dtype=dtype, device=DEV)
    scale = hd ** -0.5
    ops.attention_prefill4(q, out, s.cache, s.dev_tables, s.stride, ints(first), ints(starts), len(runs), max(runs), nh, nkv, hd, scale, window=window)
    seqs = [i for i, r in enumerate(runs) for _ in range(r)]
    pos = [p + j for r, p in zip(runs, starts) for j in range(r)]
    want, tol = s.expect(q[3:T - 4, :nh * hd], seqs, [(max(0, p + 1 - window) if window else 0, p + 1) for p in pos], scale)
    near(out[3:T - 4], want, tol)
    assert bool((out[:3] == 9).all()) and bool((out[T - 4:] == 9).all())


@pytest.mark.parametrize("runs, starts, window", (((3,), (3000,), 0), ((130, 40), (900, 2100), 0), ((100,), (2000,), 1500), ((257,), (0,), 0)))
@pytest.mark.parametrize("nh, nkv, hd, dtype", ((8, 1, 64, BF), (2, 2, 128, BF), (4, 2, 64, F32)))
def test_prefill_behind_long_contexts(ops, nh, nkv, hd, dtype, runs, starts, window):
    gen = torch.Generator().manual_seed(sum(starts))
    s = Sequences(ops, nh, nkv, hd, 16, [r + p for r, p in zip(runs, starts)], gen, dtype)
    first = np.concatenate([[0], np.cumsum(runs)])
    T = int(first[-1])
    q, out = queries(T, nh * hd, dtype, gen), torch.empty(T, nh * hd, dtype=dtype, device=DEV)
    args = (q, out, s.cache, s.dev_tables, s.stride, ints(first), ints(starts), len(runs), max(runs), nh, nkv, hd, hd ** -0.5)
    seqs = [i for i, r in enumerate(runs) for _ in range(r)]
    pos = [p + j for r, p in zip(runs, starts) for j in range(r)]
    rows = list(range(0, T, 7)) + [T - 1]
    want, tol = s.expect(q[rows], [seqs[i] for i in rows], [(max(0, pos[i] + 1 - window) if window else 0, pos[i] + 1) for i in rows], hd ** -0.5)
    for kw in (dict(max_context=max(r + p for r, p in zip(runs, starts))), {}):
        ops.attention_prefill4(*args, window=window, **kw)
        near(out[rows], want, tol)
    again = out.clone()
    ops.attention_prefill4(*args, window=window)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", (BF, F32))
def test_infinities_and_nan_stay_with_the_rows_that_see_them(ops, dtype):
    """A token whose key (or value) is not finite: rows before it, rows of other heads and rows whose window has passed it are as ever."""
    nh, nkv, hd, page, n, bad = 4, 2, 64, 16, 90, 50
    gen = torch.Generator().manual_seed(1)
    s = Sequences(ops, nh, nkv, hd, page, (n,), gen, dtype)
    rows = torch.randn(2, 3 * nkv * hd, generator=gen).to(dtype)
    rows[0, nkv * hd + 5] = float("nan")          # token 50: the first kv head's key
    rows[1, -1] = float("inf")                    # token 51: the second's value
    ops.rope_cache4(rows.to(DEV), nkv, nkv, hd, s.cache, s.slots[0][bad:bad + 2].to(torch.int32))
    s.held = plain.parts(s.cache, nkv, hd)
    q = queries(n, nh * hd, dtype, gen)
    scale, window = hd ** -0.5, 20
    for w in (0, window):
        out, one = torch.empty(n, nh * hd, dtype=dtype, device=DEV), torch.empty(n, nh * hd, dtype=dtype, device=DEV)
        ops.attention_prefill4(q, out, s.cache, s.dev_tables, s.stride, ints([0, n]), ints([0]), 1, n, nh, nkv, hd, scale, window=w)
        ops.attention_decode4(q, one, s.cache, s.dev_tables, s.stride, ints([0] * n), ints(range(1, n + 1)), nh, nkv, hd, scale, n, window=w)
        want, tol = s.expect(q, [0] * n, [(max(0, p + 1 - w) if w else 0, p + 1) for p in range(n)], scale)
        for got in (out, one):
            got = got.double().view(n, nh, hd)
            for g in range(nkv):
                mine = torch.arange(n, device=DEV)
                sees = (mine >= bad + g) & ((mine - w < bad + g) if w else True)
                of = slice(g * nh // nkv, (g + 1) * nh // nkv)
                assert bool(got[sees][:, of].isnan().all())
                near(got[~sees][:, of], want[~sees][:, of], tol[~sees][:, of])


@pytest.mark.parametrize("dtype", (BF, F32))
def test_large_scores_and_constant_keys(ops, dtype):
    """Scores far beyond what exp holds, keys all alike (step 0), a scale of 0."""
    nh, nkv, hd, page, n = 8, 2, 64, 16, 70
    gen = torch.Generator().manual_seed(4)
    s = Sequences(ops, nh, nkv, hd, page, (n, n), gen, dtype)
    x = torch.randn(n, 3 * nkv * hd, generator=gen)
    x[:, nkv * hd:2 * nkv * hd] = 0.75
    ops.rope_cache4(x.to(dtype).to(DEV), nkv, nkv, hd, s.cache, s.slots[1].to(torch.int32))
    s.held = plain.parts(s.cache, nkv, hd)
    q, out = queries(4, nh * hd, dtype, gen), torch.empty(4, nh * hd, dtype=dtype, device=DEV)
    for scale in (hd ** -0.5, 200.0, 0.0):
        ops.attention_decode4(q, out, s.cache, s.dev_tables, s.stride, ints([0, 1, 0, 1]), ints([n, n, 9, 9]), nh, nkv, hd, scale, n)
        want, tol = s.expect(q, [0, 1, 0, 1], [(0, n), (0, n), (0, 9), (0, 9)], scale)
        near(out, want, tol)


def test_pages_that_are_none_hide_their_tokens(ops):
    nh, nkv, hd, page = 4, 2, 64, 16
    gen = torch.Generator().manual_seed(6)
    s = Sequences(ops, nh, nkv, hd, page, (64, 64), gen, BF)
    tables = s.dev_tables.clone().view(2, -1)
    tables[0, 1], tables[1] = s.pages, -1
    q, out = queries(2, nh * hd, BF, gen), torch.empty(2, nh * hd, dtype=BF, device=DEV)
    ops.attention_decode4(q, out, s.cache, tables.view(-1), s.stride, ints([0, 1]), ints([64, 64]), nh, nkv, hd, 0.125, 64)
    s.slots[0] = torch.cat([s.slots[0][:16], s.slots[0][32:]])
    want, tol = s.expect(q, [0, -1], [(0, 48), (0, 0)], 0.125)
    near(out, want, tol)
    runs = torch.empty(2, nh * hd, dtype=BF, device=DEV)
    ops.attention_prefill4(q, runs, s.cache, tables.view(-1), s.stride, ints([0, 1, 2]), ints([63, 63]), 2, 1, nh, nkv, hd, 0.125)
    near(runs, want, tol)


@pytest.mark.parametrize("dtype", (BF, F32))
def test_other_places_signs_and_ranges(ops, dtype):
    """Rows from any element on (2 or 4 bytes of alignment), a negative scale, keys and values far from 0 and far apart in size."""
    nh, nkv, hd, page = 6, 2, 64, 32
    gen = torch.Generator().manual_seed(11)
    lengths = (77, 200, 31)
    s = Sequences(ops, nh, nkv, hd, page, lengths, gen, dtype)
    x = torch.randn(sum(lengths), 3 * nkv * hd, generator=gen) * torch.exp(3 * torch.randn(sum(lengths), 1, generator=gen)) + 5 * torch.randn(3 * nkv * hd, generator=gen)
    wide = torch.zeros(sum(lengths), 3 * nkv * hd + 9, dtype=dtype, device=DEV)
    wide[:, 3:-6] = x.to(dtype).to(DEV)
    ops.rope_cache4(wide[:, 3:-6], nkv, nkv, hd, s.cache, torch.cat(s.slots).to(torch.int32))
    s.held = plain.parts(s.cache, nkv, hd)
    q = queries(3, nh * hd, dtype, gen, extra=5)
    out = torch.full((3, nh * hd + 7), 9.0, dtype=dtype, device=DEV)
    for scale in (0.05, -0.05):
        want, tol = s.expect(q[:, 1:nh * hd + 1], range(3), [(0, n) for n in lengths], scale)
        ops.attention_decode4(q[:, 1:], out[:, 5:], s.cache, s.dev_tables, s.stride, ints(range(3)), ints(lengths), nh, nkv, hd, scale, max(lengths))
        near(out[:, 5:nh * hd + 5], want, tol)
        ops.attention_prefill4(q[:, 1:], out[:, 1:], s.cache, s.dev_tables, s.stride, ints(range(4)), ints(n - 1 for n in lengths), 3, 1, nh, nkv, hd, scale)
        near(out[:, 1:nh * hd + 1], want, tol)
        assert bool((out[:, nh * hd + 5:] == 9).all()) and bool((out[:, 0] == 9).all())


def test_scores_that_rise_and_fall_along_a_context(ops):
    """m follows late (scores up to 2^6 above it are taken as they are): steps of every size up and down, in every wave's tokens."""
    nh, nkv, hd, page, n = 2, 1, 32, 16, 700
    gen = torch.Generator().manual_seed(12)
    for dtype in (BF, F32):
        s = Sequences(ops, nh, nkv, hd, page, (n,), gen, dtype)
        along = torch.cumsum(torch.randn(n, generator=gen), 0) * torch.linspace(0.1, 3, n)
        x = torch.randn(n, 3 * hd, generator=gen)
        x[:, hd:2 * hd] += along.view(-1, 1)
        ops.rope_cache4(x.to(dtype).to(DEV), 1, 1, hd, s.cache, s.slots[0].to(torch.int32))
        s.held = plain.parts(s.cache, nkv, hd)
        q = queries(n, nh * hd, dtype, gen) + 0.3
        out = torch.empty(n, nh * hd, dtype=dtype, device=DEV)
        ops.attention_prefill4(q, out, s.cache, s.dev_tables, s.stride, ints([0, n]), ints([0]), 1, n, nh, nkv, hd, hd ** -0.5)
        want, tol = s.expect(q, [0] * n, [(0, p + 1) for p in range(n)], hd ** -0.5)
        near(out, want, tol)
        one = torch.empty(n, nh * hd, dtype=dtype, device=DEV)
        ops.attention_decode4(q, one, s.cache, s.dev_tables, s.stride, ints([0] * n), ints(range(1, n + 1)), nh, nkv, hd, hd ** -0.5, n)
        near(one, want, tol)


def test_a_cache_of_more_than_4_gib(ops):
    nh, nkv, hd, page = 4, 2, 256, 16
    pages = (1 << 32) // (nkv * 16 * (hd + 8)) + 40
    gen = torch.Generator().manual_seed(13)
    cache = torch.empty(ops.cache4_shape(pages, nkv, hd, page), dtype=torch.uint8, device=DEV)
    n = 50
    mine = [pages - 1, 3, pages - 7, pages - 20]
    slots = torch.tensor([mine[t // page] * page + t % page for t in range(n)], dtype=torch.int32, device=DEV)
    x = torch.randn(n, 3 * nkv * hd, generator=gen).to(BF).to(DEV)
    ops.rope_cache4(x, nkv, nkv, hd, cache, slots)
    k, v = (torch.empty(n, nkv * hd, dtype=F32, device=DEV) for _ in range(2))
    ops.cache4_rows(cache, slots, k, v)
    small, there = torch.zeros(ops.cache4_shape(4, nkv, hd, page), dtype=torch.uint8, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV)
    ops.rope_cache4(x, nkv, nkv, hd, small, there)
    k2, v2 = (torch.empty_like(k) for _ in range(2))
    ops.cache4_rows(small, there, k2, v2)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    q = queries(1, nh * hd, BF, gen)
    one, two = torch.empty_like(q), torch.empty_like(q)
    ops.attention_decode4(q, one, cache, ints(mine), 4, ints([0]), ints([n]), nh, nkv, hd, 0.06, n)
    ops.attention_decode4(q, two, small, ints(range(4)), 4, ints([0]), ints([n]), nh, nkv, hd, 0.06, n)
    assert torch.equal(one, two)


class Served:
    """A few sequences on their way through a model's attention: a prompt's portion or a token of each at a time, written and attended over."""

    def __init__(self, ops, nh, nkv, hd, page, room, seqs, dtype, seed):
        self.gen = torch.Generator().manual_seed(seed)
        self.size = (nh, nkv, hd)
        self.ops, self.page, self.dtype, self.stride = ops, page, dtype, -(-room // page)
        pages = seqs * self.stride + 1
        self.tables = torch.randperm(pages, generator=self.gen)[:seqs * self.stride].to(torch.int32).to(DEV).view(seqs, -1)
        self.cache = garbage(ops, pages, nkv, hd, page, self.gen)
        self.room, self.lens = room, [0] * seqs
        self.buffers = {}

    def inputs(self, runs):
        """A step's rows, runs[i] of sequence i, in buffers that stay where they are from one step of the same runs to the next."""
        nh, nkv, hd = self.size
        T = sum(runs)
        seq = [i for i, r in enumerate(runs) for _ in range(r)]
        pos = [self.lens[i] + j for i, r in enumerate(runs) for j in range(r)]
        table = self.tables.cpu()
        angle = torch.tensor(pos).view(-1, 1) * 10000.0 ** (-torch.arange(hd // 2) * 2 / hd)
        new = dict(qkv=torch.randn(T, (nh + 2 * nkv) * hd, generator=self.gen).to(self.dtype), slots=torch.tensor([int(table[s, p // self.page]) * self.page + p % self.page for s, p in zip(seq, pos)]),
                   cos_sin=torch.stack([angle.cos(), angle.sin()], -1), seq=torch.tensor(seq), ctx=torch.tensor(pos) + 1,
                   run_start=torch.tensor([0] + list(np.cumsum(runs))), seq_start=torch.tensor(self.lens))
        for i, r in enumerate(runs):
            self.lens[i] += r
        held = self.buffers.setdefault(tuple(runs), {k: torch.empty(v.shape, dtype=v.dtype if v.is_floating_point() else torch.int32, device=DEV) for k, v in new.items()}
                                       | dict(q=torch.empty(T, nh * hd, dtype=self.dtype, device=DEV), out=torch.empty(T, nh * hd, dtype=self.dtype, device=DEV),
                                              k=torch.empty(T, nkv * hd, dtype=self.dtype, device=DEV), v=torch.empty(T, nkv * hd, dtype=self.dtype, device=DEV)))
        for k, v in new.items():
            held[k].copy_(v)
        return held

    def step(self, b, runs, scratch=None):
        nh, nkv, hd = self.size
        self.ops.rope_cache4(b["qkv"], nh, nkv, hd, self.cache, b["slots"], cos_sin=b["cos_sin"], q_out=b["q"])
        if max(runs) == 1:
            self.ops.attention_decode4(b["q"], b["out"], self.cache, self.tables.view(-1), self.stride, b["seq"], b["ctx"], nh, nkv, hd, hd ** -0.5, self.room, scratch=scratch)
        else:
            self.ops.attention_prefill4(b["q"], b["out"], self.cache, self.tables.view(-1), self.stride, b["run_start"], b["seq_start"], len(runs), max(runs), nh, nkv, hd,
                                        hd ** -0.5, max_context=self.room, scratch=scratch)
        self.ops.cache4_rows(self.cache, b["slots"], b["k"], b["v"])

    def check(self, b):
        """The outputs against 64 bits over what the cache holds now; what was read back against the same."""
        nh, nkv, hd = self.size
        held = plain.parts(self.cache, nkv, hd)
        t = torch.arange(self.room, device=DEV)
        slots = [(self.tables[i].long()[t // self.page] * self.page + t % self.page) for i in range(len(self.lens))]
        rows = b["q"].shape[0]
        some = sorted(set(range(0, rows, 5)) | {rows - 1})
        want, tol = plain.attend(b["q"][some].double().view(-1, nh, hd), held, [slots[int(b["seq"][r])] for r in some], [(0, int(b["ctx"][r])) for r in some], nh, nkv, hd ** -0.5, self.dtype)
        near(b["out"][some], want, tol)
        at = b["slots"].long()
        kc, ks, kl, vc, vs, vl = held
        assert torch.equal(b["k"], (kl + ks * kc)[at].flatten(1).to(self.dtype)) and torch.equal(b["v"], (vl + vs * vc)[at].flatten(1).to(self.dtype))
        # and the cache holds what was written: the rotated keys' range, an entry off by a step at most
        x = b["qkv"].double().view(rows, -1, hd)[:, nh + nkv:]
        assert bool(((b["v"].double().view(rows, nkv, hd) - x).abs() <= vs[at] * 0.6 + 2.0 ** -8 * x.abs().amax(-1, keepdim=True)).all())


@pytest.mark.parametrize("nh, nkv, hd, page, dtype", ((8, 2, 64, 16, BF), (4, 1, 128, 48, BF), (4, 4, 32, 32, F32)))
def test_steps_as_they_are_served(ops, nh, nkv, hd, page, dtype):
    """Prompts in portions, then tokens: every step's rows attend over what the steps before have left in the pages."""
    w = Served(ops, nh, nkv, hd, page, 400, 3, dtype, 21)
    for runs in ((40, 1, 130), (1, 200, 3), (7, 2, 1), (1, 1, 1), (1, 1, 1), (20, 1, 1)):
        b = w.inputs(runs)
        w.step(b, runs)
        w.check(b)


@pytest.mark.parametrize("how", ("graph", "program"))
@pytest.mark.parametrize("runs, before, room", (((1, 1, 1), (290, 3, 90), 700), ((1,), (3000,), 4000), ((9, 1, 64), (30, 300, 0), 700)))
def test_steps_captured_and_replayed(ops, how, runs, before, room):
    """A captured (or recorded) step replayed with other rows, other lengths and other pages' contents, eager steps in between: every replay
    gives what the eager step gives, bit for bit."""
    nh, nkv, hd, page = 8, 2, 64, 16
    w = Served(ops, nh, nkv, hd, page, room, len(runs), BF, 22)
    w.lens = list(before)
    w.cache.zero_()
    T = sum(runs)
    need = (ops.attention_decode4_scratch(T, nh, nkv, hd, room) if max(runs) == 1
            else ops.attention_prefill4_scratch(T, nh, nkv, hd, room, max(runs), len(runs)))
    scratch = torch.empty(max(need, 1), dtype=F32, device=DEV)
    b = w.inputs(runs)
    w.step(b, runs, scratch)
    torch.cuda.synchronize()
    if how == "graph":
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            w.step(b, runs, scratch)
        again = graph.replay
    else:
        program = ops.StepProgram()
        with ops.recording(program):
            w.step(b, runs, scratch)
        assert len(program) == 3
        again = program.run
    for _ in range(4):
        b = w.inputs(runs)
        for x in ("q", "out", "k", "v"):
            b[x].zero_()
        again()
        torch.cuda.synchronize()
        w.check(b)
        got = {x: b[x].clone() for x in ("q", "out", "k", "v")}
        w.step(b, runs)
        torch.cuda.synchronize()
        assert all(torch.equal(b[x], got[x]) for x in got)


def test_two_graphs_with_one_scratch(ops):
    """Two captured steps of different sizes share a scratch buffer; replayed in turn on one stream, each is right every time."""
    nh, nkv, hd, page = 8, 1, 64, 16
    need = max(ops.attention_decode4_scratch(r, nh, nkv, hd, 5000) for r in (1, 2))
    assert need > 0
    scratch, stream, work = torch.empty(need, dtype=F32, device=DEV), torch.cuda.Stream(), []
    for r, before in ((1, (4000,)), (2, (3000, 1200))):
        w = Served(ops, nh, nkv, hd, page, 5000, r, BF, 30 + r)
        w.lens, runs = list(before), (1,) * r
        w.cache.zero_()
        b = w.inputs(runs)
        w.step(b, runs, scratch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            w.step(b, runs, scratch)
        work.append((w, runs, graph))
    for _ in range(3):
        held = [w.inputs(runs) for w, runs, _ in work]
        scratch.fill_(float("nan"))
        for _, _, graph in work + work[:1]:
            graph.replay()
        torch.cuda.synchronize()
        for (w, _, _), b in zip(work, held):
            w.check(b)


def test_work_goes_to_the_current_stream(ops):
    """On a side stream behind a long copy chain: what is read there is what the stream's earlier work has written."""
    w = Served(ops, 8, 2, 64, 16, 300, 2, BF, 41)
    w.lens = [100, 250]
    w.cache.zero_()
    runs = (1, 1)
    b = w.inputs(runs)
    rows = b["qkv"].clone()
    torch.cuda.synchronize()
    stream, big = torch.cuda.Stream(), torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    with torch.cuda.stream(stream):
        b["qkv"].zero_()
        for _ in range(4):
            big.copy_(big.flip(0))
        b["qkv"].copy_(rows)
        w.step(b, runs)
    stream.synchronize()
    w.check(b)


@pytest.mark.parametrize("nh, nkv, hd, rows, dtype", ((4, 4, 64, 300, BF), (8, 4, 32, 300, F32), (12, 12, 128, 90, BF), (2, 2, 256, 140, BF), (2, 2, 256, 140, F32)))
def test_many_rows_of_short_contexts(ops, nh, nkv, hd, rows, dtype):
    gen = torch.Generator().manual_seed(rows + hd)
    lengths = torch.randint(0, 75, (rows,), generator=gen).tolist()
    s = Sequences(ops, nh, nkv, hd, 16, lengths, gen, dtype)
    q, out = queries(rows, nh * hd, dtype, gen), torch.full((rows, nh * hd), 9.0, dtype=dtype, device=DEV)
    for window in (0, 33):
        ops.attention_decode4(q, out, s.cache, s.dev_tables, s.stride, ints(range(rows)), ints(lengths), nh, nkv, hd, hd ** -0.5, 75, window=window)
        some = list(range(0, rows, 3))
        want, tol = s.expect(q[some], some, [(max(0, lengths[r] - window) if window else 0, lengths[r]) for r in some], hd ** -0.5)
        near(out[some], want, tol)


@pytest.mark.parametrize("nh, nkv, hd, seqs, dtype", ((32, 4, 64, 40, BF), (8, 8, 128, 60, BF), (16, 2, 32, 70, F32), (16, 2, 32, 70, BF), (8, 1, 256, 40, BF)))
def test_many_short_prompts(ops, nh, nkv, hd, seqs, dtype):
    gen = torch.Generator().manual_seed(seqs + hd)
    runs = torch.randint(1, 70, (seqs,), generator=gen).tolist()
    starts = [0 if i % 3 else i for i in range(seqs)]
    s = Sequences(ops, nh, nkv, hd, 16, [r + p for r, p in zip(runs, starts)], gen, dtype)
    first = np.concatenate([[0], np.cumsum(runs)])
    T = int(first[-1])
    q, out = queries(T, nh * hd, dtype, gen), torch.full((T, nh * hd), 9.0, dtype=dtype, device=DEV)
    ops.attention_prefill4(q, out, s.cache, s.dev_tables, s.stride, ints(first), ints(starts), seqs, max(runs), nh, nkv, hd, hd ** -0.5, max_context=140)
    seq, pos = [i for i, r in enumerate(runs) for _ in range(r)], [p + j for r, p in zip(runs, starts) for j in range(r)]
    some = list(range(0, T, 31)) + [T - 1]
    want, tol = s.expect(q[some], [seq[i] for i in some], [(0, pos[i] + 1) for i in some], hd ** -0.5)
    near(out[some], want, tol)


@pytest.mark.parametrize("dtype", (BF, F32))
@pytest.mark.parametrize("nh, nkv, hd, page", ((64, 1, 64, 16), (33, 1, 32, 16), (40, 2, 128, 1008), (20, 1, 256, 16)))
def test_many_heads_of_one_kv_head(ops, nh, nkv, hd, page, dtype):
    gen = torch.Generator().manual_seed(nh)
    lengths = (5, 1100, 64, 333)
    s = Sequences(ops, nh, nkv, hd, page, lengths, gen, dtype)
    q, out = queries(4, nh * hd, dtype, gen), torch.empty(4, nh * hd, dtype=dtype, device=DEV)
    for window in (0, 50):
        ops.attention_decode4(q, out, s.cache, s.dev_tables, s.stride, ints(range(4)), ints(lengths), nh, nkv, hd, hd ** -0.5, max(lengths), window=window)
        want, tol = s.expect(q, range(4), [(max(0, n - window) if window else 0, n) for n in lengths], hd ** -0.5)
        near(out, want, tol)


def test_nothing_to_do(ops):
    """No rows, no sequences, bounds of 0, runs that name rows and contexts that do not exist."""
    nh, nkv, hd = 4, 2, 64
    gen = torch.Generator().manual_seed(3)
    s = Sequences(ops, nh, nkv, hd, 16, (40, 40), gen, BF)
    q = queries(4, nh * hd, BF, gen)
    nine = lambda: torch.full((4, nh * hd), 9.0, dtype=BF, device=DEV)
    decode = lambda out, bound, **k: ops.attention_decode4(q, out, s.cache, s.dev_tables, s.stride, ints([0, 1, 0, 1]), ints([40, 3, 0, -2 ** 31]), nh, nkv, hd, 0.1, bound, **k)
    prefill = lambda out, runs, starts, n, most, **k: ops.attention_prefill4(q, out, s.cache, s.dev_tables, s.stride, ints(runs), ints(starts), n, most, nh, nkv, hd, 0.1, **k)
    for call in (lambda out: decode(out, 40, rows=0), lambda out: prefill(out, [0], [], 0, 4), lambda out: prefill(out, [0, 2, 4], [3, 3], 2, 0), lambda out: prefill(out, [2, 2, 2], [3, 3], 2, 4),
                 lambda out: prefill(out, [4, 1, 0], [3, 3], 2, 4), lambda out: prefill(out, [7, 9, 2 ** 31 - 1], [3, 3], 2, 4)):
        out = nine()
        call(out)
        assert bool((out == 9).all())
    out = nine()
    decode(out, 0)
    assert not out.any()
    out = nine()
    prefill(out, [0, 2, 4], [-2 ** 31, -2], 2, 2)
    assert not out.any()
    out = nine()
    prefill(out, [0, 1, 2 ** 31 - 1], [2 ** 31 - 1, 36], 2, 4, max_context=39)      # (rows 1 to 3: positions 36 to 38; row 0 sees what the bound allows)
    want, tol = s.expect(q, [0, 1, 1, 1], [(0, 39), (0, 37), (0, 38), (0, 39)], 0.1)
    near(out, want, tol)


@pytest.mark.parametrize("nh, nkv, hd, runs, starts, window, dtype", (
    (32, 4, 64, (1100,), (0,), 0, BF), (32, 4, 64, (700, 555), (30, 0), 200, BF), (16, 2, 32, (1500, 600), (0, 77), 0, BF), (8, 8, 128, (900, 1000), (200, 0), 0, BF),
    (32, 4, 64, (64,), (8000,), 0, BF), (8, 2, 128, (130, 99), (8000, 5000), 0, BF), (8, 2, 128, (300, 299), (3000, 2500), 2500, BF), (32, 4, 32, (90,), (7000,), 0, BF),
    (32, 4, 64, (500, 333), (200, 0), 0, F32), (16, 2, 256, (600, 300), (0, 100), 0, BF)))
def test_long_runs(ops, nh, nkv, hd, runs, starts, window, dtype):
    gen = torch.Generator().manual_seed(sum(runs) + hd)
    s = Sequences(ops, nh, nkv, hd, 16, [r + p for r, p in zip(runs, starts)], gen, dtype)
    first = np.concatenate([[0], np.cumsum(runs)])
    T = int(first[-1])
    q, out = queries(T, nh * hd, dtype, gen), torch.full((T, nh * hd), 9.0, dtype=dtype, device=DEV)
    args = (q, out, s.cache, s.dev_tables, s.stride, ints(first), ints(starts), len(runs), max(runs), nh, nkv, hd, hd ** -0.5)
    ops.attention_prefill4(*args, window=window)
    seq, pos = [i for i, r in enumerate(runs) for _ in range(r)], [p + j for r, p in zip(runs, starts) for j in range(r)]
    some = sorted(set(range(0, T, T // 40)) | {0, 1, 2, 3, 4, T - 2, T - 1})
    want, tol = s.expect(q[some], [seq[i] for i in some], [(max(0, pos[i] + 1 - window) if window else 0, pos[i] + 1) for i in some], hd ** -0.5)
    near(out[some], want, tol)
    assert not bool(out.isnan().any())
    again = out.clone()
    ops.attention_prefill4(*args, window=window)
    assert torch.equal(again, out)


@pytest.mark.parametrize("nh, hd, rows", ((1, 32, 400), (1, 64, 400), (1, 128, 400), (1, 256, 400), (32, 64, 1600), (32, 128, 1600)))
@pytest.mark.parametrize("dtype", (BF, F32))
def test_scores_of_far_off_entries_stay_exact(ops, dtype, nh, hd, rows):
    """Two tokens whose scores are nearly alike, of keys and queries around 20: the value of one is 1 everywhere and of the other -1 (step 0,
    nothing of p is rounded), so that the output is tanh of half the scores' difference and its error half the scores'.

    What the scores may be off by, root of the mean square: a sum over hd entries comes about in hd / 32 matrix instructions, the j-th of them
    at no more than j 32 / hd of (16 + 8) sum|q|, and is multiplied with step * scale; each rounds by up to u = 2^-24 of what it holds, evenly (so
    u / sqrt 3).  Two roundings more at up to two thirds of that for the terms beside it (16 step and low, times sum q).  Twice all this, for
    instructions that cut where others round; two tokens; half of it in the output, which is rounded itself (at most half a unit in its last place)."""
    gen = torch.Generator().manual_seed(hd + nh)
    x = torch.randn(2, 3 * hd, generator=gen) * 20 + 20
    x[0, 2 * hd:], x[1, 2 * hd:] = 1, -1
    cache = torch.zeros(ops.cache4_shape(1, 1, hd, 16), dtype=torch.uint8, device=DEV)
    ops.rope_cache4(x.to(dtype).to(DEV), 1, 1, hd, cache, ints(range(2)))
    kc, ks, kl, _, vs, vl = plain.parts(cache, 1, hd)
    assert not vs[:2].any() and vl[0, 0] == 1 and vl[1, 0] == -1
    k, scale = (kl + ks * kc)[:2, 0], hd ** -0.5
    q = torch.randn(rows * nh, hd, generator=gen).double().to(DEV) * 20 + 20
    between = k[0] - k[1]
    q = (q - (q @ between / (between @ between)).view(-1, 1) * between).to(dtype)
    s = q.double() @ k.T * scale
    want = torch.tanh((s[:, 0] - s[:, 1]) / 2)
    out = torch.empty(rows, nh * hd, dtype=dtype, device=DEV)
    ops.attention_decode4(q.view(rows, -1), out, cache, ints([0]), 1, ints([0] * rows), ints([2] * rows), nh, 1, hd, scale, 2)
    off = out.view(rows * nh, hd).double() - want.view(-1, 1)
    u, n = 2.0 ** -24, hd // 32
    held = 24 * q.double().abs().sum(1) * ks[:2].max() * scale
    scores = 2 * (2 * (sum((j / n) ** 2 for j in range(1, n + 1)) + 2 * (2 / 3) ** 2)) ** 0.5 * u / 3 ** 0.5 * held
    tol = scores / 2 + torch.finfo(dtype).eps / 2 * want.abs()
    rms = lambda v: float(v.square().mean().sqrt())
    assert rms(off) <= rms(tol), (rms(off), rms(tol))


@pytest.mark.parametrize("window", (20, 0))
def test_the_longest_context_that_slots_can_number(ops, window):
    """A context of 2^31 - 16 tokens, all of whose pages but the last two are none: the tokens at its end are seen."""
    nh, nkv, hd, page, n = 2, 1, 32, 16, 2 ** 31 - 16
    gen = torch.Generator().manual_seed(51)
    cache = filled(ops, 5, nkv, hd, page, gen, list(range(80)))
    tables = torch.full((n // page,), -1, dtype=torch.int32, device=DEV)
    tables[-2:] = ints([3, 1])
    q, out = queries(1, nh * hd, BF, gen), torch.full((1, nh * hd), 9.0, dtype=BF, device=DEV)
    slots = torch.cat([torch.arange(48, 64, device=DEV), torch.arange(16, 32, device=DEV)])
    want, tol = plain.attend(q.double().view(1, nh, hd), plain.parts(cache, nkv, hd), [slots], [(32 - window if window else 0, 32)], nh, nkv, 0.2, BF)
    ops.attention_decode4(q, out, cache, tables, n // page, ints([0]), ints([n]), nh, nkv, hd, 0.2, n, window=window)
    near(out, want, tol)
    out.fill_(9.0)
    ops.attention_prefill4(q, out, cache, tables, n // page, ints([0, 1]), ints([n - 1]), 1, 1, nh, nkv, hd, 0.2, max_context=n, window=window)
    near(out, want, tol)


def test_runs_in_front_of_their_sequence_see_nothing(ops):
    """Rows at positions below 0, down to the smallest, under windows of any size: zeros; the run's rows from position 0 on as ever."""
    nh, nkv, hd = 4, 2, 64
    gen = torch.Generator().manual_seed(52)
    s = Sequences(ops, nh, nkv, hd, 16, (40, 40), gen, BF)
    q = queries(6, nh * hd, BF, gen)
    for window in (0, 1, 2 ** 31 - 1):
        out = torch.full((6, nh * hd), 9.0, dtype=BF, device=DEV)
        ops.attention_prefill4(q, out, s.cache, s.dev_tables, s.stride, ints([0, 2, 6]), ints([-2 ** 31, -2]), 2, 4, nh, nkv, hd, 0.1, window=window)
        want, tol = s.expect(q, [-1, -1, 1, 1, 1, 1], [(0, 0)] * 4 + [(0, 1), (1, 2) if window == 1 else (0, 2)], 0.1)
        near(out, want, tol)


@pytest.mark.parametrize("dtype", (BF, F32))
def test_how_far_a_token_is_off_with_entries_far_from_zero(ops, dtype):
    """Half a kept step from low on (a nearest code; the highest entry, which step's rounding moves by up to 15 * 2^-8 of a step, is no further
    off).  Below low, which float rows have where it was rounded up: low - x <= low - min x <= 2^-8 |min x|.  Reading back in 32 bits rounds once."""
    gen = torch.Generator().manual_seed(53)
    nkv, hd, T = 2, 64, 400
    far = torch.where(torch.rand(T, 1, generator=gen) < 0.5, -1.0, 1.0) * torch.exp(torch.rand(T, 1, generator=gen) * 9)
    x = (torch.randn(T, 3 * nkv * hd, generator=gen) + far).to(dtype).to(DEV)
    cache = torch.zeros(ops.cache4_shape(25, nkv, hd, 16), dtype=torch.uint8, device=DEV)
    ops.rope_cache4(x, nkv, nkv, hd, cache, ints(range(T)))
    k, v = (torch.empty(T, nkv * hd, device=DEV) for _ in range(2))
    ops.cache4_rows(cache, ints(range(T)), k, v)
    _, ks, kl, _, vs, vl = plain.parts(cache, nkv, hd)
    below = False
    for got, want, step, low in ((k, x[:, nkv * hd:2 * nkv * hd], ks, kl), (v, x[:, 2 * nkv * hd:], vs, vl)):
        a, b = got.double().view(T, nkv, hd), want.double().view(T, nkv, hd)
        off, least = (a - b).abs(), b.amin(-1, keepdim=True).abs()
        once = 2.0 ** -24 * a.abs()
        assert bool((off <= torch.where(b < low[:T], 2.0 ** -8 * least, step[:T] / 2) + once).all())
        below = below or bool((off > 2 * step[:T] + once).any())
    assert below == (dtype == F32)


@pytest.mark.parametrize("nh, nkv, hd, rows, dtype", ((4, 4, 32, 300, BF), (12, 12, 128, 90, F32)))
def test_many_rows_of_short_contexts_in_workgroups_of_two_waves(ops, nh, nkv, hd, rows, dtype):
    """1,024 workgroups and more for contexts of up to 75 tokens: two waves each, of 32 entries in bfloat16 and of 128 in float32."""
    gen = torch.Generator().manual_seed(rows + hd)
    lengths = torch.randint(0, 76, (rows,), generator=gen).tolist()
    s = Sequences(ops, nh, nkv, hd, 32, lengths, gen, dtype)
    q, out = queries(rows, nh * hd, dtype, gen), torch.full((rows, nh * hd), 9.0, dtype=dtype, device=DEV)
    for window in (0, 33):
        ops.attention_decode4(q, out, s.cache, s.dev_tables, s.stride, ints(range(rows)), ints(lengths), nh, nkv, hd, hd ** -0.5, 75, window=window)
        some = list(range(0, rows, 3))
        want, tol = s.expect(q[some], some, [(max(0, lengths[r] - window) if window else 0, lengths[r]) for r in some], hd ** -0.5)
        near(out[some], want, tol)


@pytest.mark.parametrize("nh, nkv, hd, rows, ctx, bound", ((8, 2, 64, 40, 200, 200), (8, 2, 128, 40, 300, 300), (4, 1, 32, 40, 700, 700), (2, 1, 256, 30, 100, 100), (8, 2, 64, 3, 3000, 3000),
                                                           (40, 2, 64, 60, 90, 90), (64, 2, 128, 6, 900, 30000), (40, 1, 32, 1100, 40, 40), (36, 1, 64, 1100, 40, 40), (34, 1, 128, 1100, 40, 40),
                                                           (40, 2, 32, 800, 200, 2000), (40, 2, 64, 800, 200, 2000), (40, 2, 128, 800, 200, 2000)))
def test_single_tokens_keep_16_bits_of_their_weights(ops, nh, nkv, hd, rows, ctx, bound):
    """Values around 0, whose weighted sums are small beside what they are sums of: the tolerance of 32-bit rows (sums over 16 + c), the output's
    rounding, and of p step, kept in two bfloat16 numbers, 2^-8 of 2^-8, times c - 8, which is at most 8."""
    gen = torch.Generator().manual_seed(hd + rows)
    n = -(-ctx // 16)
    cache = torch.zeros(ops.cache4_shape(n, nkv, hd, 16), dtype=torch.uint8, device=DEV)
    ops.rope_cache4(torch.randn(ctx, 3 * nkv * hd, generator=gen).to(BF).to(DEV), nkv, nkv, hd, cache, ints(range(ctx)))
    q, out = queries(rows, nh * hd, BF, gen), torch.empty(rows, nh * hd, dtype=BF, device=DEV)
    lens = [max(2, ctx - 7 * r % ctx) for r in range(rows)]
    ops.attention_decode4(q, out, cache, ints(range(n)), n, ints([0] * rows), ints(lens), nh, nkv, hd, hd ** -0.5, bound)
    held = plain.parts(cache, nkv, hd)
    some = list(range(0, rows, max(1, rows // 25)))
    want, tol = plain.attend(q[some].double().view(-1, nh, hd), held, [torch.arange(ctx, device=DEV)] * len(some), [(0, lens[r]) for r in some], nh, nkv, hd ** -0.5, F32)
    near(out[some], want, tol + 2.0 ** -8 * want.abs() + 2.0 ** -16 * 8 * held[4].max())


@pytest.mark.parametrize("nh, nkv, hd", ((8, 4, 32), (8, 4, 64), (8, 4, 128), (8, 4, 256)))
def test_many_runs_of_one_or_two_tokens(ops, nh, nkv, hd):
    """1,200 workgroups of one tile of rows for contexts of up to 62 tokens: two waves each."""
    gen = torch.Generator().manual_seed(hd)
    seqs = 300
    runs, starts = torch.randint(0, 3, (seqs,), generator=gen).tolist(), torch.randint(0, 60, (seqs,), generator=gen).tolist()
    s = Sequences(ops, nh, nkv, hd, 16, [r + p for r, p in zip(runs, starts)], gen, BF)
    first = np.concatenate([[0], np.cumsum(runs)])
    T = int(first[-1])
    q, out = queries(T, nh * hd, BF, gen), torch.full((T, nh * hd), 9.0, dtype=BF, device=DEV)
    ops.attention_prefill4(q, out, s.cache, s.dev_tables, s.stride, ints(first), ints(starts), seqs, 2, nh, nkv, hd, hd ** -0.5, max_context=62)
    seq, pos = [i for i, r in enumerate(runs) for _ in range(r)], [p + j for r, p in zip(runs, starts) for j in range(r)]
    some = list(range(0, T, 5)) + [T - 1]
    want, tol = s.expect(q[some], [seq[i] for i in some], [(0, pos[i] + 1) for i in some], hd ** -0.5)
    near(out[some], want, tol)
