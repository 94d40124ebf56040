"""The paged cache's attention where held numbers leave the usual range:
infinities and NaN, scales far apart, rows that see nothing, and what a call
keeps, against the definition in 64 bits."""
import math

import numpy as np
import pytest

from tests.test_gpu_cache import CHUNKS, EIGHT, FEW, PAIRS, TOKENS, dt, held_rows, make_batch, make_cache, queries, scale_of

pytestmark = pytest.mark.gpu

EIGHT_PAIRS = [p for p in PAIRS if p[0] in EIGHT]


def place(cache, batch, s, position):
    """(page, row) of a position of sequence s."""
    return int(batch.page_table[s, position // cache.page_rows]), position % cache.page_rows


def definition(q, k, v, scale, causal, first, sizes=None):
    """(out, lse, tolerance of out, of lse) of one sequence's rows, in 64 bits,
    with the tolerances of tests/test_gpu_cache.py's `expected`, all rows at
    once.  Values that are no numbers count where a row sees them only.

    `sizes` are the scales [length, heads] of 8-bit values, for rows whose
    probabilities span more than an fp16 does: P times its value's scale is one
    fp16, where the row's largest stands at 2^6 at least and a half step is 2^-25,
    so each value v held as v / size is off by up to 2^-31 max_j(p_j size_j) /
    size of itself."""
    import torch
    n, heads, width = q.shape
    length, group = k.shape[0], heads // k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).tiny
    if length == 0:
        zeros = torch.zeros(n, heads, width, dtype=torch.float64, device=q.device)
        lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
        return zeros, lse, zeros + tiny, torch.zeros_like(lse)
    q64 = q.double().transpose(0, 1)                                               # [heads, n, width]
    k, v = (x.repeat_interleave(group, 1).permute(1, 2, 0) for x in (k, v))        # [heads, width, length]
    seen = torch.arange(length, device=q.device)[None] <= first + torch.arange(n, device=q.device)[:, None]
    if not causal:
        seen = torch.ones_like(seen)
    some = seen.any(1)
    s = ((q64 @ k) * scale).masked_fill(~seen, -math.inf)
    big = ((q64.abs() @ k.abs()) * abs(scale)).masked_fill(~seen, 0).amax(2)       # [heads, n]
    lse = torch.logsumexp(s, 2)
    p = torch.exp(s - torch.where(some, lse, torch.zeros_like(lse))[..., None])
    finite = torch.where(torch.isfinite(v), v, torch.zeros_like(v)).transpose(1, 2)
    out, a = p @ finite, p @ finite.abs()
    of = seen.double()[None].expand(heads, -1, -1)
    held = [(of @ x.double().transpose(1, 2)) > 0 for x in (torch.isnan(v), torch.isposinf(v), torch.isneginf(v))]
    out = torch.where(held[1], out + math.inf, out)
    out = torch.where(held[2], out - math.inf, out)
    out = torch.where(held[0], torch.full_like(out, math.nan), out)
    each = (width + 3) * 2.0 ** -24 * big + 2.0 ** -18
    count = seen.sum(1).double()
    tol = u * out.abs() + (u + 2 * each + count * 2.0 ** -24)[..., None] * a + tiny
    if sizes is not None:
        sizes = sizes.repeat_interleave(group, 1).T                                # [heads, length]
        weight = (p * sizes[:, None]).amax(2, keepdim=True)
        tol = tol + 2.0 ** -31 * weight * (of @ (finite.abs() / sizes[..., None]))
    lse_tol = each + count * 2.0 ** -24 + 2.0 ** -23 * lse.abs()
    return out.transpose(0, 1), lse.T, tol.transpose(0, 1), lse_tol.T


def check(cache, batch, starts, q, out, lse, scale, causal=True, spread=False):
    """The sequences' rows against the definition; a result that is above the
    type's largest, by its tolerance too, has to be an infinity.  `spread`: the
    probabilities span more than an fp16 does."""
    import torch
    got, got_lse = out.double(), lse.double()
    for s in range(len(starts) - 1):
        a, b = int(starts[s]), int(starts[s + 1])
        if a == b:
            continue
        length = int(batch.lengths[s])
        k, v = held_rows(cache, batch.page_table[s], length)
        sizes = None
        if spread and length:
            pages = batch.page_table[s, :-(-length // cache.page_rows)].long()
            sizes = scale_of(cache.value_scales[pages]).transpose(1, 2).reshape(-1, cache.heads)[:length]
        o, l, tol, lse_tol = definition(q[a:b], k, v, scale, causal, length - (b - a), sizes)
        at, largest = (s, length, b - a), torch.finfo(q.dtype).max
        assert torch.equal(torch.isnan(got[a:b]), torch.isnan(o)), at
        infinite = torch.isinf(o) | (o.abs() - tol > largest)
        assert torch.equal(got[a:b][infinite], torch.sign(o[infinite]) * math.inf), at
        fine = torch.isfinite(o) & (o.abs() + tol < largest)
        off = (got[a:b] - o).abs()
        assert bool((off <= tol)[fine].all()), (*at, float((off / tol)[fine].max()))
        assert torch.equal(torch.isnan(got_lse[a:b]), torch.isnan(l)), at
        assert torch.equal(torch.isneginf(got_lse[a:b]), torch.isneginf(l)), at
        fine = torch.isfinite(l)
        off = (got_lse[a:b] - l).abs()
        assert bool((off <= lse_tol)[fine].all()), (*at, float((off / lse_tol)[fine].max()))


def pages_of(lengths, page_rows):
    return sum(-(-n // page_rows) for n in lengths) + 2


# The rows a call brings, and a table's columns: what a table has places for
# decides which kernel takes a call, and whether items are cut.
SHAPES = [(TOKENS, None), (FEW, None), (FEW, 600), (CHUNKS, None), (CHUNKS, 9600)]


@pytest.mark.parametrize("storage,dtype", EIGHT_PAIRS)
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_a_value_row_that_was_no_number_makes_those_that_see_it_none(storage, dtype, width, rows, columns):
    """Scale byte 255 of a value row reads as NaN, and so does what sees it."""
    lengths, new = rows
    pages = pages_of(lengths, 16)
    cache = make_cache(storage, pages, 2, 16, width, 511)
    batch, starts = make_batch(lengths, new, 16, pages, 512, columns=columns)
    for s, n in enumerate(lengths):
        if n > 2:
            page, row = place(cache, batch, s, n // 2)
            cache.value_scales[page, 0, row] = 255
    q = queries(int(starts[-1]), 4, width, dtype, 513)
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, width ** -0.5)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_an_infinity_among_the_values_stays_one(dtype, width, rows, columns):
    """A seen value of infinity makes its column infinite, not NaN, and no
    other column anything else."""
    lengths, new = rows
    pages = pages_of(lengths, 16)
    cache = make_cache(dtype, pages, 2, 16, width, 521)
    batch, starts = make_batch(lengths, new, 16, pages, 522, columns=columns)
    for s, n in enumerate(lengths):
        if n:
            page, row = place(cache, batch, s, n // 2)
            cache.values[page, 0, row, 5] = -math.inf
            cache.values[page, 1, row, 40] = math.inf
    q = queries(int(starts[-1]), 4, width, dtype, 523)
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, width ** -0.5)


@pytest.mark.parametrize("storage,dtype", PAIRS)
@pytest.mark.parametrize("columns", [None, 40, 9600])
def test_rows_that_see_nothing_beside_values_that_are_no_numbers(storage, dtype, columns):
    """More new rows than a length holds: the first rows see no key and get
    zeros, whatever the values hold that other rows of their tile see."""
    import torch
    for lengths, new in (([3, 1], [5, 7]), ([70, 300], [150, 310])):
        pages = pages_of(lengths, 16)
        cache = make_cache(storage, pages, 2, 16, 64, 501)
        batch, starts = make_batch(lengths, new, 16, pages, 502, columns=columns)
        for s, n in enumerate(lengths):
            for position in (0, n - 1):
                page, row = place(cache, batch, s, position)
                if storage in EIGHT:
                    cache.value_scales[page, :, row] = 255
                else:
                    cache.values[page, :, row, 3] = math.nan
                    cache.values[page, :, row, 60] = math.inf
        q = queries(int(starts[-1]), 4, 64, dtype, 503)
        out, lse = cache.attend(batch, q, return_lse=True)
        for s, n in enumerate(lengths):
            a = int(starts[s])
            b = a + new[s] - n
            assert bool((out[a:b] == 0).all()) and bool(torch.isneginf(lse[a:b]).all()), s
        check(cache, batch, starts, q, out, lse, 0.125)
        cache.check()


@pytest.mark.parametrize("storage,dtype", EIGHT_PAIRS)
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("jump", [24, 40, 80])
@pytest.mark.parametrize("rows,columns", [(FEW, None), (FEW, 600), (CHUNKS, None), (CHUNKS, 9600)])
def test_a_large_value_behind_a_row_cannot_change_it(storage, dtype, width, jump, rows, columns):
    """The last new row's values are 2^jump times the others."""
    lengths, new = rows
    pages = pages_of(lengths, 16)
    cache = make_cache(storage, pages, 2, 16, width, 531)
    batch, starts = make_batch(lengths, new, 16, pages, 532, columns=columns)
    q = queries(int(starts[-1]), 4, width, dtype, 533)
    for s, n in enumerate(lengths):
        if new[s] > 1:
            page, row = place(cache, batch, s, n - 1)
            cache.value_scales[page, :, row] += jump
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, width ** -0.5)


@pytest.mark.parametrize("storage,dtype", EIGHT_PAIRS)
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("jump", [30, 60, 90])
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_a_large_value_of_little_weight(storage, dtype, width, jump, rows, columns):
    """A seen key whose probability is about 2^-60 of the others' and whose
    value is 2^jump times theirs."""
    lengths, new = rows
    pages = pages_of(lengths, 16)
    cache = make_cache(storage, pages, 2, 16, width, 541)
    batch, starts = make_batch(lengths, new, 16, pages, 542, columns=columns)
    q = queries(int(starts[-1]), 4, width, dtype, 543).abs()
    for s, n in enumerate(lengths):
        if n > 3:
            for position in (1, n // 2):
                page, row = place(cache, batch, s, position)
                # -100 a column: scores of -60 in log2 at |q| of 0.8 each
                cache.keys[page, :, row] = -100 if storage == "int8" else -96.0
                size = 60 * math.log(2) / (width ** -0.5 * 0.8 * width * 100)
                cache.key_scales[page, :, row] = 127 + round(math.log2(size))
                cache.value_scales[page, :, row] += jump
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, width ** -0.5, spread=True)


@pytest.mark.parametrize("storage,dtype", EIGHT_PAIRS)
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_value_scales_over_their_whole_range(storage, dtype, width, rows, columns):
    """Every row's values at a scale of its own, from 2^-100 to 2^0, their
    largest first and last, and columns in which the large rows hold zeros."""
    import torch
    lengths, new = rows
    pages = pages_of(lengths, 16)
    cache = make_cache(storage, pages, 2, 16, width, 551)
    batch, starts = make_batch(lengths, new, 16, pages, 552, columns=columns)
    g = torch.Generator("cuda").manual_seed(553)
    cache.value_scales.copy_(torch.randint(27, 128, cache.value_scales.shape, generator=g, device="cuda").to(torch.uint8))
    large = cache.value_scales > 60
    values = cache.values.view(torch.uint8)
    values[..., 7] = torch.where(large, torch.zeros_like(values[..., 7]), values[..., 7])
    q = queries(int(starts[-1]), 4, width, dtype, 554)
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, width ** -0.5)


@pytest.mark.parametrize("storage,dtype", EIGHT_PAIRS)
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("scales,size", [((137, 147), 2.0 ** -16), ((95, 100), 2.0 ** 14), ((90, 150), 2.0 ** -16),
                                         ((90, 150), 2.0 ** -7), ((1, 20), 2.0 ** 15)])
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_key_scales_beyond_the_queries_type(storage, dtype, width, scales, size, rows, columns):
    """Keys whose elements are above 65504 or below fp16's smallest step, under
    queries that make ordinary scores of them."""
    import torch
    lengths, new = rows
    pages = pages_of(lengths, 16)
    cache = make_cache(storage, pages, 2, 16, width, 561)
    batch, starts = make_batch(lengths, new, 16, pages, 562, columns=columns)
    g = torch.Generator("cuda").manual_seed(563)
    cache.key_scales.copy_(torch.randint(scales[0], scales[1] + 1, cache.key_scales.shape, generator=g, device="cuda").to(torch.uint8))
    q = queries(int(starts[-1]), 4, width, "float32", 564) * size
    q = q.clamp(-65000, 65000).to(dt(dtype))
    for causal in (True, False):
        out, lse = cache.attend(batch, q, causal=causal, return_lse=True)
        check(cache, batch, starts, q, out, lse, width ** -0.5, causal, spread=True)


@pytest.mark.parametrize("storage", ["int8", "float8_e4m3fn"])
@pytest.mark.parametrize("low", [100, 110, 118])
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_tiny_queries_over_large_keys(storage, low, rows, columns):
    """bf16 queries of 2^-low over keys of 2^low: ordinary scores."""
    lengths, new = rows
    pages = pages_of(lengths, 16)
    cache = make_cache(storage, pages, 2, 16, 64, 571)
    batch, starts = make_batch(lengths, new, 16, pages, 572, columns=columns)
    cache.key_scales.fill_(120 + low)
    q = (queries(int(starts[-1]), 4, 64, "float32", 573) * 2.0 ** -low).to(dt("bfloat16"))
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, 0.125)


def test_a_batch_whose_starts_change_is_read_as_it_stands():
    """read without a number of rows after starts were updated in place, to
    more and to fewer."""
    import torch
    cache = make_cache("float16", 30, 2, 16, 64, 581)
    batch, _ = make_batch([40, 60], [5, 7], 16, 30, 582)
    held = [held_rows(cache, batch.page_table[s], n)[0] for s, n in enumerate((40, 60))]
    for new in ((5, 7), (30, 41), (2, 1), (0, 0), (0, 6)):
        batch.starts.copy_(torch.tensor([0, new[0], sum(new)], dtype=torch.int32))
        k, v = cache.read(batch)
        assert k.shape == v.shape == (sum(new), 2, 64) and batch.rows() == sum(new)
        want = torch.cat([held[s][len(held[s]) - n:] for s, n in enumerate(new)])
        assert torch.equal(k.double(), want)


@pytest.mark.parametrize("storage,dtype", [("float16", "float16"), ("int8", "bfloat16")])
@pytest.mark.parametrize("columns", [None, 600])
def test_starts_that_grow_past_the_bound_of_their_batch(storage, dtype, columns):
    """max_rows chooses kernels: results are the definition's all the same."""
    import torch
    from whispereacp_b200 import CacheBatch
    lengths, new = CHUNKS
    pages = pages_of(lengths, 16)
    cache = make_cache(storage, pages, 2, 16, 64, 585)
    made, starts = make_batch(lengths, new, 16, pages, 586, columns=columns)
    batch = CacheBatch(made.page_table, made.lengths, torch.zeros_like(made.starts))
    assert batch.max_rows == 0
    batch.starts.copy_(made.starts)
    q = queries(int(starts[-1]), 4, 64, dtype, 587)
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, 0.125)


def test_tensors_that_require_gradients_are_refused():
    """The operators have no gradient; results that silently lack one would
    train nothing.  Without grad mode they are taken as they are."""
    import torch
    from whispereacp_b200 import PagedCache
    cache = make_cache("float16", 8, 2, 16, 64, 591)
    batch, _ = make_batch([20], [2], 16, 8, 592)
    plain = queries(2, 2, 64, "float16", 593)
    leaf = plain.clone().requires_grad_()
    for call in (lambda x: cache.attend(batch, x), lambda x: cache.append(batch, x, plain),
                 lambda x: cache.append(batch, plain, x), lambda x: cache.attend(batch, plain, out=x),
                 lambda x: cache.read(batch, x, plain.clone()), lambda x: cache.read(batch, plain.clone(), x),
                 lambda x: cache.attend(batch, plain, lse=torch.zeros(2, 2, device="cuda", requires_grad=True))):
        with pytest.raises(ValueError, match="gradient"):
            call(leaf)
    pool = cache.keys.clone().requires_grad_()
    for pools in ((pool, cache.values), (cache.keys, pool)):
        with pytest.raises(ValueError, match="gradient"):
            PagedCache(*pools)
    with torch.no_grad():
        assert torch.equal(cache.attend(batch, leaf), cache.attend(batch, plain))
        cache.append(batch, leaf, leaf)
    assert torch.equal(cache.attend(batch, leaf.detach()), cache.attend(batch, plain))


def test_caches_of_a_thread_and_stream_share_a_workspace():
    """A decoder's layers follow one another on one stream: their caches need
    one workspace, not one each; a thread's ends with it."""
    import threading
    import torch
    caches = [make_cache("float16", 80, 2, 16, 64, 601 + i) for i in range(6)]
    batch, starts = make_batch([600, 500], [200, 1], 16, 80, 602, columns=9600)
    q = queries(201, 2, 64, "float16", 603)
    out, lse = torch.empty_like(q), torch.empty(201, 2, device="cuda")

    def step():
        for cache in caches:
            cache.attend(batch, q, out=out, lse=lse)

    caches[0].attend(batch, q, out=out, lse=lse)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    step()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before
    check(caches[-1], batch, starts, q, out, lse, 0.125)
    for _ in range(3):
        thread = threading.Thread(target=step)
        thread.start()
        thread.join()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("storage,dtype", EIGHT_PAIRS)
@pytest.mark.parametrize("byte", [2, 6, 20, 40, 80, 180, 230, 245])
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_value_scales_of_any_size(storage, dtype, byte, rows, columns):
    """All values tiny, or all large, beside a page of zeros as untouched memory
    holds them (scale byte 0)."""
    lengths, new = rows
    pages = pages_of(lengths, 16)
    cache = make_cache(storage, pages, 2, 16, 64, 621)
    batch, starts = make_batch(lengths, new, 16, pages, 622, columns=columns)
    cache.value_scales.fill_(byte)
    for s, n in enumerate(lengths):
        if n > 20:
            cache.value_scales[int(batch.page_table[s, 0])] = 0
    q = queries(int(starts[-1]), 4, 64, dtype, 623)
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, 0.125)


@pytest.mark.parametrize("storage", ["int8", "float8_e4m3fn"])
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("most", [100, 200])
def test_key_scales_of_every_sequence_s_own(storage, width, most):
    """Items of one tile of rows between items of two, over keys of a scale for
    each sequence: no tile takes another block's."""
    import torch
    new = [most if s % 3 else 300 for s in range(36)]
    lengths = [n + 97 * (s % 11) for s, n in enumerate(new)]
    pages = pages_of(lengths, 32)
    cache = make_cache(storage, pages, 6, 32, width, 631)
    batch, starts = make_batch(lengths, new, 32, pages, 632)
    byte = torch.empty(pages, dtype=torch.uint8, device="cuda")
    for s, n in enumerate(lengths):
        byte[batch.page_table[s, :-(-n // 32)].long()] = 104 + 5 * s % 23
    cache.key_scales.copy_(byte[:, None, None].expand_as(cache.key_scales))
    q = queries(int(starts[-1]), 6, width, "float16", 633)
    for causal in (True, False):
        out, lse = cache.attend(batch, q, causal=causal, return_lse=True)
        check(cache, batch, starts, q, out, lse, width ** -0.5, causal, spread=True)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("gap", [10.5, 16.47, 20.47])
@pytest.mark.parametrize("rows,columns", [(1, None), (5, None), (5, 600), (130, None), (130, 9600)])
def test_large_values_of_small_probabilities(dtype, gap, rows, columns):
    """One key of nearly all the probability and small values before 400 keys of
    2^-gap each and values of ten thousands, which are the result."""
    import torch
    width = 64
    cache = make_cache(dtype, 40, 2, 16, width, 641)
    batch, starts = make_batch([400 + rows], [rows], 16, 40, 642, columns=columns)
    cache.keys.zero_()
    cache.values.abs_().mul_(1e4)
    page, row = place(cache, batch, 0, 0)
    cache.keys[page, :, row] = gap * math.log(2) / (width * 0.125)
    cache.values[page, :, row] = 1e-3
    q = torch.ones(rows, 2, width, dtype=dt(dtype), device="cuda")
    out, lse = cache.attend(batch, q, return_lse=True)
    check(cache, batch, starts, q, out, lse, 0.125)
