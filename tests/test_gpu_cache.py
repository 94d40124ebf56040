"""The paged key/value cache (include/wsp_cache.h through the Python binding)
against its definition in 64 bits: rows written, quantised and read back, and
attention of single tokens and of chunks, where either can go wrong."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EIGHT = {"float8_e4m3fn": (448.0, 3), "int8": (127.0, None)}
PAIRS = [("float16", "float16"), ("bfloat16", "bfloat16"), ("int8", "float16"), ("int8", "bfloat16"),
         ("float8_e4m3fn", "float16"), ("float8_e4m3fn", "bfloat16")]


def dt(name):
    import torch
    return getattr(torch, name)


# ------------------------------------------------------------ the definition

def scale_of(byte):
    import torch
    b = byte.double()
    return torch.where(b == 255, torch.full_like(b, math.nan), torch.where(b == 0, torch.zeros_like(b), torch.exp2(b - 127)))


def quantised(x, storage):
    """(values, bytes) of rows [..., width] in 64 bits: the smallest E >= -126
    with |x| <= L 2^E, and the nearest representable multiple, ties to even."""
    import torch
    largest, bits = EIGHT[storage]
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    safe = torch.where(fine & (top > 0), top, torch.ones_like(top))
    e = torch.ceil(torch.log2(safe / largest))
    e = torch.where(safe > largest * torch.exp2(e), e + 1, e)
    e = torch.where(safe <= largest * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    y = torch.where(fine, x, torch.zeros_like(x)) * torch.exp2(-e)
    if bits:
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - bits)
        y = torch.round(y / step) * step
    else:
        y = torch.round(y)
    y = torch.where(fine, y * torch.exp2(e), torch.full_like(y, math.nan))
    return y, torch.where(fine, e + 127, torch.full_like(e, 255)).squeeze(-1).to(torch.uint8)


def held_rows(cache, table_row, length):
    """[length, heads, width] of one sequence in 64 bits, no more than its table
    has places for; rows of no page are zeros."""
    import torch
    length = min(length, len(table_row) * cache.page_rows)
    out = torch.zeros(length, cache.heads, cache.head_width, dtype=torch.float64, device="cuda")
    k, v = out, out.clone()
    columns = table_row.tolist()
    for c in range(-(-length // cache.page_rows)):
        page = columns[c] if c < len(columns) else -1
        if not 0 <= page < cache.pages:
            continue
        n = min(cache.page_rows, length - c * cache.page_rows)
        for pool, scale, to in ((cache.keys, cache.key_scales, k), (cache.values, cache.value_scales, v)):
            x = pool[page].to(torch.float32).double()
            if scale is not None:
                x = x * scale_of(scale[page])[..., None]
            to[c * cache.page_rows:c * cache.page_rows + n] = x.transpose(0, 1)[:n]
    return k, v


def expected(q, k, v, scale, causal, first):
    """(out, lse, tolerance of out, of lse) of one sequence's rows [n, heads,
    width] over its held rows, in 64 bits; row i stands at position first + i.

    Tolerances.  u is half a step of the output's type, relative.  The result
    is rounded once: u |o|.  A probability may be rounded to 16 bits before it
    meets its value: u A, A = sum_j p_j |v_j|.  A score's fp32 sum of D
    products is off by at most (D + 3) 2^-24 sum_d |q_d k_d| scale, absolute,
    which is its exponential's relative error, with 2^-18 for the exponential
    itself; it counts twice, in the sum of p and in that of p v.  The sums over
    L keys add L 2^-24.
    """
    import torch
    n, heads, width = q.shape
    group = heads // k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    q64 = q.double()
    out = torch.zeros(n, heads, width, dtype=torch.float64, device=q.device)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
    tol, lse_tol = torch.zeros_like(out), torch.zeros(n, heads, dtype=torch.float64, device=q.device)
    for i in range(n):
        seen = min(first + i + 1, k.shape[0]) if causal else k.shape[0]
        if seen <= 0:
            continue
        kk, vv = (x[:seen].repeat_interleave(group, 1) for x in (k, v))
        s = torch.einsum("hd,jhd->hj", q64[i], kk) * scale
        big = torch.einsum("hd,jhd->hj", q64[i].abs(), kk.abs()).amax(1) * abs(scale)
        lse[i] = torch.logsumexp(s, 1)
        p = torch.exp(s - lse[i][:, None])
        out[i] = torch.einsum("hj,jhd->hd", p, vv)
        each = ((width + 3) * 2.0 ** -24 * big + 2.0 ** -18)
        a = torch.einsum("hj,jhd->hd", p, vv.abs())
        tol[i] = u * out[i].abs() + (u + 2 * each[:, None] + seen * 2.0 ** -24) * a + torch.finfo(q.dtype).tiny
        lse_tol[i] = each + seen * 2.0 ** -24 + 2.0 ** -23 * lse[i].abs()
    return out, lse, tol, lse_tol


# ------------------------------------------------------------------- helpers

def make_cache(storage, pages, heads, page_rows, width, seed, order="heads", fill="normal"):
    """A cache whose every row holds something; order "rows" puts a page's rows
    before its heads, "pages" puts heads before pages."""
    import torch
    from whispereacp_b200 import PagedCache
    g = torch.Generator("cuda").manual_seed(seed)
    extents = {"heads": (pages, heads, page_rows, width), "rows": (pages, page_rows, heads, width),
               "pages": (heads, pages, page_rows, width)}[order]
    back = {"heads": (0, 1, 2, 3), "rows": (0, 2, 1, 3), "pages": (1, 0, 2, 3)}[order]
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(extents, generator=g, device="cuda")
        if storage in EIGHT:
            # the values by torch's own conversions: the tests of append check these against the definition
            e = torch.randint(118, 123, (pages, heads, page_rows), generator=g, device="cuda", dtype=torch.uint8)
            pools.append((x * 40).clamp(-127, 127).round().to(torch.int8) if storage == "int8" else (x * 100).to(dt(storage)))
            scales.append(e)
        else:
            pools.append(x.to(dt(storage)))
    pools = [p.permute(back) for p in pools]
    return PagedCache(*pools, *scales)


def bits_of(t):
    import torch
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def make_batch(lengths, new, page_rows, pages, seed, columns=None, lead=0):
    """(CacheBatch, starts): distinct pages in a shuffled order."""
    import torch
    from whispereacp_b200 import CacheBatch
    rng = np.random.default_rng(seed)
    columns = columns or max(1, max(-(-n // page_rows) for n in lengths))
    order = rng.permutation(pages)
    table = rng.integers(0, pages, (len(lengths), columns))
    used = 0
    for s, n in enumerate(lengths):
        need = min(columns, -(-n // page_rows))
        table[s, :need] = order[used:used + need]
        used += need
    assert used <= pages
    starts = lead + np.concatenate([[0], np.cumsum(new)])
    tensors = [torch.tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda") for x in (table, lengths, starts)]
    return CacheBatch(*tensors, max_rows=max(new)), starts


def check_attend(cache, batch, starts, q, out, lse, scale, causal):
    import torch
    got, got_lse = out.double(), lse.double()
    for s in range(len(starts) - 1):
        a, b = int(starts[s]), int(starts[s + 1])
        if a == b:
            continue
        length = int(batch.lengths[s])
        k, v = held_rows(cache, batch.page_table[s], length)
        o, l, tol, lse_tol = expected(q[a:b], k, v, scale, causal, length - (b - a))
        # A held NaN (100 times a normal value may be above e4m3's 448) makes
        # the rows that see it NaN, here and there.
        none, none_lse = torch.isnan(o), torch.isnan(l)
        assert torch.equal(torch.isnan(got[a:b]), none) and torch.equal(torch.isnan(got_lse[a:b]), none_lse)
        off = (got[a:b] - o).abs()
        assert bool((off <= tol)[~none].all()), (s, length, b - a, float((off / tol.clamp(min=1e-300))[~none].max()))
        empty = torch.isinf(l)
        assert torch.equal(torch.isneginf(got_lse[a:b]), empty)
        off, lse_tol = (got_lse[a:b] - l).abs()[~empty & ~none_lse], lse_tol[~empty & ~none_lse]
        assert bool((off <= lse_tol).all()), (s, length, b - a, float((off / lse_tol).max()))


def queries(rows, heads, width, dtype, seed, strided=False):
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    if strided:
        wide = torch.randn(rows, heads + 3, width, generator=g, device="cuda").to(dt(dtype))
        return wide[:, 2:heads + 2]
    return torch.randn(rows, heads, width, generator=g, device="cuda").to(dt(dtype))


# -------------------------------------------------------------------- append

@pytest.mark.parametrize("source", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("storage", ["float16", "bfloat16", "int8", "float8_e4m3fn"])
@pytest.mark.parametrize("width,heads,page_rows,order", [(64, 5, 16, "heads"), (128, 3, 32, "rows"), (64, 1, 256, "pages")])
def test_append_and_read_are_the_definition(storage, source, width, heads, page_rows, order):
    """Every value and scale byte exactly; a row of zeros, rows whose largest
    magnitude stands at and beside the border of a scale, tiny and huge rows,
    infinities and NaN; rows of no sequence and rows behind the pages alone."""
    import torch
    cache = make_cache(storage, 40, heads, page_rows, width, 3, order)
    lengths, new = [7, 0, 40, 33, 300], [7, 0, 1, 18, 70]
    batch, starts = make_batch(lengths, new, page_rows, 40, 4, lead=2)
    rows = int(starts[-1]) + 3
    g = torch.Generator("cuda").manual_seed(5)
    k, v = (torch.randn(rows, heads + 2, width, generator=g, device="cuda")[:, 1:heads + 1] for _ in range(2))
    k[3] = 0
    largest = EIGHT.get(storage, (1.0, None))[0]
    for i, factor in enumerate((1.0, 1.0 + 2.0 ** -7, 1.0 - 2.0 ** -7, 0.5, 2.0)):
        k[4 + i, :, 0] = largest * factor * 2.0 ** -6
        k[4 + i, :, 1:] *= 2.0 ** -4
    k[20] *= 2.0 ** -13
    v[21] *= 2.0 ** 12
    if source != "float16":
        k[22] *= 2.0 ** -120
        v[23] *= 2.0 ** 100 if storage != "float16" else 1.0
    v[24, 0, 5], v[25, 0, 6], k[26, 0, 0] = math.inf, math.nan, -math.inf
    k, v = k.to(dt(source)), v.to(dt(source))
    before = [bits_of(t).clone() for t in (cache.keys, cache.values)]
    cache.append(batch, k, v)
    untouched = torch.ones(cache.pages, page_rows, dtype=torch.bool, device="cuda")
    for s in range(len(lengths)):
        for i in range(new[s]):
            r, position = int(starts[s]) + i, lengths[s] - new[s] + i
            page, row = int(batch.page_table[s, position // page_rows]), position % page_rows
            untouched[page, row] = False
            for x, pool, scale in ((k, cache.keys, cache.key_scales), (v, cache.values, cache.value_scales)):
                if storage in EIGHT:
                    y, byte = quantised(x[r], storage)
                    assert torch.equal(scale[page, :, row], byte), (s, i)
                    assert torch.equal((pool[page, :, row].float().double() * scale_of(byte)[:, None]).nan_to_num(7e9), y.nan_to_num(7e9)), (s, i)
                else:
                    assert torch.equal(pool[page, :, row].nan_to_num(3), x[r].to(pool.dtype).nan_to_num(3)), (s, i)
    for t, was in zip((cache.keys, cache.values), before):
        assert torch.equal(bits_of(t).transpose(1, 2)[untouched], was.transpose(1, 2)[untouched])
    for target in ("float32", "float16", "bfloat16"):
        sentinel = [torch.full((rows, heads, width), 77.0, dtype=dt(target), device="cuda") for _ in range(2)]
        cache.read(batch, *sentinel)
        for got, which in zip(sentinel, (0, 1)):
            for s in range(len(lengths)):
                held = held_rows(cache, batch.page_table[s], lengths[s])[which]
                want = held[lengths[s] - new[s]:].to(torch.float32).to(dt(target))
                assert torch.equal(got[int(starts[s]):int(starts[s + 1])].nan_to_num(3), want.nan_to_num(3)), (target, s)
            assert bool((got[:int(starts[0])] == 77).all()) and bool((got[int(starts[-1]):] == 77).all())


def test_rows_of_no_page_are_not_written_and_read_as_zeros():
    import torch
    cache = make_cache("float16", 8, 2, 16, 64, 1)
    batch, starts = make_batch([40, 20], [40, 20], 16, 8, 2, columns=2)  # sequence 0's rows 32.. lie behind the table
    batch.page_table[1, 0] = -1
    batch.page_table[1, 1] = 8
    before = cache.keys.clone()
    k = queries(60, 2, 64, "float16", 3)
    cache.append(batch, k, k)
    changed = (cache.keys != before).any(-1).any(1).sum(1)
    assert int(changed.sum()) == 32
    a, b = cache.read(batch)
    assert torch.equal(a[:32], k[:32]) and torch.equal(b[:32], k[:32])
    assert bool((a[32:] == 0).all()) and bool((b[32:] == 0).all())


def test_more_new_rows_than_a_length_holds():
    """Rows before position 0 have no place: not written, read as zeros, and
    their attention sees nothing."""
    import torch
    cache = make_cache("bfloat16", 8, 2, 16, 64, 1)
    batch, starts = make_batch([3, 0], [5, 2], 16, 8, 2)
    k = queries(7, 2, 64, "bfloat16", 3)
    before = cache.keys.clone()
    cache.append(batch, k, k)
    assert int((cache.keys != before).any(-1).any(1).sum()) == 3
    a, _ = cache.read(batch)
    assert bool((a[:2] == 0).all()) and torch.equal(a[2:5], k[2:5]) and bool((a[5:] == 0).all())
    for causal in (True, False):
        out, lse = cache.attend(batch, k, causal=causal, return_lse=True)
        check_attend(cache, batch, starts, k, out, lse, 0.125, causal)
        empty = 2 if causal else 0
        assert bool((out[:empty] == 0).all()) and bool(torch.isneginf(lse[:empty]).all())
        assert bool((out[5:] == 0).all()) and bool(torch.isneginf(lse[5:]).all())


# ------------------------------------------------------------------ attention

# (lengths with the new rows, new rows): single tokens, chunks of a few rows
# and of several tiles, ends inside and at pages and tiles, sequences without
# new rows and without any row.
TOKENS = ([1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 449, 1000, 0, 3], [1] * 13 + [0])
FEW = ([4, 64, 66, 200, 9, 31], [4, 3, 2, 5, 0, 7])
CHUNKS = ([130, 257, 129, 500, 128, 640, 1, 70], [130, 129, 1, 260, 128, 17, 1, 0])


@pytest.mark.parametrize("storage,dtype", PAIRS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("width,heads,group,page_rows,rows", [
    (64, 3, 1, 16, TOKENS), (128, 2, 4, 64, TOKENS), (64, 2, 3, 32, FEW), (128, 1, 8, 128, FEW),
    (64, 2, 1, 16, CHUNKS), (128, 1, 3, 256, CHUNKS), (64, 1, 7, 64, CHUNKS), (128, 2, 1, 16, CHUNKS)])
def test_attention_is_the_definition(storage, dtype, causal, width, heads, group, page_rows, rows):
    lengths, new = rows
    pages = sum(-(-n // page_rows) for n in lengths) + 2
    cache = make_cache(storage, pages, heads, page_rows, width, 7)
    batch, starts = make_batch(lengths, new, page_rows, pages, 8)
    q = queries(int(starts[-1]), heads * group, width, dtype, 9)
    scale = 1 / math.sqrt(width)
    out, lse = cache.attend(batch, q, causal=causal, return_lse=True)
    check_attend(cache, batch, starts, q, out, lse, scale, causal)
    again, lse_again = cache.attend(batch, q, causal=causal, return_lse=True)
    assert np.array_equal(bits_of(out).cpu().numpy(), bits_of(again).cpu().numpy())  # the same bits every time
    assert np.array_equal(bits_of(lse).cpu().numpy(), bits_of(lse_again).cpu().numpy())
    cache.check()


@pytest.mark.parametrize("order", ["heads", "rows", "pages"])
@pytest.mark.parametrize("storage,dtype,width", [("float16", "float16", 64), ("int8", "bfloat16", 128), ("float8_e4m3fn", "float16", 64), ("bfloat16", "bfloat16", 128)])
@pytest.mark.parametrize("rows", [TOKENS, CHUNKS])
def test_attention_over_strided_pools_rows_and_a_stride_in_the_table(order, storage, dtype, width, rows):
    """Queries out of a wider projection, results into one, the pools' orders,
    a table wider than its columns, and rows of no sequence left alone."""
    import torch
    from whispereacp_b200 import CacheBatch
    lengths, new = rows
    pages = sum(-(-n // 16) for n in lengths) + 2
    cache = make_cache(storage, pages, 2, 16, width, 17, order)
    batch, starts = make_batch(lengths, new, 16, pages, 18, lead=3)
    wide = torch.full((len(lengths), batch.page_table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, :-5] = batch.page_table
    batch = CacheBatch(wide[:, :-5], batch.lengths, batch.starts, max_rows=max(new))
    total = int(starts[-1]) + 4
    q = queries(total, 4, width, dtype, 19, strided=True)
    target = torch.full((total, 9, width), 5.0, dtype=dt(dtype), device="cuda")
    lse = torch.full((total, 4), 5.0, device="cuda")
    cache.attend(batch, q, out=target[:, 1:5], lse=lse, scale=0.2)
    check_attend(cache, batch, starts, q, target[:, 1:5], lse, float(np.float32(0.2)), True)
    assert bool((target[:, 0] == 5).all()) and bool((target[:, 5:] == 5).all())
    outside = torch.ones(total, dtype=torch.bool, device="cuda")
    outside[int(starts[0]):int(starts[-1])] = False
    assert bool((target[outside] == 5).all()) and bool((lse[outside] == 5).all())


@pytest.mark.parametrize("storage,dtype", PAIRS)
@pytest.mark.parametrize("rows", [TOKENS, FEW, CHUNKS])
def test_what_a_row_does_not_see_cannot_change_it(storage, dtype, rows):
    """Pages' rows behind the lengths hold NaN, and the last held rows hold
    infinities and NaN: only rows that see those may change."""
    import torch
    lengths, new = rows
    pages = sum(-(-n // 32) for n in lengths) + 2
    cache = make_cache(storage, pages, 2, 32, 64, 27)
    batch, starts = make_batch(lengths, new, 32, pages, 28)
    q = queries(int(starts[-1]), 4, 64, dtype, 29)
    clean, clean_lse = cache.attend(batch, q, return_lse=True)
    untouched = torch.ones(pages, 32, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lengths):
        for p in range(n):
            untouched[int(batch.page_table[s, p // 32]), p % 32] = False

    def poison(page, row, value):
        for pool, scale in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
            if scale is not None:
                scale[page, :, row] = 255
            else:
                pool[page, :, row] = value

    page, row = torch.nonzero(untouched, as_tuple=True)
    poison(page, row, math.nan)
    out, lse = cache.attend(batch, q, return_lse=True)
    assert torch.equal(bits_of(out), bits_of(clean)) and torch.equal(bits_of(lse), bits_of(clean_lse))
    for s, n in enumerate(lengths):
        if new[s] > 1:
            poison(int(batch.page_table[s, (n - 1) // 32]), (n - 1) % 32, math.inf if s % 2 else math.nan)
    out, lse = cache.attend(batch, q, return_lse=True)
    for s in range(len(lengths)):
        a, b = int(starts[s]), int(starts[s + 1])
        if new[s] > 1:
            assert bool(torch.isnan(out[b - 1]).any()), s
            b -= 1
        assert torch.equal(torch.isfinite(out[a:b]), torch.isfinite(clean[a:b]))
    # the rows before the poisoned ones: the definition's values still
    for s in range(len(lengths)):
        a, b = int(starts[s]), int(starts[s + 1])
        if new[s] > 1:
            k, v = held_rows(cache, batch.page_table[s], lengths[s])
            k, v = k[:-1], v[:-1]
            o, l, tol, lse_tol = expected(q[a:b - 1], k, v, 0.125, True, lengths[s] - new[s])
            assert torch.equal(torch.isnan(out[a:b - 1]), torch.isnan(o))
            assert bool(((out[a:b - 1].double() - o).abs() <= tol)[~torch.isnan(o)].all())
            assert bool(((lse[a:b - 1].double() - l).abs() <= lse_tol)[~torch.isnan(l) & ~torch.isinf(l)].all())


@pytest.mark.parametrize("storage,dtype", [("bfloat16", "bfloat16"), ("int8", "float16")])
def test_chunks_of_a_long_context_whose_last_key_is_no_number(storage, dtype):
    """Whole items of many heads: every row that shares the last key's block is
    computed again, alone, while the CTA's other warps wait for its next item."""
    import torch
    length, new, heads = 6000, 300, 160
    cache = make_cache(storage, 400, heads, 16, 128, 217)
    batch, starts = make_batch([length], [new], 16, 400, 218)
    page, row = int(batch.page_table[0, (length - 1) // 16]), (length - 1) % 16
    for pool, scale in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        if scale is not None:
            scale[page, :, row] = 255
        else:
            pool[page, :, row] = math.nan
    q = queries(int(starts[-1]), heads, 128, dtype, 219)
    out, lse = cache.attend(batch, q, return_lse=True)
    cache.check()
    a, b = int(starts[0]), int(starts[-1])
    assert bool(torch.isnan(out[b - 1]).all()) and bool(torch.isnan(lse[b - 1]).all())
    for h in range(0, heads, 53):
        k, v = (x[:-1, h:h + 1].contiguous() for x in held_rows(cache, batch.page_table[0], length))
        o, l, tol, lse_tol = expected(q[a:b - 1, h:h + 1], k, v, 128 ** -0.5, True, length - new)
        assert bool(((out[a:b - 1, h:h + 1].double() - o).abs() <= tol).all())
        assert bool(((lse[a:b - 1, h:h + 1].double() - l).abs() <= lse_tol).all())


@pytest.mark.parametrize("storage,dtype", [("float16", "float16"), ("bfloat16", "bfloat16"), ("int8", "float16")])
def test_large_scores_and_large_values(storage, dtype):
    """Scores in the hundreds, a maximum that grows tile by tile, and values
    whose scales differ by 2^20."""
    import torch
    lengths, new = [700, 300], [1, 150]
    pages = 70
    cache = make_cache(storage, pages, 2, 16, 64, 37)
    batch, starts = make_batch(lengths, new, 16, pages, 38)
    for s in range(2):
        for p in range(lengths[s]):
            page, row = int(batch.page_table[s, p // 16]), p % 16
            factor = 2.0 ** (p * 5 // lengths[s])
            if storage == "int8":
                cache.key_scales[page, :, row] = 118 + p * 5 // lengths[s]
                cache.value_scales[page, :, row] = 110 + (p * 7919) % 21
            else:
                cache.keys[page, :, row] *= factor
                cache.values[page, :, row] *= 2.0 ** ((p * 7919) % 10 - 5)
    q = queries(int(starts[-1]), 2, 64, dtype, 39) * 4
    for causal in (True, False):
        out, lse = cache.attend(batch, q, causal=causal, return_lse=True)
        check_attend(cache, batch, starts, q, out, lse, 0.125, causal)


def test_rows_of_no_page_take_part_as_zeros_and_those_outside_the_table_do_not():
    cache = make_cache("float16", 20, 2, 16, 64, 47)
    for new in ([1, 1], [140, 2]):
        # 150 rows, of which the table has places for 144
        batch, starts = make_batch([150, 70], new, 16, 20, 48, columns=9)
        batch.page_table[0, 3] = -1
        batch.page_table[1, 1] = 20
        q = queries(int(starts[-1]), 2, 64, "float16", 49)
        out, lse = cache.attend(batch, q, return_lse=True)
        check_attend(cache, batch, starts, q, out, lse, 0.125, True)


@pytest.mark.parametrize("storage,dtype,width", [("bfloat16", "bfloat16", 64), ("int8", "float16", 64), ("float8_e4m3fn", "bfloat16", 128)])
def test_one_long_context_split_over_the_gpu(storage, dtype, width):
    """One sequence of one head over 40000 rows: its keys are split; next to a
    short one, and with a chunk."""
    for new in ([1, 1, 1], [9, 1, 2], [200, 1, 0]):
        lengths = [40000, 5, 3]
        cache = make_cache(storage, 320, 1, 128, width, 57)
        batch, starts = make_batch(lengths, new, 128, 320, 58)
        q = queries(int(starts[-1]), 1, width, dtype, 59)
        out, lse = cache.attend(batch, q, return_lse=True)
        check_attend(cache, batch, starts, q, out, lse, 1 / math.sqrt(width), True)
        cache.check()


def test_pools_whose_offsets_pass_32_bits():
    """9 GB of pools; the sequences' pages lie at both ends."""
    import torch
    from whispereacp_b200 import CacheBatch, PagedCache
    pages, heads, page_rows, width = 36000, 16, 64, 64
    keys, values = (torch.empty(pages, heads, page_rows, width, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ids = [35999, 0, 35990, 17, 35000, 35001, 30000, 35002]
    for page in ids:
        keys[page].normal_()
        values[page].normal_()
    cache = PagedCache(keys, values)
    table = torch.tensor([ids[:4], ids[4:]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([250, 200], dtype=torch.int32, device="cuda")
    for new in ([1, 1], [130, 1]):
        starts = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device="cuda")
        batch = CacheBatch(table, lengths, starts)
        k, v = queries(sum(new), heads, width, "bfloat16", 67), queries(sum(new), heads, width, "bfloat16", 68)
        cache.append(batch, k, v)
        a, b = cache.read(batch)
        assert torch.equal(a, k) and torch.equal(b, v)
        q = queries(sum(new), heads, width, "bfloat16", 69)
        out, lse = cache.attend(batch, q, return_lse=True)
        check_attend(cache, batch, starts.tolist(), q, out, lse, 0.125, True)


# Calls of little work are one kernel's whatever their rows; what a table has
# places for bounds the work, so the same sequences in a wide table are another's.

def wide_batches(monkeypatch):
    import sys
    here = sys.modules[__name__]
    plain = here.make_batch

    def wide(lengths, new, page_rows, pages, seed, columns=None, lead=0):
        return plain(lengths, new, page_rows, pages, seed, columns=(64 * 2400) // page_rows, lead=lead)

    monkeypatch.setattr(here, "make_batch", wide)


@pytest.mark.parametrize("storage,dtype", PAIRS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("width,heads,group,page_rows,rows", [
    (64, 2, 1, 16, CHUNKS), (128, 1, 3, 256, CHUNKS), (64, 1, 7, 64, CHUNKS), (128, 2, 1, 16, CHUNKS),
    (64, 2, 3, 32, FEW), (128, 1, 8, 128, FEW)])
def test_attention_under_a_wide_table(monkeypatch, storage, dtype, causal, width, heads, group, page_rows, rows):
    wide_batches(monkeypatch)
    test_attention_is_the_definition(storage, dtype, causal, width, heads, group, page_rows, rows)


@pytest.mark.parametrize("storage,dtype", PAIRS)
def test_unseen_keys_under_a_wide_table(monkeypatch, storage, dtype):
    wide_batches(monkeypatch)
    test_what_a_row_does_not_see_cannot_change_it(storage, dtype, CHUNKS)


@pytest.mark.parametrize("storage,dtype", [("float16", "float16"), ("bfloat16", "bfloat16"), ("int8", "float16")])
def test_large_scores_under_a_wide_table(monkeypatch, storage, dtype):
    wide_batches(monkeypatch)
    test_large_scores_and_large_values(storage, dtype)


@pytest.mark.parametrize("storage,dtype", [("float16", "float16"), ("int8", "bfloat16")])
def test_scales_under_a_wide_table(monkeypatch, storage, dtype):
    wide_batches(monkeypatch)
    for scale in (0.0, -0.3):
        test_a_scale_below_or_at_zero(storage, dtype, ([200, 300], [90, 130]), scale)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("columns", [20, 9600])
def test_first_keys_of_score_minus_infinity(dtype, width, columns):
    """The first 70 keys weigh nothing: the row's first numbers come in the
    middle of a block."""
    import torch
    cache = make_cache(dtype, 40, 2, 16, width, 401)
    batch, starts = make_batch([300], [130], 16, 40, 402, columns=columns)
    for p in range(70):
        cache.keys[int(batch.page_table[0, p // 16]), :, p % 16] = -math.inf
    q = queries(130, 2, width, dtype, 403).abs() + 0.01
    out, lse = cache.attend(batch, q, return_lse=True)
    k, v = held_rows(cache, batch.page_table[0], 300)
    o, l, tol, lse_tol = expected(q, k[70:], v[70:], width ** -0.5, True, 100)
    assert bool(((out.double() - o).abs() <= tol).all())
    assert bool(((lse.double() - l).abs() <= lse_tol).all())


def test_two_streams_under_a_wide_table(monkeypatch):
    wide_batches(monkeypatch)
    test_two_streams_at_once()


@pytest.mark.parametrize("storage,dtype", PAIRS)
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("most", [9, 16, 17, 31, 33, 63, 65])
def test_chunks_around_the_kernels_limits(storage, dtype, width, most):
    """The row counts where one kernel ends and the other begins, of a group of
    one, alone and beside single tokens and an empty sequence."""
    cache = make_cache(storage, 400, 2, 16, width, 301)
    for new in ([most], [most, 1, 0, most - 1]):
        lengths = [max(n, 1) + 40 * i for i, n in enumerate(new)]
        for columns in (20, 9600):
            batch, starts = make_batch(lengths, new, 16, 400, 302, columns=columns)
            q = queries(sum(new), 2, width, dtype, 303)
            out, lse = cache.attend(batch, q, return_lse=True)
            check_attend(cache, batch, starts, q, out, lse, width ** -0.5, True)


# ------------------------------------------------------- streams and graphs

def test_a_step_captured_and_replayed_with_other_contents():
    """append and attend captured once; between replays the caller rewrites
    lengths, table, rows and queries in place.  Two graphs alive at once, each
    with its own workspace, replayed on two streams at once."""
    import torch
    lengths, new = [30, 100, 300], [1, 1, 1]
    cache = make_cache("float16", 64, 4, 16, 64, 77)
    batch, starts = make_batch(lengths, new, 16, 64, 78, columns=20)
    graphs = []
    for n in range(2):
        q, k, v = (queries(3, 4, 64, "float16", 79 + n * 3 + i) for i in range(3))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cache.attend(batch, q, return_lse=True)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            if n == 0:
                cache.append(batch, k, v)
            out, lse = cache.attend(batch, q, return_lse=True)
        graphs.append((graph, q, k, v, out, lse))
    graph, q, k, v, out, lse = graphs[0]
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check_attend(cache, batch, starts, q, out, lse, 0.125, True)
        a, _ = cache.read(batch)
        assert torch.equal(a, k)
        batch.lengths += 1
        q.copy_(queries(3, 4, 64, "float16", 90 + step))
        k.copy_(queries(3, 4, 64, "float16", 95 + step))
    graph.replay()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (g, *_rest), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for _, q, k, v, out, lse in graphs:
        check_attend(cache, batch, starts, q, out, lse, 0.125, True)


@pytest.mark.parametrize("columns", [40, 400])
def test_a_mixed_batch_captured_and_replayed(columns):
    """Chunks, tokens and the join of both in one graph, an append before and a
    read behind them; the contents change between the replays."""
    import torch
    lengths, new = [700, 100, 300, 64], [150, 1, 20, 0]
    cache = make_cache("int8", 128, 2, 32, 128, 177)
    batch, starts = make_batch([n + 51 for n in lengths], new, 32, 128, 178, columns=columns)
    batch.lengths -= 51  # pages for every replay's rows
    rows = int(starts[-1])
    q = queries(rows, 6, 128, "bfloat16", 179)
    k, v = queries(rows, 2, 128, "bfloat16", 180), queries(rows, 2, 128, "bfloat16", 181)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(batch, q, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(batch, k, v)
        out, lse = cache.attend(batch, q, return_lse=True)
        again, all_lse = cache.attend(batch, q, causal=False, return_lse=True)
        kr, vr = cache.read(batch, dtype=torch.float32, rows=rows)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check_attend(cache, batch, starts, q, out, lse, 128 ** -0.5, True)
        check_attend(cache, batch, starts, q, again, all_lse, 128 ** -0.5, False)
        first, last = int(starts[0]), int(starts[-1])
        assert torch.equal(kr[first:last].double(), quantised(k[first:last], "int8")[0])
        assert torch.equal(vr[first:last].double(), quantised(v[first:last], "int8")[0])
        batch.lengths += 17
        q.copy_(queries(rows, 6, 128, "bfloat16", 190 + step))
        k.copy_(queries(rows, 2, 128, "bfloat16", 195 + step))
    cache.check()


def test_two_streams_at_once():
    import torch
    cache = make_cache("int8", 200, 4, 16, 64, 107)
    batch, starts = make_batch([1000, 900, 20], [1, 1, 1], 16, 200, 108)
    chunk, chunk_starts = make_batch([1000, 900, 20], [200, 3, 20], 16, 200, 108)
    q, qc = queries(3, 8, 64, "float16", 109), queries(223, 8, 64, "float16", 110)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = []
    for _ in range(10):
        results.append((cache.attend(batch, q, return_lse=True, stream=streams[0]),
                        cache.attend(chunk, qc, return_lse=True, stream=streams[1].cuda_stream)))
    torch.cuda.synchronize()
    for (o, l), (oc, lc) in results[:1] + results[-1:]:
        check_attend(cache, batch, starts, q, o, l, 0.125, True)
        check_attend(cache, chunk, chunk_starts, qc, oc, lc, 0.125, True)
    assert all(torch.equal(o, results[0][0][0]) and torch.equal(oc, results[0][1][0]) for (o, _), (oc, _) in results)


def test_a_cache_over_memory_of_its_own():
    """wsp_cache_create without memory: zeroed pools of the library."""
    import ctypes
    import torch
    from whispereacp_b200 import _native as N
    lib = N.library()
    handle = ctypes.c_void_p()
    shape = N.CCacheShape(2, 64, 16, 4, N.WSP_CACHE_INT8)
    N.check(lib.wsp_cache_create(ctypes.byref(shape), 0, None, ctypes.byref(handle)))
    memory = N.CCacheMemory()
    N.check(lib.wsp_cache_get_memory(handle, ctypes.byref(memory)))
    assert (memory.page_stride, memory.head_stride, memory.row_stride) == (2048, 1024, 64)
    batch, starts = make_batch([20], [20], 16, 4, 1)
    k = queries(20, 2, 64, "float16", 2)
    out = torch.empty_like(k)
    rows = [N.CCacheRows(t.data_ptr(), 128, 64, N.WSP_FLOAT16) for t in (k, k, out, out)]
    N.check(lib.wsp_cache_append(handle, batch._ref, 20, ctypes.byref(rows[0]), ctypes.byref(rows[1]), None))
    N.check(lib.wsp_cache_read(handle, batch._ref, 20, ctypes.byref(rows[2]), ctypes.byref(rows[3]), None))
    torch.cuda.synchronize()
    assert torch.equal(out.double(), quantised(k, "int8")[0])
    lib.wsp_cache_destroy(handle)


# ------------------------------------------------- as a decoder would use it

def test_windows_at_their_own_tokens_follow_the_decoder():
    """A Whisper decoder layer stack over paged caches (projections in torch),
    two windows that stand at different tokens, against the lockstep decoder
    run one window at a time: prompts as chunks, then single tokens.

    The logits stay within the bound the decoder itself is held to (2e-2), and
    so within twice that of the decoder's."""
    import torch
    from tests.helpers import make_decoder, stored_tensors
    from oracle import oracle as O
    from whispereacp_b200 import CacheBatch, PagedCache
    from whispereacp_b200 import synthetic as S
    from whispereacp_b200.decoder import DecoderShape
    shape = DecoderShape(width=128, heads=2, layers=2, feed_forward_width=256, vocabulary_size=500, max_positions=64,
                         cross_positions=50)
    tensors = stored_tensors(S.normal_weights(shape, seed=5), "float16")
    encoder = S.encoder_output(2, shape.cross_positions, shape.width, seed=6)
    tokens = [[int(t) for t in S.teacher_tokens(n, seed=7 + n, high=499)] for n in (9, 5)]
    w = {n.replace("model.decoder.", ""): torch.tensor(v, device="cuda") for n, v in tensors.items()}
    H, D = shape.heads, 64

    def linear(x, name):
        y = x @ w[name + ".weight"].T
        return y + w[name + ".bias"] if name + ".bias" in w else y

    def norm(x, name):
        return torch.nn.functional.layer_norm(x, (shape.width,), w[name + ".weight"], w[name + ".bias"], 1e-5)

    rows16 = torch.float16
    selfs = [PagedCache.allocate(12, H, 16, D) for _ in range(shape.layers)]
    crosses = [PagedCache.allocate(10, H, 16, D) for _ in range(shape.layers)]
    i32 = dict(dtype=torch.int32, device="cuda")
    cross_table = torch.tensor([[7, 1, 3, 9], [0, 2, 8, 4]], **i32)
    X = shape.cross_positions
    start = CacheBatch(cross_table, torch.tensor([X, X], **i32), torch.tensor([0, X, 2 * X], **i32), max_rows=X)
    e = torch.tensor(np.ascontiguousarray(encoder).reshape(2 * X, shape.width), device="cuda")
    for l in range(shape.layers):
        k, v = (linear(e, f"layers.{l}.encoder_attn.{p}_proj").to(rows16).view(-1, H, D) for p in "kv")
        crosses[l].append(start, k, v)
    table = torch.tensor([[5, 3, 11, 0], [1, 2, 10, 4]], **i32)

    def step(new, held):
        """new: each window's tokens of this step; the logits of every one."""
        counts = [len(t) for t in new]
        rows = sum(counts)
        starts = torch.tensor([0, counts[0], rows], **i32)
        own = CacheBatch(table, torch.tensor([h + n for h, n in zip(held, counts)], **i32), starts, max_rows=max(counts))
        other = CacheBatch(cross_table, torch.tensor([X, X], **i32), starts, max_rows=max(counts))
        ids = torch.tensor([t for ts in new for t in ts], device="cuda")
        places = torch.tensor([h + i for h, n in zip(held, counts) for i in range(n)], device="cuda")
        x = w["embed_tokens.weight"][ids] + w["embed_positions.weight"][places]
        for l in range(shape.layers):
            at = f"layers.{l}."
            y = norm(x, at + "self_attn_layer_norm")
            q, k, v = (linear(y, at + f"self_attn.{p}_proj").to(rows16).view(rows, H, D) for p in "qkv")
            selfs[l].append(own, k, v)
            x = x + linear(selfs[l].attend(own, q).float().reshape(rows, -1), at + "self_attn.out_proj")
            q = linear(norm(x, at + "encoder_attn_layer_norm"), at + "encoder_attn.q_proj").to(rows16).view(rows, H, D)
            o = crosses[l].attend(other, q, causal=False)
            x = x + linear(o.float().reshape(rows, -1), at + "encoder_attn.out_proj")
            x = x + linear(torch.nn.functional.gelu(linear(norm(x, at + "final_layer_norm"), at + "fc1")), at + "fc2")
        return norm(x, "layer_norm") @ w["embed_tokens.weight"].T

    # window 0 starts with 4 tokens, window 1 with 1; then 1 and 3, then single ones
    plan = [(4, 1), (1, 3), (1, 0), (1, 1), (2, 0)]
    held, got = [0, 0], [[], []]
    for counts in plan:
        new = [tokens[b][held[b]:held[b] + n] for b, n in enumerate(counts)]
        logits = step(new, held)
        got[0].append(logits[:counts[0]])
        got[1].append(logits[counts[0]:])
        held = [h + n for h, n in zip(held, counts)]
    for b in range(2):
        mine = torch.cat(got[b]).cpu().numpy()
        _, truth = O.reference_decode(O.Shape(**shape.__dict__), tensors, encoder[b], tokens[b])
        decoder = make_decoder(O.Shape(**shape.__dict__), tensors, "float16")
        decoder.begin_sequence(encoder[b])
        lockstep = decoder.step([tokens[b]]).logits[0]
        assert np.isfinite(mine).all()
        assert float(np.abs(mine - np.asarray(truth)).max()) <= 2e-2
        assert float(np.abs(mine - lockstep).max()) <= 4e-2


# ------------------------------------------------------- more of the range

@pytest.mark.parametrize("storage,dtype,width", [("float16", "float16", 64), ("int8", "bfloat16", 64), ("bfloat16", "bfloat16", 128)])
def test_many_sequences_of_every_kind(storage, dtype, width):
    """90 sequences -- more than one round of a warp's lanes -- with no rows,
    single ones, 2 to 16 (tiles of 8 and of 16), and chunks, in one batch."""
    rng = np.random.default_rng(5)
    for most in (1, 3, 16, 150):
        new = [int(rng.integers(0, most + 1)) for _ in range(90)]
        new[17], new[88] = most, most
        lengths = [n + int(rng.integers(0, 300)) for n in new]
        lengths[3], new[3] = 0, 0
        pages = sum(-(-n // 32) for n in lengths) + 3
        cache = make_cache(storage, pages, 2, 32, width, 6)
        batch, starts = make_batch(lengths, new, 32, pages, 7)
        q = queries(int(starts[-1]), 4, width, dtype, 8)
        for causal in (True, False):
            out, lse = cache.attend(batch, q, causal=causal, return_lse=True)
            check_attend(cache, batch, starts, q, out, lse, 1 / math.sqrt(width), causal)


@pytest.mark.parametrize("storage,source", [("float16", "float16"), ("bfloat16", "float32"), ("int8", "bfloat16"), ("float8_e4m3fn", "float16")])
def test_append_and_read_of_many_rows(storage, source):
    """Thousands of rows: blocks of several rows, ragged."""
    import torch
    rng = np.random.default_rng(11)
    lengths = [int(n) for n in rng.integers(1, 260, 60)]
    pages = sum(-(-n // 16) for n in lengths) + 2
    cache = make_cache(storage, pages, 3, 16, 64, 12)
    batch, starts = make_batch(lengths, lengths, 16, pages, 13)
    k, v = (queries(int(starts[-1]), 3, 64, source, 14 + i) for i in range(2))
    cache.append(batch, k, v)
    a, b = cache.read(batch, dtype=torch.float32)
    for x, got in ((k, a), (v, b)):
        want = quantised(x, storage)[0] if storage in EIGHT else x.to(dt(storage)).double()
        assert torch.equal(got.double(), want)


@pytest.mark.parametrize("storage,dtype", PAIRS)
@pytest.mark.parametrize("rows", [([33, 200, 5], [1, 1, 1]), ([200, 300], [90, 130])])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_a_scale_below_or_at_zero(storage, dtype, rows, scale):
    """At scale 0 every seen key weighs the same."""
    lengths, new = rows
    pages = sum(-(-n // 16) for n in lengths) + 2
    cache = make_cache(storage, pages, 2, 16, 64, 21)
    batch, starts = make_batch(lengths, new, 16, pages, 22)
    q = queries(int(starts[-1]), 2, 64, dtype, 23)
    out, lse = cache.attend(batch, q, scale=scale, return_lse=True)
    check_attend(cache, batch, starts, q, out, lse, float(np.float32(scale)), True)


def test_batches_that_ask_for_nothing_or_for_the_impossible():
    """No sequences, no rows, no columns, and rows outside the arrays."""
    import torch
    from whispereacp_b200 import CacheBatch
    cache = make_cache("float16", 8, 2, 16, 64, 31)
    i32 = dict(dtype=torch.int32, device="cuda")
    q = queries(6, 2, 64, "float16", 32)
    target = torch.full_like(q, 9.0)
    none = CacheBatch(torch.zeros(0, 4, **i32), torch.zeros(0, **i32), torch.zeros(1, **i32), max_rows=0)
    cache.append(none, q, q)
    cache.attend(none, q, out=target)
    cache.read(none, target, target.clone())
    assert bool((target == 9).all())
    # a table without columns: no keys at all
    bare = CacheBatch(torch.zeros(2, 0, **i32), torch.tensor([30, 4], **i32), torch.tensor([0, 1, 6], **i32), max_rows=5)
    cache.append(bare, q, q)
    out, lse = cache.attend(bare, q, return_lse=True)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())
    # starts past the arrays' rows: the sequences inside are done, that one is not
    table = torch.tensor([[0, 1], [2, 3]], **i32)
    past = CacheBatch(table, torch.tensor([20, 30], **i32), torch.tensor([0, 4, 90], **i32), max_rows=86)
    target.fill_(9.0)
    cache.attend(past, q, out=target)
    k, v = held_rows(cache, table[0], 20)
    o, _, tol, _ = expected(q[:4], k, v, 0.125, True, 16)
    assert bool(((target[:4].double() - o).abs() <= tol).all()) and bool((target[4:] == 9).all())
    with pytest.raises(ValueError, match="a batch of 1 sequences"):
        CacheBatch(table, torch.tensor([20], **i32), torch.tensor([0, 4], **i32))


def test_refusals_of_the_binding():
    import torch
    from whispereacp_b200 import CacheBatch, ModelError, PagedCache
    cache = make_cache("float16", 8, 2, 16, 64, 41)
    batch, _ = make_batch([20], [2], 16, 8, 42)
    q = queries(2, 4, 64, "float16", 43)
    with pytest.raises(ModelError, match="queries must be"):
        cache.attend(batch, q[0])
    with pytest.raises(ModelError, match="queries must be"):
        cache.attend(batch, queries(2, 4, 128, "float16", 43))
    with pytest.raises(ModelError, match="multiple"):
        cache.attend(batch, q[:, :3])
    with pytest.raises(ModelError, match="have its type"):
        cache.attend(batch, q.bfloat16())
    with pytest.raises(ModelError, match="16-bit"):
        cache.attend(batch, q.float())
    with pytest.raises(ValueError, match="contiguous in the last"):
        cache.attend(batch, q.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="16-byte"):
        cache.attend(batch, torch.zeros(2 * 4 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(2, 4, 64))
    with pytest.raises(ValueError, match="must be on"):
        cache.attend(batch, q.cpu())
    with pytest.raises(ValueError, match="lse"):
        cache.attend(batch, q, lse=torch.zeros(2, 3, device="cuda"))
    with pytest.raises(ValueError, match="finite"):
        cache.attend(batch, q, scale=float("nan"))
    with pytest.raises(ValueError, match="together"):
        cache.read(batch, keys=q)
    with pytest.raises(ValueError, match="rows are"):
        cache.append(batch, q[:, :2].double(), q[:, :2].double())
    with pytest.raises(ValueError, match="one dtype"):
        cache.append(batch, q[:, :2], q[:, :2].float())
    with pytest.raises(ValueError, match="alike"):
        PagedCache(cache.keys, cache.values.float())
    with pytest.raises(ValueError, match="no scales"):
        PagedCache(cache.keys, cache.values, torch.zeros(8, 2, 16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="scale bytes"):
        PagedCache(cache.keys.to(torch.int8), cache.values.to(torch.int8))
    with pytest.raises(ModelError, match="64 or 128"):
        PagedCache.allocate(4, 2, 16, 96)
    with pytest.raises(ModelError, match="a page has"):
        PagedCache.allocate(4, 2, 24, 64)
    cache.close()
    with pytest.raises(ValueError, match="closed"):
        cache.attend(batch, q)
