"""The serving operators where they are easily wrong: the bits of weights and sticks, lengths, books, layouts of queries, which
kernel runs."""
import ctypes
import math

import pytest
import torch
import torch.compiler.config

import serving_reference as R

gpu = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


# ---- attention ----------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_decode_weights_keep_their_bits(cuda_device, dtype):
    """Values that cancel: what is left of o shows the errors of the weights themselves, not the rounding of the output.

    Bound, relative to sum a|v|.  Scores of up to 0.1 (8 columns): dz = 10 * 2^-24 * 0.1, three times at most in a weight.  beta and
    1 - beta: the exponential 2^-22 (halved by 1 / (1 + e)), three roundings of 2^-24, the reciprocal 2^-23: 2^-21.4; a weight has
    up to three of them and three products: 1.3e-6.  The sums in 32 bits, perhaps truncated: 3 * 2^-23.  Together below 2^-19.
    Weights in 16 bits would be off by up to 2^-18, a quarter of these rows by more than the bound."""
    import stickbreaking_attention_b200 as sb
    gen = torch.Generator().manual_seed(60)
    seqs, heads, d = 64, 8, 8
    q, k = (0.1 * (2 * torch.rand(shape, generator=gen) - 1) for shape in ((seqs, heads, 1, d), (seqs, heads, 3, d)))
    q, k = (10 * q).to(dtype), k.to(dtype)                            # |<q, k>| <= 8 * 0.1, times 1/8
    z = (k.double() @ q.double().transpose(2, 3)).squeeze(3) / 8      # (seqs, heads, 3)
    beta = torch.sigmoid(z)
    a = beta * torch.stack(((1 - beta[..., 1]) * (1 - beta[..., 2]), 1 - beta[..., 2], torch.ones_like(beta[..., 2])), -1)
    v = torch.zeros(seqs, heads, 3, d, dtype=torch.float64)
    v[..., 2, :] = (1 + torch.rand(seqs, heads, d, generator=gen)).to(dtype).double()
    for j in (1, 0):                                                  # each takes away what the newer ones sum up to
        v[..., j, :] = (-(a[..., None] * v).sum(2) / a[..., j, None]).to(dtype).double()
    want = (a[..., None] * v).sum(2)
    bound = (2.0 ** -19 + 3 * 10 * 2.0 ** -24 * 0.1) * (a[..., None] * v.abs()).sum(2) + R.EPS[dtype] / 2 * want.abs() + R.SMALLEST[dtype]
    pages = [torch.nn.functional.pad(t.to(dtype), (0, 0, 0, 13)).to(cuda_device) for t in (k, v)]
    table = torch.arange(seqs, dtype=torch.int32, device=cuda_device)[:, None]
    lens = torch.full((seqs,), 3, dtype=torch.int32, device=cuda_device)
    with torch.no_grad():
        o, _ = sb.sb_attn_decode(q.to(cuda_device), *pages, table, lens, inv_temp=0.125, attend_current=True)
    sb.check_status(cuda_device)
    off = (o[:, :, 0].cpu().double() - want).abs() / bound
    assert float(off.max()) <= 1.0, f"{float(off.max()):.3g} times what rounding explains"


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("bits", [30, 60, 155])
def test_decode_sticks_that_wear_down_slowly(cuda_device, dtype, bits):
    """Thousands of keys that take 1/192 of the stick each, and behind them one that would take all of the rest: its weight is what
    is left of the stick, and it has the only value that is not 0.  2000 sequences with the same pages, so that few are cut.

    Bound: the reference's, and of the weight itself 2^-145 (a stick of few bits, 2^-149 to 2^-126, loses up to one of its steps of
    2^-149 per tile, of which 12 are left at a time), in fp16 2^-40 (weights are held in steps of 2^-39)."""
    import stickbreaking_attention_b200 as sb
    seqs, d, page, z = 2000, 8, 64, -5.25
    newer = math.ceil(bits * math.log(2) / math.log1p(math.exp(z)))
    n = newer + 1
    pages = -(-n // page)
    k, v = (torch.zeros(pages, 1, page, d, dtype=dtype) for _ in range(2))
    k[..., 0] = z
    k[0, 0, 0, 0] = 30.0
    large = 60000.0 if dtype == FP16 else 1e38
    v[0, 0, 0] = large
    q = torch.zeros(1, 1, 1, d, dtype=dtype)
    q[..., 0] = 1.0
    table, lens = torch.arange(pages, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    o, rem, o_err, rem_err = R.decode(q, k, v, table, lens, scale=1.0, attend_current=True)
    o_err = o_err + (2.0 ** -40 if dtype == FP16 else 2.0 ** -145) * large
    dev = lambda t: t.to(cuda_device)
    with torch.no_grad():
        got = sb.sb_attn_decode(dev(q).expand(seqs, 1, 1, d), dev(k), dev(v), dev(table).expand(seqs, pages).contiguous(),
                                dev(lens).expand(seqs).contiguous(), inv_temp=1.0, attend_current=True)
    sb.check_status(cuda_device)
    R.check_decode(got, tuple(t.expand(seqs, *t.shape[1:]) for t in (o, rem, o_err, rem_err)))


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("heads,new", [(2, 2), (2, 3), (4, 2), (2, 4), (6, 1), (8, 1), (10, 1), (4, 3)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_of_one_to_six_query_rows(cuda_device, dtype, heads, new, d):
    """Rows that share a product's columns in every way there is, cut and whole items, newest keys and values that are no numbers."""
    import stickbreaking_attention_b200 as sb
    lens, page = [0, 1, 3, 16, 113, 1500], 16
    gen = torch.Generator().manual_seed(62)
    k, v, table, lengths = R.make_cache(gen, lens, 2, page, d, dtype, shift=0.2)
    q = (torch.randn(len(lens), heads, new, d, generator=gen) + 0.2).to(dtype)
    want = R.decode(q, k, v, table, lengths)
    for b, n in enumerate(lens):                    # the newest token of each: no row attends to it
        if n:
            at = table[b, (n - 1) // page].long(), slice(None), (n - 1) % page
            k[at], v[at] = float("nan"), float("inf")
    with torch.no_grad():
        got = sb.sb_attn_decode(*(t.to(cuda_device) for t in (q, k, v, table, lengths)))
    sb.check_status(cuda_device)
    R.check_decode(got, want)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- lengths of 31 bits ----------------------------------------------------------------------------------------------------

LONGEST = 2 ** 31 - 16


@gpu
def test_extend_refuses_lengths_that_31_bits_do_not_hold(cuda_device):
    """Rows with room for more than 2^31 tokens: a sequence grows up to 2^31 - 16 and no further, and a refused call changes nothing."""
    import stickbreaking_attention_b200 as sb
    page, columns = 65536, 32770
    table = torch.full((3, columns), -1, dtype=torch.int32, device=cuda_device)
    lens, refs = ints(10, 5, 0), torch.zeros(32768 + 4, dtype=torch.int32, device=cuda_device)
    table[0, 0], table[1, 0], refs[0], refs[1] = 0, 1, 1, 1

    def extend(counts, what=None):
        before = [t.clone() for t in (table, lens, refs)]
        sb.kv_extend(table, lens, refs, counts, page)
        if what is None:
            return sb.check_status(cuda_device)
        with pytest.raises(sb._cabi.SbError, match=what):
            sb.check_status(cuda_device)
        for t, old in zip((table, lens, refs), before):
            assert torch.equal(t, old)

    for more in (2 ** 31 - 1, 2 ** 31 - 10, 2 ** 31 - 11, LONGEST - 9):
        extend(ints(more, 2 * page, 1), "length")
    extend(2 ** 31 - 1, "length")
    extend(ints(LONGEST - 10, 3, 1))
    assert lens.tolist() == [LONGEST, 8, 1] and int(refs.sum()) == 32768 + 2
    assert table[0, :3].tolist() == [0, 2, 3] and table[0, 32767:].tolist() == [32768, -1, -1]
    assert table[1, :2].tolist() == [1, -1] and table[2, :2].tolist() == [32769, -1]
    extend(1, "length")
    extend(ints(0, 1, 1))


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("attend_current", [False, True])
def test_decode_of_the_longest_sequences(cuda_device, dtype, attend_current):
    """2^31 - 16 tokens, nearly all of them in one page that the row names 32766 times; longer ones are refused."""
    import stickbreaking_attention_b200 as sb
    gen = torch.Generator().manual_seed(61)
    page, d, columns, new = 65536, 8, 32770, 2
    k, v = (torch.randn(3, 1, page, d, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(4, 2, new, d, generator=gen).to(dtype)
    table = torch.zeros(4, columns, dtype=torch.int32)
    table[:, 32766], table[:, 32767] = 1, 2
    lens = torch.tensor([LONGEST, LONGEST + 1, 2 ** 31 - 1, 100], dtype=torch.int32)
    dev = lambda t: t.to(cuda_device)
    kp, vp, tab, lengths = dev(k), dev(v), dev(table), dev(lens)
    newest = torch.randn(4, 1, 1, d, generator=gen).to(dtype)
    with torch.no_grad():
        for refused in (sb.kv_append, None):
            if refused:
                refused(dev(newest[:1]), dev(newest[:1]), kp, vp, tab[:1], lengths[:1])       # of the longest, the last slot but 15
                sb.check_status(cuda_device)
                refused(dev(newest[1:3]), dev(newest[1:3]), kp, vp, tab[1:3], lengths[1:3])
            else:
                o, rem = sb.sb_attn_decode(dev(q), kp, vp, tab, lengths, attend_current=attend_current)
            with pytest.raises(sb._cabi.SbError, match="length"):
                sb.check_status(cuda_device)
    k[2, 0, page - 17], v[2, 0, page - 17] = newest[0, 0, 0], newest[0, 0, 0]
    assert torch.equal(kp.cpu(), k) and torch.equal(vp.cpu(), v)
    assert bool(o[1:3].isnan().all()) and bool(rem[1:3].isnan().all())
    short = torch.tensor([[1, 2], [0, -1]], dtype=torch.int32)              # older keys have no weight left
    want = R.decode(q[[0, 3]], k, v, short, torch.tensor([LONGEST - 32766 * page, 100], dtype=torch.int32), attend_current=attend_current)
    R.check_decode((o[[0, 3]], rem[[0, 3]]), want)


# ---- books and lengths that cannot be --------------------------------------------------------------------------------------

def small_cache(sb, device, lens=(6, 4, 0, 0)):
    """Four sequences, six pages of four tokens; pools with a number for every element."""
    cache = sb.PagedKVCache(2, 6, 1, 4, 8, 4, 16, dtype=FP32, device=device)
    cache.extend(ints(*lens))
    sb.check_status(device)
    for t, at in ((cache.k, 0), (cache.v, 10 ** 6)):
        t.copy_(torch.arange(at, at + t.numel(), dtype=FP32, device=device).view(t.shape))
    return cache


def everything(cache):
    return [t.clone() for t in (cache.page_table, cache.seq_lens, cache.page_refs, cache.k, cache.v)]


def refused(sb, device, cache, call, what):
    """`call` changes nothing and leaves a status."""
    before = everything(cache)
    call()
    with pytest.raises(sb._cabi.SbError, match=what):
        sb.check_status(device)
    for name, t, old in zip(("page_table", "seq_lens", "page_refs", "k", "v"), everything(cache), before):
        assert torch.equal(t, old), name


@gpu
@pytest.mark.parametrize("count", [-1, -2 ** 31])
@pytest.mark.parametrize("page", [0, 2, 5])
def test_compact_refuses_negative_counts(cuda_device, page, count):
    """A page that is neither free nor in use: where there are such, fewer pages in front are free than pages behind are in use."""
    import stickbreaking_attention_b200 as sb
    cache = small_cache(sb, cuda_device)
    cache.page_refs[page] = count
    refused(sb, cuda_device, cache, cache.compact, "negative")
    cache.page_refs.fill_(-1)
    refused(sb, cuda_device, cache, cache.compact, "negative")


@gpu
def test_compact_of_large_pools_refuses_negative_counts(cuda_device):
    """The last of 40000 pages (the counts are read in more than one turn, 16 at a time, the last ones singly)."""
    import stickbreaking_attention_b200 as sb
    cache = sb.PagedKVCache(1, 40003, 1, 1, 8, 2, 64, dtype=BF16, device=cuda_device)
    cache.k.zero_(), cache.v.zero_()
    cache.extend(ints(20, 30))
    cache.free(ints(0))
    cache.page_refs[-1] = -1
    refused(sb, cuda_device, cache, cache.compact, "negative")
    cache.page_refs[-1] = 0
    cache.compact()
    sb.check_status(cuda_device)
    assert cache.page_table[1, :30].tolist() == [*range(20, 30), *range(20)]
    assert cache.page_refs[:32].tolist() == [1] * 30 + [0] * 2


@gpu
@pytest.mark.parametrize("page", [-1, 6, 2 ** 31 - 1, 5])          # 5: a page of the cache, but a free one
def test_compact_leaves_entries_without_a_place_alone(cuda_device, page):
    import stickbreaking_attention_b200 as sb
    cache = small_cache(sb, cuda_device)
    cache.free(ints(0))
    cache.extend(ints(0, 4, 0, 0))                  # sequence 1 has pages 2 and 0; 2 moves to 1
    cache.page_table[1, 1] = page
    cache.compact()
    with pytest.raises(sb._cabi.SbError, match="page"):
        sb.check_status(cuda_device)
    assert cache.page_table[1].tolist() == [1, page, -1, -1] and cache.page_refs.tolist() == [1, 1, 0, 0, 0, 0]
    assert torch.equal(cache.k[:, 1].cpu(), torch.arange(384, dtype=FP32).view(2, 6, 1, 4, 8)[:, 2])


@gpu
@pytest.mark.parametrize("length", [-1, 17, 2 ** 31 - 1, -2 ** 31])
def test_compact_refuses_lengths_that_cannot_be(cuda_device, length):
    import stickbreaking_attention_b200 as sb
    cache = small_cache(sb, cuda_device)
    cache.free(ints(0))                             # pages 0 and 1 are free: compact has something to do
    cache.seq_lens[3] = length
    refused(sb, cuda_device, cache, cache.compact, "length")
    cache.seq_lens[3] = 0
    cache.compact()
    sb.check_status(cuda_device)
    assert cache.page_table[1].tolist() == [0, -1, -1, -1] and cache.page_refs.tolist() == [1, 0, 0, 0, 0, 0]


@gpu
@pytest.mark.parametrize("length", [-1, 17, 2 ** 31 - 1, -2 ** 31])
def test_free_refuses_lengths_that_cannot_be(cuda_device, length):
    import stickbreaking_attention_b200 as sb
    cache = small_cache(sb, cuda_device)
    cache.seq_lens[3] = length
    for seqs in (ints(3), ints(0, 3), ints(3, 1, 1), ints(*[1] * 300, 3)):
        refused(sb, cuda_device, cache, lambda: cache.free(seqs), "length")
    cache.free(ints(0, 1))                          # the others can be freed
    sb.check_status(cuda_device)
    assert cache.page_refs.tolist() == [0] * 6 and cache.seq_lens.tolist() == [0, 0, 0, length]
    for call in (lambda: cache.extend(ints(1, 1, 0, 0)), lambda: cache.extend(1)):
        refused(sb, cuda_device, cache, call, "length")
    for call in (lambda: cache.fork(ints(3), ints(2)), lambda: cache.fork(ints(0), ints(3))):
        refused(sb, cuda_device, cache, call, "listed")


@gpu
@pytest.mark.parametrize("page", [-1, 6, 2 ** 31 - 1, -2 ** 31, 5, 2])      # 5: a free page; 2: sequence 1's, counted once
@pytest.mark.parametrize("seqs", [[0, 1], [1, 0, 0], [0, 1] * 200])
def test_free_counts_no_page_below_0(cuda_device, page, seqs):
    """Rows that name a page which nobody counts for them: the sequences are empty afterwards, and no count is negative."""
    import stickbreaking_attention_b200 as sb
    cache = small_cache(sb, cuda_device)
    cache.page_table[0, 0] = page                   # page 0 stays counted: nothing names it any more
    cache.free(ints(*seqs))
    with pytest.raises(sb._cabi.SbError, match="page"):
        sb.check_status(cuda_device)
    assert cache.page_refs.tolist() == [1, 0, 0, 0, 0, 0]
    assert cache.seq_lens.tolist() == [0] * 4 and bool((cache.page_table == -1).all())


@gpu
def test_free_of_many_rows_that_name_the_same_page(cuda_device):
    """600 sequences hold a page that 500 of them are counted for."""
    import stickbreaking_attention_b200 as sb
    table = torch.zeros(600, 3, dtype=torch.int32, device=cuda_device)
    lens = torch.full((600,), 3, dtype=torch.int32, device=cuda_device)
    refs = ints(500, 7)
    sb.kv_free(table, lens, refs, torch.arange(600, dtype=torch.int32, device=cuda_device), 4)
    with pytest.raises(sb._cabi.SbError, match="page"):
        sb.check_status(cuda_device)
    assert refs.tolist() == [0, 7] and not bool(lens.any()) and bool((table[:, 0] == -1).all()) and not bool(table[:, 1:].any())


@gpu
@pytest.mark.parametrize("entry", [0, 1])          # a page that would be shared; the last one, partly filled
@pytest.mark.parametrize("page", [-1, 6, 2 ** 31 - 1, -2 ** 31])
def test_fork_of_a_sequence_whose_row_names_no_page(cuda_device, entry, page):
    import stickbreaking_attention_b200 as sb
    cache = small_cache(sb, cuda_device)
    cache.page_table[0, entry] = page
    refused(sb, cuda_device, cache, lambda: cache.fork(ints(1, 0), ints(2, 3)), "page")
    cache.fork(ints(1), ints(2))                    # the other one can be forked
    sb.check_status(cuda_device)
    assert cache.seq_lens.tolist() == [6, 4, 4, 0] and cache.page_refs.tolist() == [1, 1, 2, 0, 0, 0]


@gpu
def test_fork_of_many_long_rows_looks_at_every_entry(cuda_device):
    """40 forks of rows of 70 pages, one bad entry somewhere."""
    import stickbreaking_attention_b200 as sb
    cache = sb.PagedKVCache(1, 6000, 1, 4, 8, 80, 400, dtype=FP32, device=cuda_device)
    cache.k.zero_(), cache.v.zero_()
    cache.extend(ints(*([278] * 40 + [0] * 40)))
    src, dst = ints(*range(39, -1, -1)), ints(*range(40, 80))
    for row, entry in ((0, 0), (39, 69), (17, 31), (17, 32), (8, 68)):
        page = int(cache.page_table[row, entry])
        cache.page_table[row, entry] = 6000
        refused(sb, cuda_device, cache, lambda: cache.fork(src, dst), "page")
        cache.page_table[row, entry] = page
    cache.page_table[5, 70] = 6000                  # behind the row's end: not looked at
    cache.fork(src, dst)
    sb.check_status(cuda_device)
    assert cache.seq_lens.tolist() == [278] * 80 and int(cache.page_refs.sum()) == 80 * 70


@gpu
@pytest.mark.parametrize("n,pages", [(3000, 7), (1300, 150), (65535, 2)])
def test_free_of_thousands_of_sequences(cuda_device, n, pages):
    """More entries than blocks run at a time, many of them twice; then with one that is refused, and with pages counted too few."""
    import stickbreaking_attention_b200 as sb
    gen = torch.Generator().manual_seed(63)
    max_seqs = n - n // 4
    total = max_seqs * pages
    table = torch.randperm(total, generator=gen).int().view(max_seqs, pages).to(cuda_device)
    lens = torch.randint(0, 4 * pages + 1, (max_seqs,), generator=gen, dtype=torch.int32).to(cuda_device)
    held = torch.arange(pages, device=cuda_device)[None] < ((lens + 3) // 4)[:, None]
    refs = torch.zeros(total, dtype=torch.int32, device=cuda_device)
    refs[table[held].long()] = 2                    # somebody else holds them as well
    seqs = torch.cat((torch.randperm(max_seqs, generator=gen), torch.randint(0, max_seqs, (n - max_seqs,), generator=gen)))
    seqs = seqs[torch.randperm(n, generator=gen)].int().to(cuda_device)
    before = [t.clone() for t in (table, lens, refs)]
    bad = seqs.clone()
    bad[n // 2] = max_seqs
    sb.kv_free(table, lens, refs, bad, 4)
    with pytest.raises(sb._cabi.SbError, match="listed"):
        sb.check_status(cuda_device)
    for t, old in zip((table, lens, refs), before):
        assert torch.equal(t, old)
    sb.kv_free(table, lens, refs, seqs, 4)
    sb.check_status(cuda_device)
    assert not bool(lens.any()) and torch.equal(refs, before[2] // 2) and torch.equal(table, torch.where(held, -1, before[0]))
    table.copy_(before[0]), lens.copy_(before[1])
    short = table[held].long()[::97]
    refs[short] = 0
    sb.kv_free(table, lens, refs, seqs, 4)
    with pytest.raises(sb._cabi.SbError, match="page"):
        sb.check_status(cuda_device)
    assert not bool(lens.any()) and not bool(refs.any()) and torch.equal(table, torch.where(held, -1, before[0]))


@gpu
@pytest.mark.parametrize("rows,columns,counts,needed", [(4, 50, [6, 0, 9, 200], 2 + 3 + 50), (3000, 40, [160] * 3000, 120000),
                                                        (3, 2 ** 20, [2 ** 22] * 3, 3 * 2 ** 20), (4, 50, [0, 0, 17, 12], 5 + 3)])
def test_extend_says_how_many_pages_it_needs(cuda_device, rows, columns, counts, needed):
    import stickbreaking_attention_b200 as sb
    table = torch.full((rows, columns), -1, dtype=torch.int32, device=cuda_device)
    lens, refs = torch.zeros(rows, dtype=torch.int32, device=cuda_device), torch.zeros(6, dtype=torch.int32, device=cuda_device)
    sb.kv_extend(table, lens, refs, ints(*counts), 4)
    with pytest.raises(sb._cabi.SbError, match=f" {needed} needed"):
        sb.check_status(cuda_device)
    assert not bool(lens.any()) and not bool(refs.any()) and bool((table == -1).all())


# ---- layouts ---------------------------------------------------------------------------------------------------------------

def layouts(device, dtype=BF16):
    """Queries (2, 4, 3, 64) in many layouts, and whether an output in that layout has unit stride in its last axis."""
    def numbers(*shape):
        return torch.arange(math.prod(shape), dtype=FP32, device=device).remainder(97).sub(48).div(32).to(dtype).view(shape)
    base = numbers(2, 4, 3, 64)
    yield "contiguous", base
    yield "tokens before heads", numbers(2, 3, 4, 64).transpose(1, 2)
    yield "tokens behind columns", numbers(2, 4, 64, 3).transpose(2, 3)
    yield "columns first", numbers(64, 2, 3, 4).permute(1, 3, 2, 0)
    yield "rows at odd elements", numbers(2 * 4 * 3 * 64 + 1)[1:].view(2, 4, 3, 64)
    yield "rows at odd elements, tokens before heads", numbers(2 * 3 * 4 * 64 + 1)[1:].view(2, 3, 4, 64).transpose(1, 2)
    yield "rows of odd length", numbers(2, 4, 3, 65)[..., :64]
    yield "a third of a packed projection", numbers(2, 3, 3, 4, 64)[:, :, 1].transpose(1, 2)
    yield "one batch element", numbers(1, 4, 3, 64).expand(2, -1, -1, -1)
    yield "one head", numbers(2, 1, 3, 64).expand(-1, 4, -1, -1)
    yield "one column", numbers(2, 4, 3, 1).expand(-1, -1, -1, 64)
    yield "one column, tokens before heads", numbers(2, 3, 4, 1).transpose(1, 2).expand(-1, -1, -1, 64)
    yield "windows", numbers(2, 4, 66).unfold(2, 64, 1)
    yield "every other column", numbers(2, 4, 3, 128)[..., ::2]


def announced(q, *args):
    """Strides of (o, rem) as the operator without data gives them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from stickbreaking_attention_b200 import ops
    with FakeTensorMode() as mode:
        def fake(t):
            size = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
            return torch.empty(t.storage_offset() + size, dtype=t.dtype, device="cuda").as_strided(t.shape, t.stride(), t.storage_offset())
        return tuple(t.stride() for t in ops.decode_op(fake(q), *(fake(t) for t in args), 0.125, False))


def cache_of(gen, dtype=BF16):
    return R.make_cache(gen, [40, 9], 2, 16, 64, dtype)


def test_decode_announces_rows_without_gaps():
    """Strides that compiled code goes by: those of the queries where rows are runs of elements, contiguous else."""
    cache = cache_of(torch.Generator().manual_seed(70))
    got = {name: announced(q, *cache) for name, q in layouts("cpu")}
    assert all(o[3] == 1 and rem == (12, 3, 1) for o, rem in got.values())
    contiguous, turned = (768, 192, 64, 1), (768, 64, 256, 1)
    for name in ("contiguous", "tokens behind columns", "columns first", "rows at odd elements", "rows of odd length", "one column", "windows"):
        assert got[name][0] == contiguous, name
    for name in ("tokens before heads", "rows at odd elements, tokens before heads", "a third of a packed projection"):
        assert got[name][0] == turned, name


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_decode_gives_the_layout_that_it_announces(cuda_device, dtype):
    import stickbreaking_attention_b200 as sb
    cache = cache_of(torch.Generator().manual_seed(71), dtype)
    on_gpu = [t.to(cuda_device) for t in cache]
    for name, q in layouts(cuda_device, dtype):
        with torch.no_grad():
            o, rem = sb.sb_attn_decode(q, *on_gpu)
        sb.check_status(cuda_device)
        assert (o.stride(), rem.stride()) == announced(q, *cache), name
        R.check_decode((o, rem), R.decode(q.contiguous(), *cache))


@gpu
def test_decode_compiled_with_queries_in_many_layouts(cuda_device):
    """Compiled code and eager code agree on what o holds where."""
    import stickbreaking_attention_b200 as sb
    cache = [t.to(cuda_device) for t in cache_of(torch.Generator().manual_seed(72))]

    def step(q):
        o, rem = sb.sb_attn_decode(q, *cache)
        return o.transpose(1, 2).reshape(6, -1) * 2, rem + 1

    with torch.no_grad():
        for name, q in layouts(cuda_device):
            torch.compiler.reset()
            # (code kept on the disk may be for another build's layouts)
            with torch.compiler.config.patch(force_disable_caches=True):
                eager, compiled = step(q), torch.compile(step, fullgraph=True)(q)
            assert torch.equal(eager[0], compiled[0]) and torch.equal(eager[1], compiled[1]), name
    sb.check_status(cuda_device)


# ---- which kernel ----------------------------------------------------------------------------------------------------------

@gpu
def test_decode_takes_the_tensor_cores_where_rows_are_whole_chunks(cuda_device):
    """What sb_attn_decode_path answers, and which kernels are launched."""
    import stickbreaking_attention_b200 as sb
    from stickbreaking_attention_b200 import _cabi
    lib = _cabi.load()
    simt, tensor_cores = 0, 1

    def path(dtype, d, flags=0, offset=0, odd_query=0, stride=None):
        at = 1 << 20
        p = _cabi.SbDecodeParams(struct_bytes=ctypes.sizeof(_cabi.SbDecodeParams), dtype=dtype, batch=2, heads=4, kv_heads=2, new_tokens=1,
                                 head_dim=d, page_size=16, num_pages=8, max_pages=4, logit_scale=0.125, flags=flags)
        p.q = _cabi.SbTensor(at + odd_query, 4 * d, d, d)
        p.k = p.v = _cabi.SbCache(at + offset, 0, 32 * d, 16 * d, stride or d)
        return lib.sb_attn_decode_path(p)

    with torch.cuda.device(cuda_device):
        for dtype in (1, 2):
            assert [path(dtype, d) for d in (8, 64, 72, 128, 256)] == [tensor_cores] * 5
            assert [path(dtype, d) for d in (1, 50, 100)] == [simt] * 3
            assert path(dtype, 64, offset=8) == path(dtype, 64, stride=68) == path(dtype, 64, odd_query=2) == simt
            assert path(dtype, 64, flags=_cabi.SB_FLAG_FORCE_SIMT) == simt
        assert path(0, 64) == simt and path(1, 257) == path(9, 64) == -1

    gen = torch.Generator().manual_seed(73)
    cache = [t.to(cuda_device) for t in cache_of(gen)]
    q = torch.randn(2, 4, 1, 64, generator=gen).to(BF16).to(cuda_device)
    wide = torch.full((2, *cache[0].shape[:-1], 68), float("nan"), dtype=BF16, device=cuda_device)
    wide[0, ..., :64], wide[1, ..., :64] = cache[0], cache[1]

    def ran(call):
        with torch.no_grad(), torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as profile:
            call()
            torch.cuda.synchronize()
        names = [event.name for event in profile.events() if "decode_" in event.name]
        return {kernel for kernel in ("decode_tc_kernel", "decode_simt_kernel") if any(kernel in name for name in names)}

    def on_cuda_cores():
        with sb.force_simt():
            sb.sb_attn_decode(q, *cache)

    assert ran(lambda: sb.sb_attn_decode(q, *cache)) == {"decode_tc_kernel"}
    assert ran(on_cuda_cores) == {"decode_simt_kernel"}
    assert ran(lambda: sb.sb_attn_decode(q, wide[0, ..., :64], wide[1, ..., :64], *cache[2:])) == {"decode_simt_kernel"}
    sb.check_status(cuda_device)
