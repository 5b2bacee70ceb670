"""The serving operators: attention of new tokens over a paged cache, the write into its pages, their keeping."""
import ctypes
import math
import random

import pytest
import torch

import helpers as H
import serving_reference as R

gpu = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def run_decode(sb, device, q, cache, **kw):
    with torch.no_grad():
        out = sb.sb_attn_decode(q.to(device), *(t.to(device) for t in cache), **kw)
    sb.check_status(device)
    return out


def make(seed, lens, heads, kv_heads, d, page, dtype, new=1, shift=0.0, **kw):
    gen = torch.Generator().manual_seed(seed)
    cache = R.make_cache(gen, lens, kv_heads, page, d, dtype, shift=shift, **kw)
    q = (torch.randn(len(lens), heads, new, d, generator=gen) + shift).to(dtype)
    return q, cache


# ---- attention ----------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("attend_current", [False, True])
@pytest.mark.parametrize("heads,kv_heads,new", [(1, 1, 1), (6, 2, 1), (8, 1, 1), (4, 2, 3), (24, 2, 1), (10, 2, 7)])
def test_decode_short_lengths(cuda_device, dtype, attend_current, heads, kv_heads, new):
    import stickbreaking_attention_b200 as sb
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 130, 257]
    q, cache = make(1, lens, heads, kv_heads, 64, 16, dtype, new)
    got = run_decode(sb, cuda_device, q, cache, attend_current=attend_current)
    R.check_decode(got, R.decode(q, *cache, attend_current=attend_current))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("d", [1, 8, 50, 64, 72, 96, 100, 128, 136, 256])
@pytest.mark.parametrize("page", [1, 7, 24, 64, 256])
def test_decode_head_sizes_and_pages(cuda_device, dtype, d, page):
    import stickbreaking_attention_b200 as sb
    q, cache = make(2, [300, 77, 1], 4, 2, d, page, dtype, shift=0.3)
    R.check_decode(run_decode(sb, cuda_device, q, cache), R.decode(q, *cache))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("heads,kv_heads,new", [(2, 2, 1), (8, 1, 1), (6, 1, 4)])
def test_decode_long_contexts_whose_stick_lasts(cuda_device, dtype, heads, kv_heads, new):
    import stickbreaking_attention_b200 as sb
    lens = [20011, 5000, 9]
    shift = math.sqrt((math.log(20011) + 0.5) / 7)          # scores around -log(length): every key has a weight
    q, cache = make(3, lens, heads, kv_heads, 64, 32, dtype, new, shift=shift)
    R.check_decode(run_decode(sb, cuda_device, q, cache, attend_current=True), R.decode(q, *cache, attend_current=True))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_decode_many_sequences(cuda_device, dtype):
    import stickbreaking_attention_b200 as sb
    rng = random.Random(4)
    lens = [rng.choice([0, 1, 5, 40, 100, 170]) for _ in range(700)]
    q, cache = make(4, lens, 2, 1, 64, 16, dtype, shift=0.5)
    R.check_decode(run_decode(sb, cuda_device, q, cache), R.decode(q, *cache))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("inv_temp", [0.0, 3.0, -2.0])
def test_decode_scales_and_large_scores(cuda_device, dtype, inv_temp):
    """Scores of up to some hundred in size: sticks used up at once, and keys that break nothing off."""
    import stickbreaking_attention_b200 as sb
    q, cache = make(5, [400, 65], 4, 2, 64, 16, dtype)
    R.check_decode(run_decode(sb, cuda_device, q, cache, inv_temp=inv_temp), R.decode(q, *cache, scale=inv_temp))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_decode_infinite_scores(cuda_device, dtype):
    """A key that takes the whole stick (score +inf) and keys that take nothing (-inf): no NaN comes of it."""
    import stickbreaking_attention_b200 as sb
    lens, d, page = [100], 64, 16
    q, (k, v, table, lengths) = make(6, lens, 1, 1, d, page, dtype)
    q[..., 0] = 1.0
    def key(pos): return table[0, pos // page].long(), 0, pos % page
    for pos in (99 - 1, 70, 30):
        k[key(pos)][0] = float("-inf")
    got = run_decode(sb, cuda_device, q, (k, v, table, lengths))
    k2 = k.clone()
    k2[k2 == float("-inf")] = -30000.0                                  # a score of -3750: a weight of 0 as well
    R.check_decode(got, R.decode(q, k2, v, table, lengths))
    k[key(50)][0] = float("inf")
    o, rem = run_decode(sb, cuda_device, q, (k, v, table, lengths))
    k2 = k.clone()
    k2[k2 == float("-inf")] = -30000.0
    k2[k2 == float("inf")] = 30000.0
    R.check_decode((o, rem), R.decode(q, k2, v, table, lengths))
    assert float(rem.max()) == 0.0


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("heads,new", [(2, 5), (12, 9)])
@pytest.mark.parametrize("length", [100, 113, 131])
def test_decode_keys_that_a_row_does_not_attend_to(cuda_device, dtype, heads, new, length):
    """Keys and values of the newest tokens that are no numbers: they show in the rows that attend to them and in no other."""
    import stickbreaking_attention_b200 as sb
    q, (k, v, table, lens) = make(15, [length, 40], heads, 2, 64, 16, dtype, new=new)
    for bad in (2, 4):                                        # the token from which on rows see it (keys before a query)
        k2, v2 = k.clone(), v.clone()
        pos = length - new + bad - 1
        at = table[0, pos // 16].long()
        k2[at, 0, pos % 16] = float("nan")
        v2[at, 1, pos % 16] = float("inf")
        o, rem = run_decode(sb, cuda_device, q, (k2, v2, table, lens))
        half = heads // 2
        assert not bool(torch.isfinite(o[0, :, bad:]).any(-1)[:half].any()) and bool(rem[0, :half, bad:].isnan().all())
        assert not bool(torch.isfinite(o[0, half:, bad:]).any())
        fine = lambda t: t[:, :, :bad]
        R.check_decode((fine(o), fine(rem)), R.decode(fine(q), k, v, table, lens - (new - bad)))


@gpu
def test_decode_padded_batch(cuda_device):
    """More new tokens than a sequence has: rows in front of it, and empty sequences, give o = 0, rem = 1."""
    import stickbreaking_attention_b200 as sb
    q, cache = make(7, [0, 2, 4, 90], 4, 2, 64, 16, BF16, new=5)
    o, rem = run_decode(sb, cuda_device, q, cache)
    R.check_decode((o, rem), R.decode(q, *cache))
    assert bool((o[0] == 0).all()) and bool((rem[0] == 1).all())
    assert bool((o[1, :, :4] == 0).all()) and bool((rem[1, :, :4] == 1).all())


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_decode_strides(cuda_device, dtype):
    """Token-major caches and queries as permuted views, a cache inside a larger tensor, rows that are not 16-byte aligned."""
    import stickbreaking_attention_b200 as sb
    q, (k, v, table, lens) = make(8, [130, 3, 257], 4, 2, 64, 16, dtype, new=2)
    want = R.decode(q, k, v, table, lens)
    dev = lambda t: t.to(cuda_device)
    q_view = dev(q).transpose(1, 2).contiguous().transpose(1, 2)
    token_major = [dev(t).transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    wide = torch.full((2, *k.shape[:-1], 130), float("nan"), dtype=dtype, device=cuda_device)
    wide[0, ..., 3:67], wide[1, ..., 8:72] = dev(k), dev(v)
    both = torch.stack((dev(k), dev(v)), 1)
    with torch.no_grad():
        for kk, vv in (token_major, (wide[0, ..., 3:67], wide[1, ..., 8:72]), (both[:, 0], both[:, 1])):
            table_view = torch.full((3, 40), -7, dtype=torch.int32, device=cuda_device)
            table_view[:, 5:5 + table.shape[1]] = dev(table)
            got = sb.sb_attn_decode(q_view, kk, vv, table_view[:, 5:5 + table.shape[1]], dev(lens))
            assert got[0].stride() == q_view.stride()
            sb.check_status(cuda_device)
            R.check_decode(got, want)
        got = sb.sb_attn_decode(dev(q)[..., :1].expand(q.shape), *token_major, dev(table), dev(lens))
        R.check_decode(got, R.decode(q[..., :1].expand(q.shape).contiguous(), k, v, table, lens))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_decode_refused_lengths_and_pages(cuda_device, dtype):
    """What cannot be gives NaN and a status; the other sequences are computed."""
    import stickbreaking_attention_b200 as sb
    q, (k, v, table, lens) = make(9, [100, 50, 70, 200], 2, 1, 64, 16, dtype)
    want = R.decode(q, k, v, table, lens)
    dev = [t.to(cuda_device) for t in (q, k, v)]
    bad_lens = lens.clone()
    bad_lens[1], bad_lens[2] = -1, table.shape[1] * 16 + 1
    with torch.no_grad():
        o, rem = sb.sb_attn_decode(*dev, table.to(cuda_device), bad_lens.to(cuda_device))
    with pytest.raises(sb._cabi.SbError, match="length"):
        sb.check_status(cuda_device)
    assert bool(o[1:3].isnan().all()) and bool(rem[1:3].isnan().all())
    pick = lambda x: x[[0, 3]]
    R.check_decode((pick(o), pick(rem)), tuple(pick(t) for t in want))
    for page in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        bad_table = table.clone()
        bad_table[2, 4] = page                                  # the newest page of sequence 2
        with torch.no_grad():
            o, rem = sb.sb_attn_decode(*dev, bad_table.to(cuda_device), lens.to(cuda_device))
        with pytest.raises(sb._cabi.SbError, match="page"):
            sb.check_status(cuda_device)
        assert bool(o[2].isnan().all()) and bool(rem[2].isnan().all())
        pick = lambda x: x[[0, 1, 3]]
        R.check_decode((pick(o), pick(rem)), tuple(pick(t) for t in want))
    sb.check_status(cuda_device)


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_decode_dense_row_pass_and_cuda_cores(cuda_device, dtype):
    """Every key visited, or the ones behind the used-up stick left out: same bits.  CUDA cores: the same to rounding."""
    import stickbreaking_attention_b200 as sb
    q, cache = make(10, [3000, 700], 8, 2, 64, 16, dtype)
    got = run_decode(sb, cuda_device, q, cache)
    with sb.dense_row_pass():
        dense = run_decode(sb, cuda_device, q, cache)
    assert torch.equal(got[0], dense[0]) and torch.equal(got[1], dense[1])
    with sb.force_simt():
        R.check_decode(run_decode(sb, cuda_device, q, cache), R.decode(q, *cache))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_decode_repeats_bit_for_bit_and_on_other_streams(cuda_device, dtype):
    import stickbreaking_attention_b200 as sb
    q, cache = make(11, [4000, 33, 900], 8, 2, 64, 16, dtype, shift=0.8)
    args = [t.to(cuda_device) for t in (q, *cache)]
    with torch.no_grad():
        first = sb.sb_attn_decode(*args)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        out = []
        for i in range(12):
            with torch.cuda.stream(streams[i % 3]):
                out.append(sb.sb_attn_decode(*args))
        torch.cuda.synchronize()
    for o, rem in out:
        assert torch.equal(o, first[0]) and torch.equal(rem, first[1])


@gpu
def test_decode_and_append_in_a_captured_step(cuda_device):
    """extend, append and attend captured once and replayed: the lengths grow on the device."""
    import stickbreaking_attention_b200 as sb
    page, steps, d = 16, 40, 64
    lens = [5, 0, 30]
    cache = sb.PagedKVCache(1, 40, 2, page, d, 3, 128, dtype=BF16, device=cuda_device)
    counts = torch.tensor([1, 1, 1], dtype=torch.int32, device=cuda_device)
    gen = torch.Generator().manual_seed(12)
    k, v = (torch.randn(3, 2, max(lens), d, generator=gen).to(BF16).to(cuda_device) for _ in range(2))
    ks, vs, qs = (torch.randn(steps, 3, h, 1, d, generator=gen).to(BF16).to(cuda_device) for h in (2, 2, 4))
    with torch.no_grad():
        cache.extend(torch.tensor(lens, dtype=torch.int32, device=cuda_device))
        cache.append(0, k, v)
        q_in, k_in, v_in = torch.empty_like(qs[0]), torch.empty_like(ks[0]), torch.empty_like(vs[0])

        def step():
            cache.extend(counts)
            cache.append(0, k_in, v_in)
            return cache.attend(0, q_in)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        saved = [t.clone() for t in (cache.page_table, cache.seq_lens, cache.page_refs)]
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        for t, old in zip((cache.page_table, cache.seq_lens, cache.page_refs), saved):
            t.copy_(old)
        with torch.cuda.graph(graph):
            o, rem = step()
        for i in range(steps):
            q_in.copy_(qs[i]); k_in.copy_(ks[i]); v_in.copy_(vs[i])
            graph.replay()
            if i in (0, 17, steps - 1):
                sb.check_status(cuda_device)
                assert cache.seq_lens.tolist() == [n + i + 1 for n in lens]
                R.check_decode((o, rem), R.decode(qs[i], cache.k[0], cache.v[0], cache.page_table, cache.seq_lens))


@gpu
def test_decode_pools_beyond_32_bit_offsets(cuda_device):
    """A pool of 2.7e9 elements, its last pages in use."""
    import stickbreaking_attention_b200 as sb
    pages, kv, page, d = 20600, 16, 64, 128
    pool = torch.empty(pages, kv, page, d, dtype=BF16, device=cuda_device)
    pool[-8:].normal_(generator=torch.Generator(device=cuda_device).manual_seed(13))
    table = torch.arange(pages - 1, pages - 9, -1, dtype=torch.int32, device=cuda_device)[None]
    lens = torch.tensor([500], dtype=torch.int32, device=cuda_device)
    q = torch.randn(1, kv, 1, d, device=cuda_device).to(BF16)
    with torch.no_grad():
        got = sb.sb_attn_decode(q, pool, pool, table, lens)
        small = pool[-8:].cpu()
        R.check_decode(got, R.decode(q, small, small, table.cpu() - (pages - 8), lens))
        new = torch.randn(1, kv, 3, d, device=cuda_device).to(BF16)
        sb.kv_append(new, new, pool, pool, table, lens)
        got = torch.stack([pool[table[0, p // page].long(), :, p % page] for p in (497, 498, 499)], 1)
    assert torch.equal(got, new[0])
    sb.check_status(cuda_device)


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_decode_as_many_new_tokens_as_keys(cuda_device, dtype):
    """Up to 1024 new tokens, in many blocks of rows, some in front of their sequences."""
    import stickbreaking_attention_b200 as sb
    lens, d, page = [1024, 150, 0, 1030], 8, 16
    q, cache = make(16, lens, 2, 1, d, page, dtype, new=1024, shift=0.5)
    got = run_decode(sb, cuda_device, q, cache)
    gen = torch.Generator().manual_seed(17)
    some = sorted({0, 1, 5, 15, 16, 17, 873, 874, 875, 1022, 1023, *torch.randint(0, 1024, (12,), generator=gen).tolist()})
    for t in some:                                       # token t is the last of a batch that ends with it
        ends = (cache[3] - 1023 + t).clamp(min=0).int()
        want = R.decode(q[:, :, t:t + 1], *cache[:3], ends)
        R.check_decode((got[0][:, :, t:t + 1], got[1][:, :, t:t + 1]), want)


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_decode_tables_of_enormous_capacity(cuda_device, dtype):
    """1024 sequences with room for 39 million tokens each: more tiles than 31 bits count, if all of them were in use."""
    import stickbreaking_attention_b200 as sb
    gen = torch.Generator().manual_seed(18)
    batch, page, d = 1024, 65536, 8
    k, v = (torch.randn(2, 1, page, d, generator=gen).to(dtype) for _ in range(2))
    table = torch.full((batch, 600), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(batch) % 2                # pages may be shared by any number of readers
    lens = torch.randint(0, 200, (batch,), generator=gen, dtype=torch.int32)
    lens[7], lens[500] = 4000, 65536
    q = torch.randn(batch, 1, 1, d, generator=gen).to(dtype)
    R.check_decode(run_decode(sb, cuda_device, q, (k, v, table, lens)), R.decode(q, k, v, table, lens))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_two_captured_graphs_at_once(cuda_device, dtype):
    """Two graphs with an attention each, replayed on two streams at the same time: neither uses the other's scratch."""
    import stickbreaking_attention_b200 as sb
    sets = []
    with torch.no_grad():
        for seed, lens in ((19, [9000, 40]), (20, [300, 7000, 1])):
            q, cache = make(seed, lens, 8, 2, 64, 16, dtype, shift=0.8)
            args = [t.to(cuda_device) for t in (q, *cache)]
            want = sb.sb_attn_decode(*args)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = [sb.sb_attn_decode(*args) for _ in range(5)]
            sets.append((graph, out, want, torch.cuda.Stream(), args))     # (the graph reads the inputs where they are)
        for _ in range(4):
            for graph, _, _, stream, _ in sets:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
    for _, out, want, _, _ in sets:
        for o, rem in out:
            assert torch.equal(o, want[0]) and torch.equal(rem, want[1])


@gpu
@pytest.mark.parametrize("dtype,d", [(FP32, 64), (BF16, 128), (FP16, 64), (BF16, 50)])
def test_decode_gives_the_rows_of_the_whole_attention(cuda_device, dtype, d):
    import stickbreaking_attention_b200 as sb
    lens, heads, page = [300, 17, 129], 3, 16
    gen = torch.Generator().manual_seed(14)
    q, k, v = (torch.randn(heads, sum(lens), d, generator=gen).to(dtype).to(cuda_device) for _ in range(3))
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(cuda_device)
    cache = sb.PagedKVCache(1, 40, heads, page, d, 3, 320, dtype=dtype, device=cuda_device)
    with torch.no_grad():
        o, rem = sb.sb_attn_varlen(q, k, v, cu, max(lens))
        cache.extend((cu[1:] - cu[:-1]).int())
        cache.append(0, k, v, cu)
        last = (cu[1:] - 1).long()
        got_o, got_rem = cache.attend(0, q[:, last].transpose(0, 1)[:, :, None])
    sb.check_status(cuda_device)
    tol = H.TOL[dtype]["out"]
    assert H.max_abs(got_o[:, :, 0], o[:, last].transpose(0, 1)) <= tol
    assert H.max_abs(got_rem[:, :, 0], rem[:, last].transpose(0, 1)) <= tol


# ---- append -------------------------------------------------------------------------------------------------------------

def expect_append(k, v, cache, rows):
    """`rows`: (sequence, position, row of k and v as (kv_heads, d))."""
    kp, vp, table, _ = (t.clone() for t in cache)
    page = kp.shape[2]
    for seq, pos, kr, vr in rows:
        if pos >= 0:
            at = int(table[seq, pos // page])
            kp[at, :, pos % page], vp[at, :, pos % page] = kr, vr
    return kp, vp


def same(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("d,page,new", [(64, 16, 1), (128, 24, 5), (50, 7, 3), (1, 1, 2), (72, 64, 70)])
def test_append_steps(cuda_device, dtype, d, page, new):
    import stickbreaking_attention_b200 as sb
    lens, kv = [0, 1, 64, 200, 71], 3
    gen = torch.Generator().manual_seed(20)
    cache = R.make_cache(gen, lens, kv, page, d, dtype)
    k, v = (torch.randn(len(lens), kv, new, d, generator=gen).to(dtype) for _ in range(2))
    want = expect_append(k, v, cache, [(b, n - new + t, k[b, :, t], v[b, :, t]) for b, n in enumerate(lens) for t in range(new)])
    for view in (lambda t: t, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        kp, vp, table, lengths = (t.to(cuda_device) for t in cache)
        sb.kv_append(view(k.to(cuda_device)), view(v.to(cuda_device)), kp, vp, table, lengths)
        sb.check_status(cuda_device)
        assert same(kp, want[0]) and same(vp, want[1])


@gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("cu_dtype,zero_start", [(torch.int32, True), (torch.int64, False)])
def test_append_packed(cuda_device, dtype, cu_dtype, zero_start):
    """Prompts packed with ragged lengths, one of them empty, onto sequences that hold something already; tokens behind the end."""
    import stickbreaking_attention_b200 as sb
    lens, new, kv, d, page = [40, 0, 100, 9, 33], [40, 0, 60, 12, 1], 2, 64, 16
    gen = torch.Generator().manual_seed(21)
    cache = R.make_cache(gen, lens, kv, page, d, dtype)
    k, v = (torch.randn(sum(new) + 5, kv, d, generator=gen).to(dtype).transpose(0, 1) for _ in range(2))
    ends = torch.tensor(([0] if zero_start else []) + torch.tensor(new).cumsum(0).tolist(), dtype=cu_dtype)
    rows, at = [], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        rows += [(b, n - m + t, k[:, at + t], v[:, at + t]) for t in range(m)]
        at += m
    want = expect_append(k, v, cache, rows)
    kp, vp, table, lengths = (t.to(cuda_device) for t in cache)
    sb.kv_append(k.to(cuda_device), v.to(cuda_device), kp, vp, table, lengths, ends.to(cuda_device), zero_start=zero_start)
    sb.check_status(cuda_device)
    assert same(kp, want[0]) and same(vp, want[1])


@gpu
def test_append_large_pool_of_tokens_and_views(cuda_device):
    """Many tokens per block, a cache whose pages are token-major, one that is not 16-byte aligned."""
    import stickbreaking_attention_b200 as sb
    lens, kv, d, page = [4000, 17, 2500, 1, 801], 4, 64, 32
    gen = torch.Generator().manual_seed(22)
    kp, vp, table, lengths = R.make_cache(gen, lens, kv, page, d, BF16, poison=False)
    k, v = (torch.randn(kv, sum(lens), d, generator=gen).to(BF16) for _ in range(2))
    ends = torch.tensor(lens).cumsum(0)
    rows, at = [], 0
    for b, n in enumerate(lens):
        rows += [(b, t, k[:, at + t], v[:, at + t]) for t in range(n)]
        at += n
    want = expect_append(k, v, (kp, vp, table, lengths), rows)
    dev = lambda t: t.to(cuda_device)
    shape = (*kp.shape[:-1], d + 1)
    caches = [(dev(kp), dev(vp)), tuple(dev(t).transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp)),
              tuple(torch.zeros(shape, dtype=BF16, device=cuda_device)[..., 1:] for _ in range(2))]
    for ck, cv in caches:
        ck.copy_(kp), cv.copy_(vp)
        sb.kv_append(dev(k), dev(v), ck, cv, dev(table), dev(lengths), dev(ends), zero_start=False)
        sb.check_status(cuda_device)
        assert same(ck.contiguous(), want[0]) and same(cv.contiguous(), want[1])


@gpu
def test_append_many_small_tokens(cuda_device):
    """400000 tokens of one head and 8 columns: blocks of 64 tokens."""
    import stickbreaking_attention_b200 as sb
    page, lens = 64, [150000, 1, 249999]
    gen = torch.Generator().manual_seed(24)
    pages = sum(-(-n // page) for n in lens)
    order = torch.randperm(pages, generator=gen).int()
    table = torch.full((3, 4000), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        count = -(-n // page)
        table[b, :count] = order[at:at + count]
        at += count
    k, v = (torch.randn(1, sum(lens), 8, generator=gen).to(BF16).to(cuda_device) for _ in range(2))
    kp, vp = (torch.zeros(pages, 1, page, 8, dtype=BF16, device=cuda_device) for _ in range(2))
    cu = torch.tensor([0] + lens).cumsum(0).to(cuda_device)
    sb.kv_append(k, v, kp, vp, table.to(cuda_device), torch.tensor(lens, dtype=torch.int32, device=cuda_device), cu)
    sb.check_status(cuda_device)
    for b, n in enumerate(lens):
        rows = table[b, : -(-n // page)].long().to(cuda_device)
        for pool, new in ((kp, k), (vp, v)):
            assert torch.equal(pool[rows, 0].flatten(0, 1)[:n], new[0, int(cu[b]):int(cu[b + 1])])
            assert bool((pool[rows, 0].flatten(0, 1)[n:] == 0).all())


@gpu
def test_append_refused_on_the_device(cuda_device):
    """A bad cu_seqlens: nothing is written.  A bad length or page: that token is not."""
    import stickbreaking_attention_b200 as sb
    lens, kv, d, page = [20, 40], 2, 64, 16
    gen = torch.Generator().manual_seed(23)
    cache = R.make_cache(gen, lens, kv, page, d, BF16)
    k = torch.randn(kv, 30, d, generator=gen).to(BF16)
    dev = lambda t: t.to(cuda_device)
    for ends, zero in (([20, 10], False), ([20, 31], False), ([-1, 10], False), ([1, 5, 30], True)):
        kp, vp, table, lengths = (dev(t) for t in cache)
        sb.kv_append(dev(k), dev(k), kp, vp, table, lengths, torch.tensor(ends, device=cuda_device), zero_start=zero)
        with pytest.raises(sb._cabi.SbError, match="cu_seqlens"):
            sb.check_status(cuda_device)
        assert same(kp, cache[0]) and same(vp, cache[1])
    new = torch.randn(2, kv, 3, d, generator=gen).to(BF16)
    for change, what in ((("table", 0, 1, cache[0].shape[0]), "page"), (("table", 0, 1, -5), "page"), (("lens", 0, None, 10 ** 6), "length")):
        kp, vp, table, lengths = (t.clone() for t in cache)
        if change[0] == "table":
            table[change[1], change[2]] = change[3]
        else:
            lengths[change[1]] = change[3]
        want = expect_append(new, new, (kp, vp, cache[2], lengths), [(1, 37 + t, new[1, :, t], new[1, :, t]) for t in range(3)])
        kp, vp, table, lengths = (dev(t) for t in (kp, vp, table, lengths))
        sb.kv_append(dev(new), dev(new), kp, vp, table, lengths)
        with pytest.raises(sb._cabi.SbError, match=what):
            sb.check_status(cuda_device)
        assert same(kp, want[0]) and same(vp, want[1])


# ---- the keeping of the pages ---------------------------------------------------------------------------------------------

def books_equal(cache, books):
    assert cache.seq_lens.tolist() == books.lens
    assert cache.page_refs.tolist() == books.refs
    assert torch.equal(cache.page_table.cpu(), books.table())


@gpu
@pytest.mark.parametrize("page,max_seqs,num_pages,seed", [(1, 5, 30, 0), (4, 9, 40, 1), (16, 40, 300, 2), (7, 1500, 4000, 3), (16, 3, 70000, 4)])
def test_pages_random_programs(cuda_device, page, max_seqs, num_pages, seed):
    """Random sequences of all keeping operators against the books kept in Python; refused ones change nothing."""
    import stickbreaking_attention_b200 as sb
    rng = random.Random(seed)
    layers, kv, d, max_pages = 2, 2, 4, 12
    cache = sb.PagedKVCache(layers, num_pages, kv, page, d, max_seqs, max_pages * page, dtype=FP32, device=cuda_device)
    books = R.Books(max_seqs, max_pages, num_pages, page)
    stamp, refused = 0, 0
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    for step in range(60):
        what = rng.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        before = list(books.lens)
        if what == "extend":
            counts = [rng.choice([0, 0, 1, page, rng.randint(0, 3 * page)]) for _ in range(max_seqs)]
            if rng.random() < 0.05:
                counts[rng.randrange(max_seqs)] = -1
            if rng.random() < 0.2:
                ok = books.extend(1)
                cache.extend(1)
            else:
                ok = books.extend(torch.tensor(counts))
                cache.extend(ints(counts))
            for seq in range(max_seqs):
                for pos in range(before[seq], books.lens[seq]):
                    stamp += 1
                    books.write(seq, pos, stamp)
            grown = [n - m for n, m in zip(books.lens, before)]
            if ok and sum(grown):
                values = ints([books.data[books.rows[s][i // page], i % page] for s in range(max_seqs) for i in range(before[s], books.lens[s])])
                cu = ints([0] + torch.tensor(grown).cumsum(0).tolist())
                for layer in range(layers):
                    x = (values + 0.5 * layer).float()[None, :, None].expand(kv, -1, d)
                    cache.append(layer, x, -x, cu)
        elif what == "fork":
            empty = [s for s in range(max_seqs) if books.lens[s] == 0]
            n = rng.randint(0, min(4, len(empty)))
            dst = rng.sample(empty, n)
            src = [rng.randrange(max_seqs) for _ in range(n)]
            if rng.random() < 0.1 and n:
                src[0] = rng.choice([-1, max_seqs])
            ok = books.fork(src, dst)
            cache.fork(ints(src), ints(dst))
        elif what == "free":
            seqs = [rng.randrange(max_seqs) for _ in range(rng.randint(0, max(1, max_seqs // 3)))]
            if rng.random() < 0.1:
                seqs.append(max_seqs)
            ok = books.free(seqs)
            cache.free(ints(seqs))
        else:
            ok = True
            books.compact()
            cache.compact()
        if ok:
            sb.check_status(cuda_device)
        else:
            refused += 1
            with pytest.raises(sb._cabi.SbError):
                sb.check_status(cuda_device)
        books_equal(cache, books)
        if step % 10 == 9:
            k, v = cache.k.cpu(), cache.v.cpu()
            for s in range(max_seqs):
                at = torch.tensor([books.rows[s][i // page] * page + i % page for i in range(books.lens[s])], dtype=torch.long)
                want = torch.tensor(books.tokens(s), dtype=torch.float32)
                for layer in range(layers):
                    got = k[layer].transpose(1, 2).flatten(0, 1)[at]
                    assert bool((got == (want + 0.5 * layer)[:, None, None]).all())
                    assert bool((v[layer].transpose(1, 2).flatten(0, 1)[at] == -(want + 0.5 * layer)[:, None, None]).all())


@gpu
def test_pages_of_many_sequences(cuda_device):
    """Books too long for shared memory: 6000 sequences, 2600 forks in one call, a sequence of 5000 pages."""
    import stickbreaking_attention_b200 as sb
    page, max_seqs, num_pages, max_pages = 4, 6000, 20000, 5200
    cache = sb.PagedKVCache(1, num_pages, 1, page, 8, max_seqs, max_pages * page, dtype=BF16, device=cuda_device)
    books = R.Books(max_seqs, max_pages, num_pages, page)
    rng = random.Random(31)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    counts = [rng.randint(0, 9) if s < 2600 else 0 for s in range(max_seqs)]
    counts[17] = 20000
    src = list(range(2600))
    rng.shuffle(src)
    dst = list(range(3000, 5600))
    gone = [rng.randrange(max_seqs) for _ in range(3000)]

    def step(ok, call):
        assert ok
        call()
        sb.check_status(cuda_device)
        books_equal(cache, books)

    step(books.extend(torch.tensor(counts)), lambda: cache.extend(ints(counts)))
    for s in range(max_seqs):
        for pos in range(books.lens[s]):
            books.write(s, pos, 0)
    step(books.fork(src, dst), lambda: cache.fork(ints(src), ints(dst)))
    step(books.free(gone), lambda: cache.free(ints(gone)))
    books.compact()
    step(True, cache.compact)
    step(books.extend(3), lambda: cache.extend(3))


@gpu
def test_pages_refusals_on_the_device(cuda_device):
    import stickbreaking_attention_b200 as sb
    cache = sb.PagedKVCache(1, 6, 1, 4, 8, 4, 16, dtype=BF16, device=cuda_device)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    cache.extend(ints(6, 4, 0, 0))
    sb.check_status(cuda_device)
    books = [t.clone() for t in (cache.page_table, cache.seq_lens, cache.page_refs)]
    for call, what in ((lambda: cache.extend(ints(20, 0, 0, 0)), "length"), (lambda: cache.extend(ints(0, -1, 0, 0)), "length"),
                       (lambda: cache.extend(ints(0, 0, 16, 0)), "free pages"), (lambda: cache.fork(ints(0), ints(1)), "listed"),
                       (lambda: cache.fork(ints(0, 1), ints(2, 2)), "listed"), (lambda: cache.fork(ints(4), ints(2)), "listed"),
                       (lambda: cache.fork(ints(0), ints(-1)), "listed"), (lambda: cache.fork(ints(0, 2), ints(2, 3)), "listed"),
                       (lambda: cache.fork(ints(2), ints(2)), "listed"), (lambda: cache.free(ints(0, 4)), "listed")):
        call()
        with pytest.raises(sb._cabi.SbError, match=what):
            sb.check_status(cuda_device)
        for t, old in zip((cache.page_table, cache.seq_lens, cache.page_refs), books):
            assert torch.equal(t, old)
    cache.fork(ints(0, 0), ints(2, 3))                       # one source twice, each fork its own last page
    cache.free(ints(0, 0, 0))
    cache.fork(ints(), ints())
    cache.free(ints())
    sb.check_status(cuda_device)
    assert cache.seq_lens.tolist() == [0, 4, 6, 6]
    assert cache.page_refs.tolist() == [2, 0, 1, 1, 1, 0]


@gpu
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (FP16, 50), (FP32, 6)])
@pytest.mark.parametrize("layout", ["own", "token_major", "inside", "one_layer"])
def test_fork_and_compact_copy_all_layers(cuda_device, dtype, d, layout):
    """Copied rows, all layers and heads; every other row of the pool as it was."""
    import stickbreaking_attention_b200 as sb
    layers, pages, kv, page = (1 if layout == "one_layer" else 3), 30, 5, 16
    gen = torch.Generator().manual_seed(30)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_device)

    def pool():
        x = torch.randn(layers, pages, kv, page, d, generator=gen).to(dtype).to(cuda_device)
        if layout == "token_major":
            return x.transpose(2, 3).contiguous().transpose(2, 3)
        if layout == "inside":
            wide = torch.zeros(layers, pages, kv, page, d + 3, dtype=dtype, device=cuda_device)
            wide[..., 2:d + 2] = x
            return wide[..., 2:d + 2]
        return x[0] if layout == "one_layer" else x

    k, v = pool(), pool()
    table = torch.full((6, 10), -1, dtype=torch.int32)
    table[0, :4], table[1, :2] = torch.tensor([28, 5, 29, 17]), torch.tensor([11, 2])
    table, lens = table.to(cuda_device), ints(53, 32, 0, 0, 0, 0)
    refs = torch.zeros(pages, dtype=torch.int32, device=cuda_device)
    refs[[28, 5, 29, 17, 11, 2]] = 1
    want = [t.clone() for t in (k, v)]
    sb.kv_fork(k, v, table, lens, refs, ints(0, 1, 0), ints(4, 2, 3))
    sb.check_status(cuda_device)
    for t in want:
        for new in (0, 1):
            t[..., new, :, :5, :] = t[..., 17, :, :5, :]
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert table[4, :4].tolist() == [28, 5, 29, 0] and table[3, :4].tolist() == [28, 5, 29, 1] and table[2, :2].tolist() == [11, 2]
    sb.kv_compact(k, v, table, lens, refs)                   # 8 in use: 11, 17, 28, 29 to 3, 4, 6, 7
    sb.check_status(cuda_device)
    for t in want:
        for old, new in ((11, 3), (17, 4), (28, 6), (29, 7)):
            t[..., new, :, :, :] = t[..., old, :, :, :]
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert table[0, :4].tolist() == [6, 5, 7, 4] and table[1, :2].tolist() == [3, 2] and table[4, :4].tolist() == [6, 5, 7, 0]
    assert refs.tolist() == [1, 1, 2, 2, 1, 3, 3, 3] + [0] * 22


# ---- together -------------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype,tol", [(BF16, 2e-2), (FP32, 1e-4)])
def test_a_serving_run(cuda_device, dtype, tol):
    """Prompts prefilled by sb_attn_varlen, sampled twice each (fork), stepped, some freed, the pool compacted, stepped on: every
    step's rows are those of the whole attention over the sequence's tokens."""
    import stickbreaking_attention_b200 as sb
    layers, heads, kv, d, page, prompts = 2, 4, 2, 64, 16, [37, 64, 5]
    gen = torch.Generator().manual_seed(40)
    dev = cuda_device
    cache = sb.PagedKVCache(layers, 60, kv, page, d, 6, 160, dtype=dtype, device=dev)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    tokens = {}                                     # (sequence, layer): keys and values so far
    rand = lambda *shape: torch.randn(shape, generator=gen).to(dtype)
    with torch.no_grad():
        lens = prompts + [0, 0, 0]
        cache.extend(ints(*lens))
        cu = ints(0, *torch.tensor(prompts).cumsum(0).tolist())
        for layer in range(layers):
            k, v = rand(kv, sum(prompts), d).to(dev), rand(kv, sum(prompts), d).to(dev)
            q = rand(kv, sum(prompts), d).to(dev)
            o, rem = sb.sb_attn_varlen(q, k, v, cu, max(prompts))
            assert torch.isfinite(o).all()
            cache.append(layer, k, v, cu, rows=slice(0, 3))
            for s in range(3):
                tokens[s, layer] = torch.stack((k[:, cu[s]:cu[s + 1]], v[:, cu[s]:cu[s + 1]])).cpu()
        cache.fork(ints(0, 1, 2), ints(3, 4, 5))
        for s in range(3):
            for layer in range(layers):
                tokens[s + 3, layer] = tokens[s, layer].clone()
        alive = [1] * 6
        for step in range(50):
            if step == 20:
                cache.free(ints(1, 3))
                cache.compact()
                alive[1] = alive[3] = 0
            cache.extend(ints(*alive))
            for layer in range(layers):
                k, v, q = (rand(6, h, 1, d) for h in (kv, kv, heads))
                cache.append(layer, k.to(dev), v.to(dev))
                o, rem = cache.attend(layer, q.to(dev))
                for s in range(6):
                    if not alive[s]:
                        assert bool((o[s] == 0).all()) and bool((rem[s] == 1).all())
                        continue
                    tokens[s, layer] = torch.cat((tokens[s, layer], torch.stack((k[s], v[s]))), 2)
                    if step % 7 == 0 or step in (19, 20, 21):
                        ks, vs = (t.repeat_interleave(heads // kv, 0).to(dev) for t in tokens[s, layer])
                        n = ks.shape[1]
                        whole = torch.zeros(heads, n, d, dtype=dtype, device=dev)
                        whole[:, -1] = q[s, :, 0].to(dev)
                        want_o, want_rem = sb.sb_attn_varlen(whole, ks, vs, ints(0, n), n)
                        assert H.max_abs(o[s, :, 0], want_o[:, -1]) <= tol and H.max_abs(rem[s, :, 0], want_rem[:, -1]) <= tol
        sb.check_status(dev)
        assert int((cache.page_refs > 0).sum()) <= 4 * 10
        cache.free(ints(0, 1, 2, 3, 4, 5))
        assert cache.page_refs.tolist() == [0] * 60 and bool((cache.page_table == -1).all())


@gpu
def test_serving_operators_under_compile(cuda_device):
    import stickbreaking_attention_b200 as sb
    q, cache = make(41, [40, 9], 4, 2, 64, 16, BF16)
    args = [t.to(cuda_device) for t in (q, *cache)]
    k_new = torch.randn(2, 2, 1, 64, device=cuda_device).to(BF16)

    def step(q, kp, vp, table, lens, k_new):
        sb.kv_append(k_new, k_new, kp, vp, table, lens)
        o, rem = sb.sb_attn_decode(q, kp, vp, table, lens, attend_current=True)
        return o * 2, rem

    with torch.no_grad():
        eager = step(*args, k_new)
        args[1].copy_(cache[0]), args[2].copy_(cache[1])
        compiled = torch.compile(step, fullgraph=True, backend="aot_eager")(*args, k_new)
    assert torch.equal(eager[0], compiled[0]) and torch.equal(eager[1], compiled[1])
    sb.check_status(cuda_device)


@gpu
def test_serving_refusals(cuda_device):
    import stickbreaking_attention_b200 as sb
    q, cache = make(42, [40, 9], 4, 2, 64, 16, BF16)
    q, k, v, table, lens = (t.to(cuda_device) for t in (q, *cache))
    bad = [(q.float(), k, v, table, lens), (q[:, :3], k, v, table, lens), (q[..., :32], k, v, table, lens), (q[0], k, v, table, lens),
           (q, k[:5], v, table, lens), (q, k.float(), v.float(), table, lens), (q, k.cpu(), v.cpu(), table, lens),
           (q, k, v, table.long(), lens), (q, k, v, table, lens.long()), (q, k, v, table[:1], lens), (q, k, v, table.cpu(), lens),
           (q, k, v, table[0], lens), (q[:1], k, v, table, lens), (q, k, v, table.t().contiguous().t(), lens), (q, k[0], v[0], table, lens),
           (q, k[..., ::2], v[..., ::2], table, lens)]
    with torch.no_grad():
        for args in bad:
            with pytest.raises((ValueError, sb._cabi.SbError)):
                sb.sb_attn_decode(*args)
        new = torch.zeros(2, 2, 1, 64, dtype=BF16, device=cuda_device)
        cu = torch.tensor([0, 1, 2], device=cuda_device)
        for args in ((new.float(), new, k, v, table, lens), (new[:, :1], new[:, :1], k, v, table, lens), (new[0], new[0], k, v, table, lens),
                     (new[:1], new[:1], k, v, table, lens), (new, new, k.expand(3, *k.shape), v, table, lens),
                     (new[0], new[0], k, v, table, lens, cu[:2]), (new[0], new[0], k, v, table, lens, cu.float()),
                     (new, new, k[:1].expand_as(k), v, table, lens), (new.cpu(), new.cpu(), k, v, table, lens)):
            with pytest.raises((ValueError, sb._cabi.SbError)):
                sb.kv_append(*args)
        refs = torch.zeros(k.shape[0], dtype=torch.int32, device=cuda_device)
        one = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        for call in (lambda: sb.kv_extend(table, lens, refs, one, 16), lambda: sb.kv_extend(table, lens, refs, -1, 16),
                     lambda: sb.kv_extend(table, lens, refs.long(), 1, 16), lambda: sb.kv_extend(table, lens, refs, 1, 0),
                     lambda: sb.kv_fork(k, v, table, lens, refs[:-1], one, one), lambda: sb.kv_fork(k, v, table, lens, refs, one, one[:0]),
                     lambda: sb.kv_fork(k, v, table, lens, refs, one.long(), one), lambda: sb.kv_free(table, lens, refs, one.cpu(), 16),
                     lambda: sb.kv_compact(k[0], v[0], table, lens, refs), lambda: sb.kv_compact(k[:1].expand_as(k), v, table, lens, refs)):
            with pytest.raises((ValueError, sb._cabi.SbError)):
                call()
    for args in ((q.clone().requires_grad_(True), k, v), (q, k.clone().requires_grad_(True), v)):
        with pytest.raises(NotImplementedError, match="derivative"):
            sb.sb_attn_decode(*args, table, lens)
    sb.check_status(cuda_device)
    k_old = k.clone()
    with torch.no_grad():                                      # nothing to do
        o, rem = sb.sb_attn_decode(q[:0], k, v, table[:0], lens[:0])
        assert o.shape == (0, 4, 1, 64) and rem.shape == (0, 4, 1)
        sb.kv_append(new[:, :, :0], new[:, :, :0], k, v, table, lens)
    assert torch.equal(k.nan_to_num(7.0), k_old.nan_to_num(7.0))


@gpu
def test_append_is_seen_by_autograd(cuda_device):
    """A pool that a graph has saved and that is then written to: the backward refuses."""
    import stickbreaking_attention_b200 as sb
    _, (k, v, table, lens) = make(43, [40], 1, 1, 64, 16, FP32, poison=False)
    k, v, table, lens = (t.to(cuda_device) for t in (k, v, table, lens))
    x = torch.ones_like(k, requires_grad=True)
    y = (x * k).sum()
    new = torch.zeros(1, 1, 1, 64, device=cuda_device)
    sb.kv_append(new, new, k, v, table, lens)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# ---- without a GPU --------------------------------------------------------------------------------------------------------

def test_cpu_tensors_are_refused():
    import stickbreaking_attention_b200 as sb
    q, cache = make(50, [40, 9], 4, 2, 64, 16, BF16)
    k, v, table, lens = cache
    refs = torch.zeros(k.shape[0], dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: sb.sb_attn_decode(q, *cache), lambda: sb.kv_append(q[:, :2], q[:, :2], *cache),
                 lambda: sb.kv_extend(table, lens, refs, 1, 16), lambda: sb.kv_fork(k, v, table, lens, refs, one, one),
                 lambda: sb.kv_free(table, lens, refs, one, 16), lambda: sb.kv_compact(k, v, table, lens, refs)):
        with pytest.raises(ValueError, match="CUDA device"):
            call()


def test_c_entries_refuse_bad_arguments_before_they_touch_a_device():
    from stickbreaking_attention_b200 import _cabi
    lib = _cabi.load()
    size = ctypes.sizeof

    def decode(**kw):
        p = _cabi.SbDecodeParams(struct_bytes=size(_cabi.SbDecodeParams), dtype=1, batch=2, heads=4, kv_heads=2, new_tokens=1, head_dim=64,
                                 page_size=16, num_pages=8, max_pages=4, logit_scale=0.125, page_table=256, page_table_stride=4,
                                 seq_lens=256, rem=256, workspace=256)
        p.q = p.o = _cabi.SbTensor(256, 256, 64, 64)
        p.k = p.v = _cabi.SbCache(256, 0, 2048, 1024, 64)
        for key, value in kw.items():
            setattr(p, key, value)
        return lib.sb_attn_decode(p, None)

    for kw in (dict(struct_bytes=8), dict(dtype=7), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=257),
               dict(page_size=0), dict(num_pages=0), dict(max_pages=0), dict(new_tokens=0), dict(new_tokens=1025), dict(batch=-1),
               dict(reserved=1), dict(seq_lens=None), dict(rem=None), dict(k=_cabi.SbCache(None, 0, 2048, 1024, 64)),
               dict(v=_cabi.SbCache(256, 0, -2048, 1024, 64)), dict(o=_cabi.SbTensor(256, 0, 64, 64))):
        assert decode(**kw) == 1, kw
        assert lib.sb_last_error() != b""
    assert decode(batch=0) == 0
    assert lib.sb_attn_decode(None, None) == 1 and lib.sb_kv_append(None, None) == 1 and lib.sb_kv_extend(None, None) == 1

    def append(**kw):
        p = _cabi.SbAppendParams(struct_bytes=size(_cabi.SbAppendParams), dtype=1, num_seq=2, kv_heads=2, head_dim=64, page_size=16, num_pages=8,
                                 max_pages=4, tokens=1, page_table=256, page_table_stride=4, seq_lens=256)
        p.k = p.v = _cabi.SbTensor(256, 128, 64, 64)
        p.k_cache = p.v_cache = _cabi.SbCache(256, 0, 2048, 1024, 64)
        for key, value in kw.items():
            setattr(p, key, value)
        return lib.sb_kv_append(p, None)

    for kw in (dict(struct_bytes=8), dict(dtype=-1), dict(kv_heads=0), dict(tokens=-1), dict(tokens=2 ** 32), dict(seq_lens=None),
               dict(k=_cabi.SbTensor(None, 0, 0, 0)), dict(v_cache=_cabi.SbCache(256, 0, 0, 1024, 64))):
        assert append(**kw) == 1, kw
    assert append(tokens=0) == 0 and append(num_seq=0) == 0

    def pages(name, **kw):
        p = _cabi.SbPagesParams(struct_bytes=size(_cabi.SbPagesParams), max_seqs=3, max_pages=4, num_pages=8, page_size=16, n=1, dtype=1,
                                layers=1, kv_heads=2, head_dim=64, page_table=256, page_table_stride=4, seq_lens=256, page_refs=256,
                                first=256, second=256, workspace=256, workspace_bytes=1 << 20)
        p.k_cache = p.v_cache = _cabi.SbCache(256, 0, 2048, 1024, 64)
        for key, value in kw.items():
            setattr(p, key, value)
        return getattr(lib, name)(p, None)

    for name in ("sb_kv_extend", "sb_kv_fork", "sb_kv_free", "sb_kv_compact"):
        for kw in (dict(struct_bytes=4), dict(max_seqs=0), dict(max_pages=0), dict(num_pages=(1 << 20) + 1), dict(page_size=0), dict(n=-1),
                   dict(n=65536), dict(reserved=1), dict(page_refs=None), dict(page_table_stride=3)):
            assert pages(name, **kw) == 1, (name, kw)
    for name in ("sb_kv_extend", "sb_kv_fork", "sb_kv_compact"):
        assert pages(name, workspace_bytes=16) == 2 and pages(name, workspace=None) == 2 and pages(name, workspace=128) == 2
    assert pages("sb_kv_extend", first=None, count=-1) == 1
    assert pages("sb_kv_fork", second=None) == 1 and pages("sb_kv_free", first=None) == 1
    assert pages("sb_kv_fork", layers=0) == 1 and pages("sb_kv_compact", dtype=9) == 1
    assert pages("sb_kv_fork", n=0) == 0 and pages("sb_kv_free", n=0) == 0


def test_the_books_of_the_tests():
    """The Python books against a few cases done by hand."""
    books = R.Books(4, 4, 8, 4)
    assert books.extend(torch.tensor([6, 4, 0, 0])) and books.rows == [[0, 1], [2], [], []]
    for pos in range(6):
        books.write(0, pos, pos)
    assert not books.extend(torch.tensor([0, 0, 17, 0])) and not books.fork([0], [1]) and not books.fork([0, 2], [2, 3])
    assert books.fork([0], [3]) and books.rows[3] == [0, 3] and books.tokens(3) == list(range(6)) and books.refs == [2, 1, 1, 1, 0, 0, 0, 0]
    assert books.free([0, 0]) and books.refs == [1, 0, 1, 1, 0, 0, 0, 0]
    books.compact()
    assert books.rows == [[], [2], [], [0, 1]] and books.tokens(3) == list(range(6)) and books.refs == [1, 1, 1, 0, 0, 0, 0, 0]


def test_the_decode_reference_is_the_oracles_last_row():
    from oracle import sb_oracle as O
    gen = torch.Generator().manual_seed(51)
    n, d, page = 37, 16, 8
    q, k, v = (torch.randn(1, n, d, generator=gen) for _ in range(3))
    pages = [torch.nn.functional.pad(t, (0, 0, 0, 3)).view(5, 1, page, d) for t in (k, v)]
    table, lens = torch.arange(5, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    for current in (False, True):
        want, rem = O.varlen_dense(q, k, v, [n], attend_current=current)
        got = R.decode(q[:, -2:][None], *pages, table, lens, attend_current=current)
        assert torch.allclose(got[0][0, 0].float(), want[0, -2:], atol=1e-5) and torch.allclose(got[1][0, 0].float(), rem[0, -2:], atol=1e-5)
