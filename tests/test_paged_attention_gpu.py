"""Attention over the paged cache against its definition in 64 bits."""
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _q(tokens, heads, d, dtype, seed=9):
    return torch.randn(tokens, heads, d, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _run(q, k, v, table, q_start, kv_len, window=0, sinks=0, **kw):
    from llcompiler_b200.executor import paged_attention
    dev = [R.to_device(t, DEV) for t in (q, k, v)]
    return paged_attention(*dev, table.to(DEV), q_start.to(DEV), kv_len.to(DEV), window=window, sinks=sinks, **kw)


def _check(got, q, k, v, table, q_start, kv_len, window=0, sinks=0, scale=None):
    want, size, largest = R.attention(q, k, v, table, q_start, kv_len, R.scale_of(q.shape[2]) if scale is None else scale, window, sinks)
    owned = ~want.isnan().any(-1).any(-1)
    tol = R.attention_tolerance(want, size, largest, q.dtype)
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= tol)[owned]
    assert not bad.any(), (int(bad.sum()), float((off / tol)[owned].max()))
    from llcompiler_b200 import _capi as C
    assert C.lib().llc_cuda_status() == 0


CASES = [
    # new tokens, lengths, heads, kv heads, d, page, window, sinks
    ([1], [1], 1, 1, 64, 16, 0, 0),
    ([1], [77], 12, 12, 64, 16, 0, 0),
    ([1, 1, 1], [1, 64, 65], 8, 2, 128, 16, 0, 0),
    ([1] * 5, [128, 129, 300, 517, 16], 4, 4, 128, 32, 0, 0),
    ([1, 1], [900, 431], 8, 1, 64, 128, 0, 0),
    ([1, 0, 1], [40, 33, 0], 4, 2, 64, 16, 0, 0),            # a sequence without new tokens, a token without keys
    ([1, 1, 1], [500, 64, 3], 6, 2, 128, 16, 100, 0),
    ([1, 1, 1], [500, 64, 130], 6, 2, 64, 64, 33, 4),
    ([1, 1], [700, 701], 4, 4, 64, 16, 1, 0),
    ([1, 1], [700, 701], 4, 4, 128, 32, 1, 130),
    ([2, 3, 1], [50, 3, 200], 4, 1, 128, 16, 0, 0),          # a few tokens each
    ([4, 2], [260, 259], 10, 2, 64, 32, 20, 5),
    ([5], [5], 3, 1, 128, 16, 0, 0),
    ([33], [33], 3, 1, 64, 16, 0, 0),
    ([128], [128], 2, 2, 128, 64, 0, 0),
    ([70, 1, 0, 129], [200, 150, 9, 129], 4, 2, 128, 16, 0, 0),
    ([257], [400], 2, 1, 64, 32, 0, 0),
    ([140], [500], 4, 1, 128, 128, 64, 0),
    ([140, 30], [500, 300], 5, 1, 64, 16, 7, 3),
    ([90], [300], 4, 1, 128, 16, 60, 140),
    ([12, 300], [5, 290], 2, 2, 64, 16, 0, 0),               # more new tokens than keys: the first ones see nothing
    ([64], [1000], 16, 1, 128, 256, 0, 0),
    # keys cut into parts: of chunks (at least 1536 keys each) and of few rows (each warp its share)
    ([20], [5000], 2, 1, 128, 64, 0, 0),
    ([40], [5000], 2, 2, 64, 16, 0, 0),
    ([17, 1, 35], [4001, 4999, 60], 2, 1, 64, 32, 0, 0),
    ([36], [6500], 1, 1, 64, 16, 4700, 9),
    ([1], [5000], 2, 1, 128, 16, 0, 0),
    ([3, 1], [4100, 7], 4, 2, 64, 128, 0, 0),
    ([7], [2100], 4, 1, 128, 16, 1900, 50),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("new,lens,heads,kv_heads,d,page,window,sinks", CASES)
def test_paged_attention(dtype, heads_first, new, lens, heads, kv_heads, d, page, window, sinks):
    # slots that hold no token hold NaN: none of it may reach the result
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype, heads_first=heads_first, fill=float("nan"))
    q = _q(sum(new) + 2, heads, d, dtype)
    out = torch.full(q.shape, 5.0, device=DEV, dtype=dtype)
    got = _run(q, k, v, table, q_start, kv_len, window, sinks, max_q=max(new), out=out)
    assert got is out and (out[sum(new):] == 5).all()
    _check(out, q, k, v, table, q_start, kv_len, window, sinks)


@pytest.mark.parametrize("dtype,d,page,new,lens", [
    (torch.float32, 64, 16, [1, 3], [77, 20]), (torch.float32, 128, 64, [40], [100]), (torch.bfloat16, 80, 16, [1, 9], [50, 40]), (torch.float16, 256, 32, [2], [70]),
    (torch.bfloat16, 64, 7, [1, 8], [50, 15]), (torch.float16, 33, 5, [3], [9]), (torch.float32, 1, 1, [2], [4]), (torch.bfloat16, 128, 8, [1], [30]),
])
@pytest.mark.parametrize("window,sinks", [(0, 0), (6, 2)])
def test_other_types_head_sizes_and_pages(dtype, d, page, new, lens, window, sinks):
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, 2, d, dtype, fill=float("nan"))
    q = _q(sum(new), 4, d, dtype)
    _check(_run(q, k, v, table, q_start, kv_len, window, sinks), q, k, v, table, q_start, kv_len, window, sinks)


@pytest.mark.parametrize("new,lens", [([1, 1], [200, 61]), ([50], [170])])
def test_scores_that_grow_shrink_and_overflow_the_running_maximum(new, lens):
    """Keys that score far higher or lower from block to block, and a scale of zero and below."""
    k, v, table, q_start, kv_len = R.make_batch(new, lens, 16, 2, 64, torch.bfloat16)
    q = _q(sum(new), 4, 64, torch.bfloat16)
    for b in range(len(new)):
        for j in range(lens[b]):
            at = (int(table[b, j // 16]), j % 16)
            k[at] = (k[at].float() * (0.1 + 6.0 * j / lens[b])).to(torch.bfloat16)
    for scale in (0.5, 0.0, -0.25):
        got = _run(q, k, v, table, q_start, kv_len, scale=scale)
        _check(got, q, k, v, table, q_start, kv_len, scale=scale)


@pytest.mark.parametrize("new,lens,window,sinks", [([1, 1], [300, 170], 40, 3), ([60, 2], [300, 170], 40, 3), ([1, 40], [90, 64], 0, 0), ([3, 2], [300, 60], 0, 0),
                                                   ([4, 1], [900, 30], 20, 2), ([30, 1], [5000, 30], 3600, 3)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_keys_that_are_not_visible_may_hold_anything(new, lens, window, sinks, what):
    """Keys that no token of the call sees hold NaN and infinities (they lie before the window, behind the sinks), and a
    chunk's later tokens hold them as well: the earlier tokens do not see those."""
    k, v, table, q_start, kv_len = R.make_batch(new, lens, 16, 2, 128, torch.bfloat16)
    q = _q(sum(new), 4, 128, torch.bfloat16)
    for b, (n, length) in enumerate(zip(new, lens)):
        for j in range(length):
            if window and j >= sinks and j <= length - n - window:
                at = (int(table[b, j // 16]), j % 16)
                k[at], v[at] = what, what
    got = _run(q, k, v, table, q_start, kv_len, window, sinks, max_q=max(new))
    _check(got, q, k, v, table, q_start, kv_len, window, sinks)
    if max(new) > 1:
        b = max(range(len(new)), key=lambda i: new[i])
        j = lens[b] - 1                                       # the last token of the chunk
        at = (int(table[b, j // 16]), j % 16)
        k2, v2 = k.clone(), v.clone()
        k2[at], v2[at] = what, what
        got = _run(q, k2, v2, table, q_start, kv_len, window, sinks, max_q=max(new))
        last = int(q_start[b + 1]) - 1
        assert not torch.isfinite(got[last].float()).all()
        rest = [t for t in range(sum(new)) if t != last]
        want, size, largest = R.attention(q, k, v, table, q_start, kv_len, R.scale_of(128), window, sinks)
        off = (got.double().cpu() - want).abs()[rest]
        assert (off <= R.attention_tolerance(want, size, largest, q.dtype)[rest]).all()


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [70, 40, 33]), ([30, 40, 1], [70, 40, 33])])
def test_bad_pages_read_as_zeros_and_are_counted(new, lens):
    k, v, table, q_start, kv_len = R.make_batch(new, lens, 16, 2, 64, torch.bfloat16, fill=float("nan"))
    q = _q(sum(new), 4, 64, torch.bfloat16)
    bad = torch.zeros(1, device=DEV, dtype=torch.int32)
    _run(q, k, v, table, q_start, kv_len, max_q=max(new), bad_pages=bad)
    assert int(bad) == 0                                     # the -1 past a sequence's pages are none
    table[0, 1], table[2, 2] = k.shape[0], -7
    got = _run(q, k, v, table, q_start, kv_len, max_q=max(new), bad_pages=bad)
    assert int(bad) >= 2
    _check(got, q, k, v, table, q_start, kv_len)
    bad.zero_()
    _run(q, k, v, table, q_start, kv_len, max_q=max(new), window=2, bad_pages=bad)
    # with a window of two nobody looks at sequence 0's second page; sequence 2's last token stands on its bad one
    assert int(bad) >= 1


def test_lengths_and_rows_out_of_range_stay_inside():
    """A length past the table counts as the table's reach, a negative one as nothing; a sequence with more tokens than
    max_q is left out; rows behind q are not touched."""
    k, v, table, q_start, kv_len = R.make_batch([1, 1, 4], [64, 16, 64], 16, 2, 64, torch.bfloat16, width=4)
    q = _q(6, 4, 64, torch.bfloat16)
    over = kv_len.clone()
    over[0], over[1] = 10 ** 6, -3
    out = torch.full(q.shape, 5.0, device=DEV, dtype=torch.bfloat16)
    _run(q, k, v, table, q_start, over, max_q=3, out=out)
    assert (out[2:] == 5).all() and (out[1] == 0).all()
    want, size, largest = R.attention(q, k, v, table, q_start, kv_len, R.scale_of(64), 0, 0)
    assert ((out[0].cpu().double() - want[0]).abs() <= R.attention_tolerance(want, size, largest, q.dtype)[0]).all()
    out.fill_(5.0)
    ends = q_start.clone()
    ends[3] = 1000                                            # past q's rows
    _run(q, k, v, table, ends, kv_len, out=out)
    assert torch.isfinite(out.float()).all()


def test_empty_batches_pools_and_tables():
    from llcompiler_b200.executor import kv_append, paged_attention, rotary
    bf = dict(device=DEV, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, device=DEV, dtype=torch.int32)
    pool, none = torch.zeros(3, 16, 2, 64, **bf), torch.zeros(0, 16, 2, 64, **bf)
    q, k = torch.ones(3, 4, 64, **bf), torch.ones(3, 2, 64, **bf)
    # no tokens
    assert rotary(q[:0], torch.zeros(0, device=DEV, dtype=torch.int64), R.inv_freq(32).to(DEV)).shape == (0, 4, 64)
    assert paged_attention(q[:0], pool, pool, i32(0)[None], i32(0, 0), i32(5)).shape == (0, 4, 64)
    # no sequences: nobody's rows
    out = torch.full_like(q, 5.0)
    table = torch.zeros(0, 4, device=DEV, dtype=torch.int32)
    paged_attention(q, pool, pool, table, i32(0), i32(), out=out)
    kv_append(k, k, pool, pool, table, i32(0), i32(), q=q, q_out=out)
    assert (out == 5).all() and (pool == 0).all()
    # a pool without pages: every page is a bad one and reads as zeros; a table without columns: nothing is visible
    bad = i32(0)
    assert (paged_attention(q, none, none, i32(0, 0)[None], i32(0, 3), i32(3), max_q=3, bad_pages=bad) == 0).all() and int(bad) >= 1
    assert (paged_attention(q, pool, pool, torch.zeros(1, 0, device=DEV, dtype=torch.int32), i32(0, 3), i32(3), max_q=3) == 0).all()
    bad.zero_()
    kv_append(k, k, none, none, i32(0, 0)[None], i32(0, 3), i32(3), bad_pages=bad)
    kv_append(k, k, pool, pool, torch.zeros(1, 0, device=DEV, dtype=torch.int32), i32(0, 3), i32(3), bad_pages=bad)
    assert int(bad) == 6 and (pool == 0).all()
    # rows before the first sequence are nobody's either
    out.fill_(5.0)
    kv_append(k, k, pool, pool, i32(1)[None], i32(2, 3), i32(1), q=q, q_out=out)
    assert (out[:2] == 5).all() and (out[2] == 1).all() and (pool[1, 0] == 1).all() and int(pool.sum()) == 128
    out.fill_(5.0)
    paged_attention(q, pool, pool, i32(1)[None], i32(2, 3), i32(1), max_q=1, out=out)
    assert (out[:2] == 5).all() and (out[2] == 1).all()


def test_strided_queries_and_output():
    k, v, table, q_start, kv_len = R.make_batch([3, 40], [30, 90], 16, 2, 64, torch.float16)
    qkv = _q(43, 4 + 2 + 2, 64, torch.float16)
    q = qkv[:, :4]
    from llcompiler_b200.executor import paged_attention
    dev = qkv.to(DEV)
    out = torch.full((43, 2, 4, 64), 5.0, device=DEV, dtype=torch.float16)
    args = [t.to(DEV) for t in (k, v, table, q_start, kv_len)]
    paged_attention(dev[:, :4], *args, out=out[:, 1])
    _check(out[:, 1], q, k, v, table, q_start, kv_len)
    assert (out[:, 0] == 5).all()
    # a base that is not 16-byte aligned
    flat = torch.empty(43 * 4 * 64 + 8, device=DEV, dtype=torch.float16)
    odd = flat[1 : 1 + 43 * 4 * 64].view(43, 4, 64)
    paged_attention(dev[:, :4], *args, out=odd)
    _check(odd, q, k, v, table, q_start, kv_len)


@pytest.mark.parametrize("d", [64, 128])
def test_offsets_past_32_bits(d):
    """A pool of more than 2^31 elements, with the sequence's pages at its end."""
    page, kv_heads = 64, 8
    pages = (2 ** 31 + 2 ** 27) // (page * kv_heads * d)
    new, lens = [1, 20], [150, 90]
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, torch.bfloat16, spare=0)
    small = k.shape[0]
    kc = torch.empty(pages, page, kv_heads, d, device=DEV, dtype=torch.bfloat16)
    vc = torch.empty_like(kc)
    kc[pages - small:], vc[pages - small:] = k.to(DEV), v.to(DEV)
    from llcompiler_b200.executor import kv_append, paged_attention
    far = torch.where(table >= 0, table + (pages - small), table)
    q = _q(21, 16, d, torch.bfloat16)
    got = paged_attention(q.to(DEV), kc, vc, far.to(DEV), q_start.to(DEV), kv_len.to(DEV), max_q=20)
    _check(got, q, k, v, table, q_start, kv_len)
    # and written there
    nk = _q(21, kv_heads, d, torch.bfloat16, seed=3)
    kv_append(nk.to(DEV), nk.to(DEV), kc, vc, far.to(DEV), q_start.to(DEV), kv_len.to(DEV))
    last = (int(table[1, 89 // page]), 89 % page)
    assert torch.equal(kc[pages - small + last[0], last[1]].cpu(), nk[20]) and torch.equal(vc[pages - small + last[0], last[1]].cpu(), nk[20])


def test_captured_step_replays_with_other_lengths():
    """A decoding step (append and attend) captured once and replayed while sequences grow, change places and end; two
    captured graphs on two streams at once do not disturb each other."""
    from llcompiler_b200.executor import kv_append, paged_attention
    heads, kv_heads, d, page, batch = 8, 2, 128, 16, 3
    lens = [700, 33, 260]
    k, v, table, q_start, kv_len = R.make_batch([1] * batch, [n + 5 for n in lens], page, kv_heads, d, torch.bfloat16)
    freq = R.inv_freq(d // 2)

    class Step:
        def __init__(self, seed):
            self.kc, self.vc, self.table, self.q_start = (R.to_device(t, DEV) for t in (k, v, table, q_start))
            self.kv_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
            self.x = _q(batch, heads + 2 * kv_heads, d, torch.bfloat16, seed=seed).to(DEV)
            self.freq = freq.to(DEV)

        def __call__(self):
            q = kv_append(self.x[:, heads : heads + kv_heads], self.x[:, heads + kv_heads :], self.kc, self.vc, self.table, self.q_start, self.kv_len,
                          q=self.x[:, :heads], inv_freq=self.freq)
            return paged_attention(q, self.kc, self.vc, self.table, self.q_start, self.kv_len, max_q=1), q

    steps = [Step(1), Step(2)]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, st in zip(steps, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            s()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(s())
        graphs.append(g)
    for grow in range(1, 5):
        for s in steps:
            s.kv_len += torch.tensor([1, 1, 0] if grow % 2 else [1, 0, 1], dtype=torch.int32, device=DEV)
            s.x.copy_(_q(batch, heads + 2 * kv_heads, d, torch.bfloat16, seed=100 * grow).to(DEV))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, (out, q) in zip(steps, outs):
            _check(out, q.cpu(), s.kc.cpu(), s.vc.cpu(), table, q_start, s.kv_len.cpu())


def test_one_long_sequence_among_many_short_ones():
    """More (sequence, key head, row) sums than the joining kernel gives a block each, one pair cut into many parts, and the same
    without a workspace."""
    import ctypes
    from llcompiler_b200 import _capi as C
    batch, heads, kv_heads, d, page = 80, 16, 4, 64, 16
    lens = [17] * batch
    lens[37] = 6000
    k, v, table, q_start, kv_len = R.make_batch([1] * batch, lens, page, kv_heads, d, torch.bfloat16)
    q = _q(batch, heads, d, torch.bfloat16)
    got = _run(q, k, v, table, q_start, kv_len, max_q=1)
    _check(got, q, k, v, table, q_start, kv_len)
    dev = [R.to_device(t, DEV) for t in (q, k, v, table, q_start, kv_len)]
    out = torch.full(q.shape, 5.0, device=DEV, dtype=torch.bfloat16)
    p = C.LlcPagedAttentionParams()
    p.q, p.k_cache, p.v_cache, p.page_table, p.q_start, p.kv_len = (ctypes.c_void_p(t.data_ptr()) for t in dev)
    p.out, p.dtype, p.scale = ctypes.c_void_p(out.data_ptr()), 8, R.scale_of(d)
    p.tokens, p.batch, p.heads, p.kv_heads, p.d, p.max_q = batch, batch, heads, kv_heads, d, 1
    p.num_pages, p.page_size, p.table_width, p.table_s0 = k.shape[0], page, table.shape[1], table.stride(0)
    p.q_st, p.q_sh, p.o_st, p.o_sh = q.stride(0), q.stride(1), out.stride(0), out.stride(1)
    p.kc_sp, p.kc_sn, p.kc_sh = k.stride()[:3]
    p.vc_sp, p.vc_sn, p.vc_sh = v.stride()[:3]
    assert C.lib().llc_cuda_paged_attention_workspace(ctypes.byref(p)) > 0
    C.check(C.lib().llc_cuda_paged_attention(ctypes.byref(p), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    _check(out, q, k, v, table, q_start, kv_len)


@pytest.mark.parametrize("batch", [127, 300, 700])
def test_large_batches_of_few_tokens(batch):
    """More sequences than a block has threads: single tokens, and the same with some chunks among them and sequences without any."""
    kv_heads, d, page = 1, 64, 16
    lens = [1 + (i * 13) % 40 for i in range(batch)]
    k, v, table, q_start, kv_len = R.make_batch([1] * batch, lens, page, kv_heads, d, torch.float16, width=40)
    q = _q(batch, 2, d, torch.float16)
    _check(_run(q, k, v, table, q_start, kv_len, max_q=1), q, k, v, table, q_start, kv_len)
    new = [(20 if i % 97 == 5 else (i * 7) % 3) for i in range(batch)]
    lens = [n + (i * 13) % 40 for i, n in enumerate(new)]
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, torch.float16, width=300)
    q = _q(sum(new), 2, d, torch.float16)
    _check(_run(q, k, v, table, q_start, kv_len, max_q=20), q, k, v, table, q_start, kv_len)


def test_the_same_memory_for_queries_and_output():
    for new, lens in (([1, 1, 1], [700, 40, 1300]), ([40, 1], [90, 60]), ([40], [5000])):
        k, v, table, q_start, kv_len = R.make_batch(new, lens, 16, 1, 128, torch.bfloat16)
        q = _q(sum(new), 2, 128, torch.bfloat16)
        from llcompiler_b200.executor import paged_attention
        dev = q.to(DEV)
        got = paged_attention(dev, *(t.to(DEV) for t in (k, v, table, q_start, kv_len)), max_q=max(new), out=dev)
        assert got is dev
        _check(dev, q, k, v, table, q_start, kv_len)


def test_other_streams():
    k, v, table, q_start, kv_len = R.make_batch([1] * 6, [900, 20, 450, 3, 1500, 64], 16, 2, 128, torch.bfloat16)
    q = _q(6, 8, 128, torch.bfloat16)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append(_run(q, k, v, table, q_start, kv_len, max_q=1))
    torch.cuda.synchronize()
    _check(outs[0], q, k, v, table, q_start, kv_len)
    assert all(torch.equal(o, outs[0]) for o in outs)          # and the sums do not depend on who runs beside them


def test_a_prompt_and_the_tokens_after_it_as_a_layer_uses_them():
    """QKV projection (this library's GEMM), append, attention, output projection: a prompt in two chunks, then single tokens,
    against dense causal attention in 64 bits over the whole sequence."""
    import gpu_ops as G
    from llcompiler_b200.executor import kv_append, paged_attention
    heads, kv_heads, d, page, hidden, total = 4, 2, 64, 16, 256, 90
    g = torch.Generator().manual_seed(4)
    x = torch.randn(total, hidden, generator=g).to(torch.bfloat16)
    w_qkv = (torch.randn((heads + 2 * kv_heads) * d, hidden, generator=g) / 16).to(torch.bfloat16)
    w_out = (torch.randn(hidden, heads * d, generator=g) / 16).to(torch.bfloat16)
    freq = R.inv_freq(d // 2)
    kc = torch.full((8, page, kv_heads, d), float("nan"), device=DEV, dtype=torch.bfloat16)
    vc = torch.full_like(kc, float("nan"))
    table = torch.tensor([[5, 0, 7, 2, 6, 1]], dtype=torch.int32, device=DEV)
    wq, wo, fd = w_qkv.to(DEV), w_out.to(DEV), freq.to(DEV)
    rows, contexts = [], []
    at = 0
    for n in [41, 30] + [1] * 19:
        xs = x[at : at + n].to(DEV)
        qkv = torch.empty(n, heads + 2 * kv_heads, d, device=DEV, dtype=torch.bfloat16)
        G.gemm(xs[None, None], wq.t()[None, None], qkv.view(1, 1, n, -1), prec="bf16")
        q_start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        kv_len = torch.tensor([at + n], dtype=torch.int32, device=DEV)
        q = kv_append(qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :], kc, vc, table, q_start, kv_len, q=qkv[:, :heads], inv_freq=fd)
        ctx = paged_attention(q, kc, vc, table, q_start, kv_len, max_q=n)
        y = torch.empty(n, hidden, device=DEV, dtype=torch.bfloat16)
        G.gemm(ctx.view(1, 1, n, -1), wo.t()[None, None], y[None, None], prec="bf16")
        rows.append(y)
        contexts.append(ctx)
        at += n
    got = torch.cat(rows).double().cpu()
    qkv = (x.double() @ w_qkv.double().t()).view(total, heads + 2 * kv_heads, d)
    pos = torch.arange(total)[None]
    q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
    q, k = R.rotary(q, pos, freq, [d // 2], False)[0], R.rotary(k, pos, freq, [d // 2], False)[0]
    k, v = (t.repeat_interleave(heads // kv_heads, 1) for t in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * R.scale_of(d)
    s = s.masked_fill(torch.ones(total, total).triu(1).bool(), float("-inf"))
    ctx = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v)
    want = ctx.reshape(total, -1) @ w_out.double().t()
    # Roundings to bf16 (u = 2^-8 of the value at most): q twice, k twice, v, the weights, the context, the result.  A score of
    # size |s| <= sum |q k| scale ~ 6 moves by 4 u of it at most, so a weight by 24 u at worst and by about a tenth of that in
    # the mean, where the 64 signs are independent; relative to the norm of the whole result the sum of all stays below 4 u.
    assert float((got - want).norm() / want.norm()) < 4 * 2.0 ** -8


def test_python_entry_points_refuse_what_does_not_fit():
    from llcompiler_b200.executor import kv_append, paged_attention, rotary
    k, v, table, q_start, kv_len = (t.to(DEV) for t in R.make_batch([3], [20], 16, 2, 64, torch.bfloat16))
    q, new = torch.zeros(3, 4, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(3, 2, 64, device=DEV, dtype=torch.bfloat16)
    freq, pos = R.inv_freq(32).to(DEV), torch.arange(3, device=DEV)
    refused = [
        lambda: paged_attention(q.float(), k, v, table, q_start, kv_len),
        lambda: paged_attention(q.requires_grad_(), k, v, table, q_start, kv_len),
        lambda: paged_attention(q.detach()[:, :3], k, v, table, q_start, kv_len),
        lambda: paged_attention(q.detach(), k, v, table.long(), q_start, kv_len),
        lambda: paged_attention(q.detach(), k, v, table, q_start[:1], kv_len),
        lambda: paged_attention(q.detach(), k, v[:, :8], table, q_start, kv_len),
        lambda: paged_attention(q.detach(), k, v, table, q_start, kv_len.cpu()),
        lambda: paged_attention(q.detach(), k, v, table, q_start, kv_len, window=-1),
        lambda: paged_attention(q.detach(), k, v, table, q_start, kv_len, max_q=-1),
        lambda: paged_attention(q.detach(), k, v, table, q_start, kv_len, out=new),
        lambda: paged_attention(q.detach(), k, v, table, q_start, kv_len, out=q.detach()[:1].expand(3, 4, 64)),
        lambda: paged_attention(q.detach(), k.transpose(2, 3), v.transpose(2, 3), table, q_start, kv_len),
        lambda: kv_append(new, new[:2], k, v, table, q_start, kv_len),
        lambda: kv_append(new, new, k, v, table, q_start, kv_len, positions=pos),
        lambda: kv_append(new, new, k, v, table, q_start, kv_len, q_out=q.detach()),
        lambda: kv_append(new, new, k, v, table, q_start, kv_len, inv_freq=freq.float()),
        lambda: kv_append(new, new, k, v, table, q_start, kv_len, inv_freq=freq, sections=[16, 15]),
        lambda: rotary(new, pos[:2], freq),
        lambda: rotary(new, pos.float(), freq),
        lambda: rotary(new, pos, torch.cat([freq, freq])),
        lambda: rotary(new, None, freq),
        lambda: rotary(new.to(torch.int32), pos, freq),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)
