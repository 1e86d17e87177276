"""Attention over the paged cache where rows, values or tables are not ordinary: NaN and infinite rows, tables much wider than the sequences,
wide groups, captured chunks."""
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


def _owned(q_start, tokens):
    t = torch.arange(tokens)
    return (t >= int(q_start[0])) & (t < int(q_start[-1]))


# the forms of the call: new tokens, lengths, heads, kv heads, d, page, type
FORMS = {
    "chunk": ([40, 33], [300, 90], 2, 1, 128, 64, torch.bfloat16),
    "chunk_whole_blocks": ([200], [700], 4, 1, 64, 16, torch.float16),
    "chunk_cut": ([40], [5000], 2, 1, 128, 64, torch.bfloat16),
    "chunk_cut_d64": ([70, 66], [4000, 4200], 2, 2, 64, 32, torch.float16),
    "decode": ([1, 1, 1], [77, 200, 16], 8, 2, 128, 16, torch.bfloat16),
    "decode_cut": ([1, 2], [5000, 700], 4, 1, 64, 64, torch.float16),
    "decode_cut_long": ([3], [40000], 4, 1, 128, 64, torch.bfloat16),
    "plain_f32": ([3, 1], [50, 40], 4, 2, 64, 16, torch.float32),
    "plain_d80": ([3, 1], [50, 40], 4, 2, 80, 16, torch.bfloat16),
}


@pytest.mark.parametrize("form", FORMS)
def test_a_nan_query_is_nan_in_its_own_rows_only(form):
    new, lens, heads, kv_heads, d, page, dtype = FORMS[form]
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype)
    q = _q(sum(new) + 1, heads, d, dtype)
    clean = _run(q, k, v, table, q_start, kv_len, max_q=max(new))
    row = int(q_start[len(new) // 2])
    q2 = q.clone()
    q2[row, heads - 1] = float("nan")
    got = _run(q2, k, v, table, q_start, kv_len, max_q=max(new))
    assert got[row, heads - 1].isnan().all()
    rest = _owned(q_start, len(q))[:, None].expand(-1, heads).clone()
    rest[row, heads - 1] = False
    assert torch.equal(got.cpu()[rest], clean.cpu()[rest]) and torch.isfinite(clean.cpu()[rest].float()).all()


@pytest.mark.parametrize("form", ["chunk_cut", "chunk_cut_d64", "decode_cut"])
@pytest.mark.parametrize("first", [True, False])
def test_a_part_of_the_keys_that_is_nan_makes_its_rows_nan(form, first):
    """Scores that are NaN from the first key on, up to every block's end (one of them is where the first part ends), or in the last keys
    before the new tokens."""
    from llcompiler_b200.executor import paged_attention
    new, lens, heads, kv_heads, d, page, dtype = FORMS[form]
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype)
    dev = [R.to_device(t, DEV) for t in (_q(sum(new), heads, d, dtype), k, v, table, q_start, kv_len)]
    step = 128 if "chunk" in form else 16
    last = (lens[0] - new[0]) // step
    for i in range(last):
        for j in range(i * step, (i + 1) * step) if first else range((last - 1 - i) * step, (last - i) * step):
            if j % page == 0 or j % step == 0:
                dev[1][int(table[0, j // page]), j % page : min(page, j % page + step)] = float("nan")
        got = paged_attention(*dev, max_q=max(new))
        assert got[: new[0]].isnan().all() and torch.isfinite(got[new[0] :].float()).all(), i


def _against_definition(got, q, k, v, table, q_start, kv_len, window=0, sinks=0, scale=None):
    """NaN where the definition has NaN, infinities where it has them, the rest within the tolerance (scores of infinite size are exact:
    they weigh nothing)."""
    scale = R.scale_of(q.shape[2]) if scale is None else scale
    want, size, _ = R.attention(q, k, v, table, q_start, kv_len, scale, window, sinks)
    finite_k, finite_v = (torch.where(torch.isfinite(t), t, torch.zeros((), dtype=t.dtype)) for t in (k, v))
    _, _, largest = R.attention(q, finite_k, finite_v, table, q_start, kv_len, scale, window, sinks)
    owned, got = _owned(q_start, len(q)), got.double().cpu()
    want, got = want[owned], got[owned]
    assert torch.equal(want.isnan(), got.isnan()), "NaN elsewhere"
    ends = want.isinf()
    assert torch.equal(want[ends], got[ends])
    f = torch.isfinite(want)
    tol = R.attention_tolerance(want, size[owned], largest, q.dtype)
    assert ((got - want).abs() <= tol)[f].all(), float(((got - want).abs() / tol)[f].max())


@pytest.mark.parametrize("form", [f for f in FORMS if f != "decode_cut_long"])   # the definition is slow to restate over so many keys
@pytest.mark.parametrize("window", [0, 9])
def test_rows_that_see_only_minus_infinity_are_nan_and_rows_that_see_nothing_zero(form, window):
    """softmax of -inf alone is 0 / 0, in every kernel; a token without a visible key has zeros."""
    new, lens, heads, kv_heads, d, page, dtype = FORMS[form]
    for hide in ("all", "some", "few"):
        k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype)
        q = _q(sum(new), heads, d, dtype).abs()               # positive: the product with a key of -inf is -inf
        for j in range(lens[0] if hide == "all" else lens[0] - (new[0] + 1) // 2 if hide == "some" else 20):
            k[int(table[0, j // page]), j % page] = float("-inf")
        if hide == "few" and len(new) > 1:
            kv_len[1] = new[1] // 2                           # the first of sequence 1's tokens see nothing
        got = _run(q, k, v, table, q_start, kv_len, window, max_q=max(new))
        _against_definition(got, q, k, v, table, q_start, kv_len, window)


@pytest.mark.parametrize("new,lens,heads,kv_heads,d,page,dtype", [([40], [500], 2, 1, 128, 64, torch.float16), ([33, 70, 64], [900, 1535, 70], 2, 2, 64, 16, torch.float16),
                                                                  ([40, 50], [5000, 300], 2, 1, 128, 64, torch.bfloat16), ([90], [1537], 1, 1, 64, 16, torch.float16)])
def test_the_table_of_a_chunk_may_be_as_wide_as_a_server_likes(new, lens, heads, kv_heads, d, page, dtype):
    """The keys are cut by the sequences' lengths: a table for 128 times the keys gives the same sums, bit for bit."""
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype)
    q = _q(sum(new), heads, d, dtype)
    tight = _run(q, k, v, table, q_start, kv_len, max_q=max(new))
    wide = torch.full((len(new), 64 * table.shape[1]), -1, dtype=torch.int32)
    wide[:, : table.shape[1]] = table
    got = _run(q, k, v, wide, q_start, kv_len, max_q=max(new))
    assert torch.equal(got, tight)
    _against_definition(got, q, k, v, table, q_start, kv_len)


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
@pytest.mark.parametrize("new,lens,heads,kv_heads,d,page,dtype", [([40, 33], [300, 90], 2, 1, 128, 64, torch.bfloat16), ([200], [700], 4, 1, 64, 16, torch.float16),
                                                                  ([40], [5000], 2, 1, 128, 64, torch.bfloat16), ([3, 4], [300, 90], 4, 2, 64, 16, torch.float16)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(window, sinks, new, lens, heads, kv_heads, d, page, dtype):
    """Single elements of the values, of tokens before the chunk and in it: NaN, +inf, -inf and both in a column."""
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype)
    q = _q(sum(new), heads, d, dtype)
    n, length = new[0], lens[0]
    at = lambda j: (int(table[0, j // page]), j % page)
    for j, col, what in ((0, 0, "inf"), (length - n - 1, 5, "nan"), (length - n, 9, "-inf"), (length - n // 2, 9, "-inf"), (length - n // 2, 20, "inf"), (length - 1, 20, "nan"),
                         (length - 1, 33, "inf"), (length - 2, 33, "-inf"), (length - n // 2 - 1, 40, "nan"), (length - 1, 40, "inf"), (length - n, 50, "nan")):
        v[at(j)][kv_heads - 1, col] = float(what)
    got = _run(q, k, v, table, q_start, kv_len, window, sinks, max_q=max(new))
    _against_definition(got, q, k, v, table, q_start, kv_len, window, sinks)


def _ms(call, reps=5):
    call()
    times = []
    for _ in range(reps):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return sorted(times)[reps // 2]


@pytest.mark.parametrize("where", ["early", "every", "chunk"])
def test_values_that_are_not_finite_do_not_stop_a_chunk(where):
    """An infinite value of the prompt's beginning is in the result of every later row, and so is a NaN of all values: neither needs a row's
    sum again.  Rows before the value's token in its own tile do: 16 a warp over 4096 keys, 65536 dot products of some 40 instructions, eight
    warps on four schedulers: 5.2 million issue slots at least, 2.8 ms."""
    from llcompiler_b200.executor import paged_attention
    new, length, heads, kv_heads, d, page = 512, 4096, 4, 1, 128, 64
    k, v, table, q_start, kv_len = (t.to(DEV) for t in R.make_batch([new], [length], page, kv_heads, d, torch.bfloat16))
    q = _q(new, heads, d, torch.bfloat16).to(DEV)
    clean = _ms(lambda: paged_attention(q, k, v, table, q_start, kv_len))
    if where == "every":
        v.fill_(float("nan"))
    else:
        j = 3 if where == "early" else length - new + 40
        v[int(table[0, j // page]), j % page, 0, 7] = float("inf")
    out = paged_attention(q, k, v, table, q_start, kv_len)
    assert out.isnan().all() if where == "every" else out[..., 7].isinf().all() if where == "early" else out[40:, :, 7].isinf().all() and torch.isfinite(out[:40].float()).all()
    slow = _ms(lambda: paged_attention(q, k, v, table, q_start, kv_len), 3)
    assert slow < 4 * clean + (0.05 if where != "chunk" else 10.0), (clean, slow)


def _tight_tolerance(want, size, largest, dtype):
    """R.attention_tolerance without the polynomial exponentials, which only the chunk kernel has: one rounding of the result and one of each
    weight (16-bit types), scores off by at most d 2^-23 of the largest sum |q k|, twice, and 2^-18 for the hardware's exponential
    and the sums of weights."""
    u, d = torch.finfo(dtype).eps / 2, want.shape[-1]
    return want.abs() * u * (1 + 2.0 ** -7) + size * (u + 2 * largest * d * 2.0 ** -23 + 2.0 ** -18) + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("new,lens,heads,kv_heads,d,page,dtype", [
    ([1, 1, 1], [1, 64, 300], 8, 2, 128, 16, torch.float16), ([1, 1], [5000, 700], 4, 1, 64, 64, torch.float16), ([2, 3], [517, 90], 10, 2, 128, 32, torch.float16),
    ([1, 4], [1300, 64], 8, 1, 64, 16, torch.bfloat16), ([3, 1], [50, 400], 4, 2, 64, 16, torch.float32), ([2], [900], 4, 2, 128, 16, torch.float32),
    ([3, 1], [50, 400], 4, 2, 80, 16, torch.float16), ([2], [200], 2, 1, 256, 16, torch.float32)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5)])
def test_decoding_and_plain_kernels_keep_the_bound_without_polynomials(new, lens, heads, kv_heads, d, page, dtype, window, sinks):
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype, fill=float("nan"))
    q = _q(sum(new), heads, d, dtype)
    got = _run(q, k, v, table, q_start, kv_len, window, sinks, max_q=max(new))
    want, size, largest = R.attention(q, k, v, table, q_start, kv_len, R.scale_of(d), window, sinks)
    off, tol = (got.double().cpu() - want).abs(), _tight_tolerance(want, size, largest, dtype)
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("new,lens,heads,kv_heads,width", [
    ([1, 40, 1], [300, 200, 77], 20, 1, 300), ([1, 3, 1, 0], [4700, 60, 5, 9], 32, 1, 300), ([1, 50, 2], [90, 60, 40], 34, 2, 260),      # 17 to 32 heads, beside chunks
    ([1], [77], 40, 1, 5), ([1, 1, 50], [300, 5, 60], 40, 1, 300), ([2, 1], [300, 200], 66, 2, 300), ([1, 2], [2000, 31], 128, 1, 130)])  # more than 32
@pytest.mark.parametrize("d", [64, 128])
def test_wide_groups(new, lens, heads, kv_heads, width, d):
    k, v, table, q_start, kv_len = R.make_batch(new, lens, 16, kv_heads, d, torch.bfloat16, width=width, fill=float("nan"))
    q = _q(sum(new) + 2, heads, d, torch.bfloat16)
    for window, sinks in ((0, 0), (30, 4)):
        out = torch.full(q.shape, 5.0, device=DEV, dtype=torch.bfloat16)
        _run(q, k, v, table, q_start, kv_len, window, sinks, max_q=max(new), out=out)
        assert (out[sum(new) :] == 5).all()
        _against_definition(out, q, k, v, table, q_start, kv_len, window, sinks)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_captured_chunks_replay_with_other_lengths(dtype, d):
    """A step of chunks captured once: replayed with longer and shorter caches (cut and not), other shares of the rows, and rows of nobody."""
    from llcompiler_b200.executor import paged_attention
    rows, heads, kv_heads, page, max_q = 96, 4, 2, 16, 70
    k, v, table, _, _ = R.make_batch([1, 1, 1], [5000, 5000, 400], page, kv_heads, d, dtype)
    dev = [t.to(DEV) for t in (k, v, table)]
    q = _q(rows, heads, d, dtype).to(DEV)
    q_start, kv_len = torch.tensor([0, 40, 70, 96], dtype=torch.int32, device=DEV), torch.tensor([60, 300, 26], dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    step = lambda: paged_attention(q, *dev, q_start, kv_len, max_q=max_q, out=out)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for ends, lens in (([0, 40, 70, 96], [60, 300, 26]), ([0, 70, 70, 70], [5000, 9, 400]), ([0, 33, 66, 90], [4990, 4991, 33]), ([3, 4, 5, 40], [900, 5000, 300]), ([0, 0, 0, 0], [0, 5, 9])):
        q_start.copy_(torch.tensor(ends, dtype=torch.int32))
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(_q(rows, heads, d, dtype, seed=sum(lens)))
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        owned = _owned(q_start.cpu(), rows)
        assert (out.cpu()[~owned] == 5).all()
        _against_definition(out, q.cpu(), k, v, table, q_start.cpu(), kv_len.cpu())


@pytest.mark.parametrize("form", FORMS)
def test_two_runs_give_the_same_bits(form):
    new, lens, heads, kv_heads, d, page, dtype = FORMS[form]
    k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype)
    q = _q(sum(new), heads, d, dtype)
    first = _run(q, k, v, table, q_start, kv_len, max_q=max(new))
    for _ in range(5):
        assert torch.equal(_run(q, k, v, table, q_start, kv_len, max_q=max(new)), first)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_tensors_of_another_device_than_the_current_one():
    from llcompiler_b200.executor import device_status, kv_append, paged_attention, rotary
    other = torch.device("cuda", 1)
    for new, lens in (([1, 1], [300, 77]), ([40], [300])):
        k, v, table, q_start, kv_len = R.make_batch(new, lens, 16, 2, 64, torch.bfloat16)
        q = _q(sum(new), 4, 64, torch.bfloat16)
        kc, vc = k.to(other), v.to(other)
        args = [t.to(other) for t in (table, q_start, kv_len)]
        fresh = _q(sum(new), 2, 64, torch.bfloat16, seed=2)
        kv_append(fresh.to(other), fresh.to(other), kc, vc, *args)
        got = paged_attention(q.to(other), kc, vc, *args, max_q=max(new))
        assert got.device == other and torch.cuda.current_device() == 0
        _against_definition(got, q, kc.cpu(), vc.cpu(), table, q_start, kv_len)
        pos, freq = torch.arange(sum(new)), R.inv_freq(32)
        assert torch.equal(rotary(q.to(other), pos.to(other), freq.to(other)).cpu(), rotary(q.to(DEV), pos.to(DEV), freq.to(DEV)).cpu())
        assert device_status(other) == 0


@pytest.mark.parametrize("form", FORMS)
def test_row_starts_that_do_not_grow_stay_inside(form):
    """Starts in any order name no rows, the wrong ones or the same ones twice; places stay inside the table and rows inside the tensors."""
    from llcompiler_b200.executor import kv_append
    _, _, heads, kv_heads, d, page, dtype = FORMS[form]
    reach = 4 * page                                          # every sequence fills its row of the table, the last one at the table's end
    k, v, table, _, kv_len = R.make_batch([1, 1, 1], [reach] * 3, page, kv_heads, d, dtype, spare=0)
    q = _q(8, heads, d, dtype)
    fresh = _q(8, kv_heads, d, dtype, seed=3).to(DEV)
    for starts in ([0, 9, 1, 2], [0, 8, 1, 2], [5, 2, 7, 1], [0, 1, 0, 8], [-4, 3, -9, 100], [8, 8, 0, 0], [7, -1, 6, 2]):
        for max_q in (1, 3, 8):
            out = torch.full(q.shape, 5.0, device=DEV, dtype=dtype)
            _run(q, k, v, table, torch.tensor(starts, dtype=torch.int32), kv_len, max_q=max_q, out=out)
            assert torch.isfinite(out.float()).all()
        dev = [R.to_device(t, DEV) for t in (k, v, table, torch.tensor(starts, dtype=torch.int32), kv_len)]
        kv_append(fresh, fresh, *dev, bad_pages=torch.zeros(1, device=DEV, dtype=torch.int32))
        assert torch.isfinite(dev[0].float()).all()


@pytest.mark.parametrize("form", [f for f in FORMS if f != "decode_cut_long"])
def test_rows_that_see_plus_infinity_are_nan(form):
    """inf - inf, as softmax has it: whichever block or part the score is in, beside finite ones and beside -inf."""
    new, lens, heads, kv_heads, d, page, dtype = FORMS[form]
    for at in (0, lens[0] // 2, lens[0] - 1):
        k, v, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype)
        q = _q(sum(new), heads, d, dtype).abs()
        k[int(table[0, at // page]), at % page] = float("inf")
        if at:
            k[int(table[0, 0]), 0] = float("-inf")
        got = _run(q, k, v, table, q_start, kv_len, max_q=max(new))
        _against_definition(got, q, k, v, table, q_start, kv_len)


def test_chunks_single_tokens_and_matrix_products_at_once():
    """Calls on streams of their own share SMs, tensor memory and the allocator: each gives what it gives alone."""
    import gpu_ops as G
    calls = []
    for new, lens, heads, kv_heads, d, page, dtype in (FORMS["chunk_whole_blocks"], FORMS["chunk_cut"], FORMS["chunk_cut_d64"], FORMS["decode_cut"], FORMS["decode"]):
        from llcompiler_b200.executor import paged_attention
        dev = [R.to_device(t, DEV) for t in (_q(sum(new), heads, d, dtype), *R.make_batch(new, lens, page, kv_heads, d, dtype))]
        calls.append(lambda dev=dev, n=max(new): paged_attention(*dev, max_q=n))
    a, b = (torch.randn(512, 512, generator=torch.Generator().manual_seed(i)).to(DEV, torch.bfloat16) for i in range(2))

    def product():
        y = torch.empty(512, 512, device=DEV, dtype=torch.bfloat16)
        G.gemm(a[None, None], b.t()[None, None], y[None, None], prec="bf16")
        return y
    calls.append(product)
    alone = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(20):
        for i, (c, st) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(st):
                got[i].append(c())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for gs, want in zip(got, alone) for g in gs)
