"""Rotary positions and the writing side of the paged cache against their definitions in 64 bits."""
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _x(tokens, heads, d, dtype, seed=0):
    return torch.randn(tokens, heads, d, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _check(got, want, tol):
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), float((off / tol.clamp(min=1e-300)).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,d,sections,base_pos", [
    (1, 1, 64, [32], 0), (1, 48, 128, [64], 131071), (7, 3, 64, [16, 16], 5), (130, 12, 128, [16, 24, 24], 70000),
    (33, 5, 128, [10, 20, 2], 12345678), (17, 2, 80, [7, 5, 3, 1], 1000), (5, 3, 34, [17], 31), (2500, 4, 64, [0, 32], 9), (3, 1, 2, [1], 3),
])
def test_rotary(dtype, interleaved, tokens, heads, d, sections, base_pos):
    from llcompiler_b200.executor import rotary
    x = _x(tokens, heads, d, dtype)
    g = torch.Generator().manual_seed(1)
    pos = torch.randint(0, 4000, (len(sections), tokens), generator=g) + base_pos
    freq = R.inv_freq(sum(sections))
    want, size = R.rotary(x, pos, freq, sections, interleaved)
    tol = R.rotary_tolerance(want, size, dtype)
    for pt in (torch.int64, torch.int32):
        got = rotary(x.to(DEV), pos.to(DEV, pt), freq.to(DEV), sections=sections, interleaved=interleaved)
        _check(got, want, tol)


def test_rotary_of_strided_views_in_place_and_with_negative_positions():
    from llcompiler_b200.executor import rotary
    tokens, heads, d = 37, 6, 64
    freq = R.inv_freq(32)
    pos = torch.arange(tokens)[None] - 20
    for shift in (0, 1):                       # a base that is not 16-byte aligned takes single elements
        whole = torch.randn(tokens * 3 * heads * d + 8, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        view = whole[shift : shift + tokens * 3 * heads * d].view(tokens, 3, heads, d)[:, 1]
        want, size = R.rotary(view, pos, freq, [32], False)
        dev = whole.to(DEV)
        x = dev[shift : shift + tokens * 3 * heads * d].view(tokens, 3, heads, d)[:, 1]
        got = rotary(x, pos[0].to(DEV), freq.to(DEV), out=x)
        assert got is x
        _check(x, want, R.rotary_tolerance(want, size, torch.bfloat16))
        keep = torch.ones(tokens, 3, heads, d, dtype=torch.bool)
        keep[:, 1] = False
        same = dev[shift : shift + tokens * 3 * heads * d].view(tokens, 3, heads, d).cpu()[keep]
        assert torch.equal(same, whole[shift : shift + tokens * 3 * heads * d].view(tokens, 3, heads, d)[keep])
    # heads before tokens
    x = _x(heads, tokens, d, torch.float16).transpose(0, 1)
    out = torch.empty(heads, tokens, d, device=DEV, dtype=torch.float16).transpose(0, 1)
    want, size = R.rotary(x, pos, freq, [32], True)
    rotary(R.to_device(x, DEV), pos.to(DEV), freq.to(DEV), interleaved=True, out=out)
    _check(out, want, R.rotary_tolerance(want, size, torch.float16))


def test_rotary_far_positions_keep_their_angle():
    """At position 2^30 a product in 32 bits is off by whole turns."""
    from llcompiler_b200.executor import rotary
    x = _x(4, 2, 64, torch.float32)
    pos = torch.tensor([[2 ** 30 + 1, 2 ** 31 - 1, 2 ** 24 + 1, 999999937]])
    freq = R.inv_freq(32, 500000.0)
    want, size = R.rotary(x, pos, freq, [32], False)
    # the reference's own angle is rounded once in 64 bits: 2^31 2^-53 radians, below 2^-24 |x|
    _check(rotary(x.to(DEV), pos.to(DEV), freq.to(DEV)), want, R.rotary_tolerance(want, size, torch.float32))


APPEND = [
    # new tokens, lengths, heads, kv heads, d, page, heads first, type
    ([1], [1], 4, 2, 64, 16, False, torch.bfloat16),
    ([1] * 40, list(range(1, 41)), 8, 8, 128, 16, False, torch.float16),
    ([5, 0, 33, 1, 16], [5, 7, 100, 64, 31], 12, 4, 64, 32, True, torch.bfloat16),
    ([200, 3], [333, 3], 3, 1, 128, 64, False, torch.float32),
    ([9, 2], [20, 11], 2, 2, 34, 7, True, torch.float32),
    ([0, 0], [3, 0], 2, 2, 64, 16, False, torch.bfloat16),
]


@pytest.mark.parametrize("new,lens,heads,kv_heads,d,page,heads_first,dtype", APPEND)
@pytest.mark.parametrize("turn", ["none", "places", "axes"])
def test_append_writes_the_new_tokens_and_nothing_else(new, lens, heads, kv_heads, d, page, heads_first, dtype, turn):
    from llcompiler_b200.executor import kv_append
    k_cache, v_cache, table, q_start, kv_len = R.make_batch(new, lens, page, kv_heads, d, dtype, heads_first=heads_first)
    tokens, pad = sum(new), 3                                  # three rows behind the last sequence
    qkv = _x(tokens + pad, heads + 2 * kv_heads, d, dtype, seed=5)
    q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
    pairs = d // 2
    sections = [pairs] if turn != "axes" else [pairs - 2 * (pairs // 3), pairs // 3, pairs // 3]
    freq = R.inv_freq(pairs)
    place = torch.cat([torch.arange(b - a, b) for a, b in zip(new, lens)] + [torch.zeros(pad, dtype=torch.long)]).long()
    pos = place[None] if turn != "axes" else torch.stack([place // 4 + 7, place % 4, place % 9])
    want_k, size_k = R.rotary(k, pos, freq, sections, False) if turn != "none" else (k.double(), torch.zeros(k.shape).double())
    want_q, size_q = R.rotary(q, pos, freq, sections, False) if turn != "none" else (q.double(), torch.zeros(q.shape).double())
    dev = qkv.to(DEV)
    kc, vc = R.to_device(k_cache, DEV), R.to_device(v_cache, DEV)
    q_out = torch.full((tokens + pad, heads, d), 7.0, device=DEV, dtype=dtype)
    bad = torch.zeros(1, device=DEV, dtype=torch.int32)
    more = {} if turn == "none" else {"inv_freq": freq.to(DEV), "sections": sections}
    if turn == "axes":
        more["positions"] = pos.to(DEV)
    got = kv_append(dev[:, heads : heads + kv_heads], dev[:, heads + kv_heads :], kc, vc, table.to(DEV), q_start.to(DEV), kv_len.to(DEV), q=dev[:, :heads],
                    q_out=q_out, bad_pages=bad, **more)
    assert got is q_out and int(bad) == 0
    assert (q_out[tokens:] == 7).all()
    _check(q_out[:tokens], want_q[:tokens], R.rotary_tolerance(want_q, size_q, dtype)[:tokens])
    row = 0
    ref_k, ref_v, tol_k = k_cache.double(), v_cache.double(), torch.zeros(k_cache.shape).double()
    for b, (n, length) in enumerate(zip(new, lens)):
        for j in range(length - n, length):
            at = (int(table[b, j // page]), j % page)
            ref_k[at], ref_v[at] = want_k[row], v[row].double()
            tol_k[at] = R.rotary_tolerance(want_k[row], size_k[row], dtype) if turn != "none" else 0.0
            row += 1
    _check(kc, ref_k, tol_k)
    assert torch.equal(vc.cpu().double(), ref_v)
    # keys and values alone
    kc2, vc2 = R.to_device(k_cache, DEV), R.to_device(v_cache, DEV)
    assert kv_append(dev[:, heads : heads + kv_heads], dev[:, heads + kv_heads :], kc2, vc2, table.to(DEV), q_start.to(DEV), kv_len.to(DEV), **more) is None
    assert torch.equal(kc2, kc) and torch.equal(vc2, vc)


def test_append_counts_and_skips_what_has_no_slot():
    """Page numbers that are none of the pool's, places past the table, and more new tokens than the length says."""
    from llcompiler_b200.executor import kv_append
    k_cache, v_cache = torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64)
    table = torch.tensor([[0, -1], [4, 1], [2 ** 31 - 1, 3], [2, -2 ** 31]], dtype=torch.int32)
    q_start = torch.tensor([0, 2, 4, 5, 9], dtype=torch.int32)
    kv_len = torch.tensor([17, 17, 40, 2], dtype=torch.int32)      # 40: past the table's 32 slots, counts as 32
    k = torch.arange(1, 10).float()[:, None, None].expand(9, 2, 64)
    kc, vc = k_cache.to(DEV), v_cache.to(DEV)
    bad = torch.zeros(1, device=DEV, dtype=torch.int32)
    kv_append(k.to(DEV).contiguous(), -k.to(DEV).contiguous(), kc, vc, table.to(DEV), q_start.to(DEV), kv_len.to(DEV), bad_pages=bad)
    want = torch.zeros(4, 16, 2, 64)
    want[0, 15] = 1           # sequence 0: places 15, 16; the second page is -1
    want[1, 0] = 4            # sequence 1: places 15 (page 4 of 4), 16
    want[3, 15] = 5           # sequence 2: place 31
    want[2, 0], want[2, 1] = 8, 9   # sequence 3: four tokens, length 2: places -2, -1, 0, 1
    assert torch.equal(kc.cpu(), want) and torch.equal(vc.cpu(), -want)
    assert int(bad) == 1 + 1 + 2


def test_append_finds_the_sequence_in_large_batches():
    from llcompiler_b200.executor import kv_append
    for batch in (31, 32, 33, 1000, 1025, 3000):
        new = [(i * 7) % 4 for i in range(batch)]
        tokens = sum(new)
        q_start = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        table = torch.arange(batch, dtype=torch.int32)[:, None]
        kc = torch.zeros(batch, 4, 1, 8, device=DEV)
        vc = torch.zeros_like(kc)
        k = torch.arange(1, tokens + 1).float()[:, None, None].expand(tokens, 1, 8).contiguous().to(DEV)
        kv_append(k, k, kc, vc, table.to(DEV), q_start.to(DEV), torch.tensor(new, dtype=torch.int32).to(DEV))
        want = torch.zeros(batch, 4)
        row = 0
        for b, n in enumerate(new):
            for j in range(n):
                row += 1
                want[b, j] = row
        assert torch.equal(kc[:, :, 0, 3].cpu(), want) and torch.equal(vc, kc)
