"""GPU tests of the 4-bit cache against its fp64 definitions (tests/kv4_plain.py).

Tolerances count roundings, eps/2 of a type relative to the value (bf16 2^-8, fp16 2^-11, fp32
2^-24). Appended values are exact: codes, scales and zeros are the definition's, and what is read
back is one rounding of it to the output type. An attention output has
  * the rounding to its type, eps/2 |o|;
  * a rounding of each weight to at least 11 bits before the product with the values, 2^-11 of the
    sum of w |v|;
  * the error of a score, dx, which changes a weight by the factor e^dx and, with the sum of the
    weights, an output by at most 2 dx of the sum of w |v|. A score is a sum of 128 products in
    fp32, in any order, with each of the 128 partial sums rounded or cut (2^-23 of the sum of
    |q k|), then a few fp32 steps on values up to `spread`: dx <= 136 * 2^-23 * spread, and
    2^-21 for the exponential itself.
A code is subtracted from its zero after the sums: partial sums hold codes up to 15 where the
values have |code - zero|: `spread` counts 15/|code - zero|-fold there: 16 * spread bounds it for
every key whose values are not all 0, and tests draw no other.
  * the same for an output, which is a difference of two sums, of w code and of w zero. Both stay
    below 15 `step`, step the sum of w * value scale; each of the at most n / 8 + 64 partial sums
    of n tokens (one a product of 16 tokens and one a lane's token, then the joins of lanes, warps
    and pieces) is rounded or cut, 2^-23 of it: 2 * (n / 8 + 64) * 2^-23 * 15 * step. This is what
    is left where all values are 0 and the two sums should cancel.
"""
import math

import numpy as np
import pytest
import torch

from llm_fa_b200 import (KV4Cache, _lib, device_status, kv4_append, kv4_attention, kv4_evict_move,
                         kv4_evict_select, kv4_expand, reset_device_status)

from . import kv4_plain as plain

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half a step below the normal range, where steps no longer shrink: fp16's are 2^-24, bf16's 2^-133
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


@pytest.fixture(autouse=True)
def _clean_status():
    reset_device_status()
    yield
    reset_device_status()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(B, H, cap, page, group, seed=0, extra=2, fill=None):
    """A pool and a scattered page table of B sequences of `cap` slots."""
    width = -(-cap // page)
    cache = KV4Cache.empty(B * width + extra, H, page_size=page, group=group)
    if fill is not None:
        cache.pages.fill_(fill)
    gen = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * width + extra, generator=gen)[:B * width].reshape(B, width)
    return cache, table.to(torch.int32).cuda()


def randn(*shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def filled(B, H, lens, page, group, seed=0, dtype=torch.bfloat16, fill=0xff):
    """A pool whose sequences hold `lens` tokens; what no token holds is 0xff (NaN pairs)."""
    cap = max(max(lens), 1)
    cache, table = pool(B, H, cap, page, group, seed, fill=fill)
    k = randn(B, cap, H, 128, dtype=dtype, seed=seed + 1)
    k[..., 5] *= 9
    v = randn(B, cap, H, 128, dtype=dtype, seed=seed + 2)
    kv4_append(cache, k, v, table, ints([0] * B), counts=ints(lens))
    assert device_status() == 0
    return cache, table


def check_attention(got, q, cache, table, lens, counts, **kw):
    o, lse, w, mag, step, spread = plain.attention(
        q, cache.pages.cpu().numpy(), table.cpu().numpy(), lens, counts, page=cache.page_size,
        group=cache.group, heads=cache.heads, **kw)
    dx = 136 * 2.0 ** -23 * 16 * spread + 2.0 ** -21
    got_o = got[0].double().cpu().numpy()
    tol = HALF[q.dtype] * np.abs(o) * (1 + 2.0 ** -7) + (2.0 ** -11 + 2 * dx) * mag + 1e-30
    tol += TINY[q.dtype] + 2 * (max(lens) / 8 + 64) * 2.0 ** -23 * 15 * step
    live = ~np.isnan(o)
    err = np.abs(got_o - o)
    assert (err[live] <= tol[live]).all(), (err[live] - tol[live]).max()
    if len(got) > 1:
        got_l = got[1].double().cpu().numpy()
        live = ~np.isnan(lse)
        empty = live & np.isinf(lse)
        assert (got_l[empty] == -np.inf).all()
        live &= ~empty
        assert (np.abs(got_l[live] - lse[live]) <= 2 * dx + 2.0 ** -22 * np.abs(lse[live])).all()
    return w, dx


# ---------------------------------------------------------------- append and expand
@pytest.mark.parametrize("B,T,H,start,page,group,dtype", [
    (1, 1, 1, 0, 16, 128, torch.bfloat16),
    (3, 1, 8, 37, 64, 64, torch.bfloat16),
    (2, 33, 5, 15, 16, 32, torch.float16),
    (2, 300, 3, 250, 256, 128, torch.float16),
    (1, 1000, 2, 0, 32, 64, torch.bfloat16),
    (4, 17, 32, 127, 128, 32, torch.bfloat16),
])
def test_append_and_expand(B, T, H, start, page, group, dtype):
    cache, table = pool(B, H, start + T + 3, page, group, seed=T, fill=0x5a)
    before = cache.pages.clone()
    k, v = randn(B, T, H, 128, dtype=dtype, seed=1), randn(B, T, H, 128, dtype=dtype, seed=2)
    k[..., 7] *= 20
    v[0, 0, 0] = 0.0
    starts = [start + (b % 3) for b in range(B)]
    counts = [max(0, T - 2 * b) for b in range(B)]
    n, c = ints(starts), ints(counts)
    cache.weights.fill_(3.0)
    kv4_append(cache, k, v, table, n, counts=c, seen=ints([s + 1000 for s in starts]))
    gk, gv = kv4_expand(cache, table, n, T, counts=c, dtype=dtype)
    assert device_status() == 0
    touched = np.zeros(cache.pages.shape, bool)
    held = np.zeros(cache.positions.shape, bool)
    tab, pos, wts = table.cpu().numpy(), cache.positions.cpu().numpy(), cache.weights.cpu().numpy()
    pages = cache.pages.cpu().numpy()
    for value, (x, g) in enumerate(((k, gk), (v, gv))):
        want = plain.quantise(x.double().cpu().numpy(), group)[0]
        for b in range(B):
            want[b, counts[b]:] = 0.0
        assert torch.equal(g.cpu(), torch.as_tensor(want).to(dtype))
        for b in range(B):
            for t in range(counts[b]):
                s = starts[b] + t
                p = tab[b, s // page]
                at, pairs = plain.row_offset(s % page, value, group)
                touched[p, :, at:at + 64] = True
                touched[p, :, pairs:pairs + 4 * (128 // group)] = True
                held[p, :, s % page] = True
                assert (pos[p, :, s % page] == s + 1000).all()
                if t in (0, counts[b] - 1):
                    got = plain.read_token(pages[p, H - 1], s % page, value, group)
                    assert np.array_equal(got, want[b, t, H - 1])
    assert np.array_equal(pages[~touched], before.cpu().numpy()[~touched])
    assert (wts[held] == 0).all() and (wts[~held] == 3.0).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_at_the_borders_between_codes(group, dtype):
    """Ties between codes, one-sided groups, groups of one magnitude, and the ends of the types."""
    T = 64
    x = torch.zeros(1, T, 1, 128, dtype=torch.float64)
    grid = torch.arange(128, dtype=torch.float64)
    for t in range(T):
        s = 2.0 ** (t % 12 - 6)
        if t % 4 == 0:      # (hi - lo) / 15 = s exactly: halves of s are ties
            x[0, t, 0] = s * ((grid % 31) / 2 - 7.5) + 0.0
        elif t % 4 == 1:    # positive only
            x[0, t, 0] = s * (1 + (grid * 37 % 101) / 64)
        elif t % 4 == 2:    # negative only, one zero
            x[0, t, 0] = -s * ((grid * 29 % 61) / 16)
        else:               # one value against tiny ones
            x[0, t, 0] = s * 2.0 ** -6
            x[0, t, 0, ::32] = -s * 3.25
    big = 60000.0 if dtype == torch.float16 else 1.0e38
    x[0, 60], x[0, 61, 0, 1::2], x[0, 61, 0, ::2] = big, big, -big
    x[0, 62] = 6.0e-8 if dtype == torch.float16 else 2.0e-38
    x = x.to(dtype).cuda()
    cache, table = pool(1, 1, T, 16, group)
    kv4_append(cache, x, -x, table, ints([0]))
    gk, gv = kv4_expand(cache, table, ints([0]), T, dtype=dtype)
    xd = x.double().cpu().numpy()
    for g, y in ((gk, xd), (gv, -xd)):
        want = plain.quantise(y, group)[0]
        if dtype == torch.bfloat16:
            want[0, 62] = 0.0  # scale 2^-130: counts as 0
        assert torch.equal(g.cpu(), torch.as_tensor(want).to(dtype))


def test_append_non_finite_groups_read_back_as_nan():
    x = randn(1, 3, 1, 128)
    x[0, 0, 0, 3], x[0, 1, 0, 40], x[0, 2, 0, 127] = math.inf, math.nan, -math.inf
    cache, table = pool(1, 1, 3, 16, 32)
    kv4_append(cache, x, x, table, ints([0]))
    for g in kv4_expand(cache, table, ints([0]), 3):
        nan = g[0, :, 0].isnan().view(3, 4, 32)
        assert nan.all(-1).tolist() == [[True, False, False, False], [False, True, False, False],
                                        [False, False, False, True]]
        assert torch.equal(nan.any(-1), nan.all(-1))


def test_append_and_expand_strided_views():
    B, T, H = 2, 9, 3
    wide = randn(B, H + 1, T, 256, seed=5)
    k, v = wide[:, :H, :, :128].transpose(1, 2), wide[:, 1:, :, 128:].transpose(1, 2)
    n = ints([4, 0])
    got = []
    for a, b in ((k, v), (k.contiguous(), v.contiguous())):
        cache, table = pool(B, H, 32, 16, 64)
        kv4_append(cache, a, b, table, n)
        got.append(cache.pages)
    assert torch.equal(*got)
    o = torch.full((B, H, T, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    outs = (o[..., :128].transpose(1, 2), o[..., 128:].transpose(1, 2))
    kv4_expand(cache, table, n, T, out=outs)
    for a, b in zip(outs, kv4_expand(cache, table, n, T)):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("lens,T,Hq,H,page,group,dtype", [
    ([1], 1, 1, 1, 16, 128, torch.bfloat16),
    ([15, 16, 17], 1, 8, 8, 16, 64, torch.bfloat16),
    ([0, 31, 32, 33], 1, 4, 2, 32, 32, torch.float16),
    ([255, 1, 640], 1, 32, 4, 64, 128, torch.bfloat16),
    ([1000], 1, 64, 8, 64, 64, torch.bfloat16),
    ([3, 700, 129], 5, 16, 4, 16, 64, torch.float16),
    ([2, 65], 4, 6, 2, 256, 32, torch.bfloat16),
    ([513, 90], 3, 14, 2, 128, 128, torch.float16),
    ([300], 2, 33, 1, 16, 64, torch.bfloat16),
    ([200, 7], 40, 4, 1, 64, 64, torch.bfloat16),
    ([2500], 1, 16, 1, 128, 32, torch.bfloat16),
])
@pytest.mark.parametrize("causal", [True, False])
def test_attention(lens, T, Hq, H, page, group, dtype, causal):
    B = len(lens)
    cache, table = filled(B, H, lens, page, group, seed=sum(lens))
    q = randn(B, T, Hq, 128, dtype=dtype, seed=9)
    counts = [max(0, T - b) for b in range(B)]
    out = torch.full_like(q, 7.0)
    got = kv4_attention(q, cache, table, ints(lens), counts=ints(counts), causal=causal, out=out,
                        return_lse=True)
    assert device_status() == 0
    check_attention(got, q, cache, table, lens, counts, causal=causal)
    for b in range(B):  # rows past a count keep what they held
        assert (out[b, counts[b]:] == 7.0).all()
    again, lse = kv4_attention(q, cache, table, ints(lens), counts=ints(counts), causal=causal,
                               return_lse=True)
    for b in range(B):
        assert torch.equal(again[b, :counts[b]], out[b, :counts[b]])
        assert (again[b, counts[b]:] == 0).all() and (lse[b, :, counts[b]:] == -math.inf).all()
    assert torch.equal(lse, got[1])


@pytest.mark.parametrize("scale,seed", [(1.0, 1), (1e-3, 2), (0.5, 3)])
def test_attention_scales(scale, seed):
    """A peaked and a flat softmax, against the same definition."""
    lens = [777]
    cache, table = filled(1, 2, lens, 64, 64, seed=seed)
    q = randn(1, 1, 8, 128, seed=seed, scale=2.0)
    got = kv4_attention(q, cache, table, ints(lens), softmax_scale=scale, return_lse=True)
    check_attention(got, q, cache, table, lens, [1], scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_query_rows_of_very_different_size(dtype):
    lens = [300]
    cache, table = filled(1, 1, lens, 64, 64, seed=4)
    q = randn(1, 1, 8, 128, dtype=dtype, seed=5)
    size = torch.tensor([0.0, 1e-7, 1e-4, 1.0, 8.0, 1e-2, 3.0, 30.0]).cuda()
    q = (q.float() * size[None, None, :, None]).to(dtype)
    q[0, 0, 3, :64] *= 1e-3
    got = kv4_attention(q, cache, table, ints(lens), return_lse=True)
    check_attention(got, q, cache, table, lens, [1])


def test_attention_values_of_very_different_size():
    """Scales that grow and shrink by many powers of two along the sequence."""
    B, n = 1, 700
    cache, table = pool(B, 1, n, 16, 32, fill=0xff)
    k, v = randn(B, n, 1, 128, seed=1), randn(B, n, 1, 128, seed=2)
    size = 2.0 ** ((torch.arange(n) * 37 % 41) - 20.0)
    v = (v.float() * size.cuda()[None, :, None, None]).to(torch.bfloat16)
    v[0, ::3, 0, 32:64] *= 2.0 ** -30
    v[0, 5, 0] = 0.0
    kv4_append(cache, k, v, table, ints([0]))
    q = randn(B, 1, 4, 128, seed=3)
    got = kv4_attention(q, cache, table, ints([n]), return_lse=True)
    check_attention(got, q, cache, table, [n], [1])


def test_attention_non_finite_rows_and_tokens():
    lens = [100, 40]
    cache, table = filled(2, 2, lens, 16, 64, seed=6)
    q = randn(2, 2, 4, 128, seed=7)
    clean = kv4_attention(q, cache, table, ints(lens))
    q2 = q.clone()
    q2[0, 0, 1, 5], q2[0, 1, 2, 9] = math.inf, math.nan
    got = kv4_attention(q2, cache, table, ints(lens))
    assert got[0, 0, 1].isnan().all() and got[0, 1, 2].isnan().all()
    bad = torch.zeros(2, 2, 4, dtype=torch.bool)
    bad[0, 0, 1] = bad[0, 1, 2] = True
    assert torch.equal(got[~bad.cuda()], clean[~bad.cuda()])
    # a NaN in the values of one token reaches its group alone; of a masked token, nothing
    v = randn(2, 1, 2, 128, seed=8)
    v[0, 0, 1, 70] = math.nan
    kv4_append(cache, randn(2, 1, 2, 128, seed=9), v, table, ints([50, 39]))
    got = kv4_attention(q, cache, table, ints(lens))
    assert got[0, :, 2:, 64:].isnan().all() and not got[0, :, 2:, :64].isnan().any()
    assert not got[0, :, :2].isnan().any() and not got[1].isnan().any()
    assert not kv4_attention(q, cache, table, ints([50, 39])).isnan().any()


@pytest.mark.parametrize("lens,T,Hq,H,page,group", [
    ([1, 64, 300], 1, 8, 8, 64, 64), ([1000, 0], 1, 32, 4, 16, 128), ([90, 3], 4, 8, 2, 32, 32),
    ([150], 30, 8, 1, 64, 64),
])
@pytest.mark.parametrize("decay", [0.0, 0.75, 1.0])
def test_tracked_weights(lens, T, Hq, H, page, group, decay):
    B = len(lens)
    cache, table = filled(B, H, lens, page, group, seed=sum(lens))
    cache.weights.copy_(torch.rand(cache.weights.shape, generator=torch.Generator().manual_seed(1)))
    if decay == 0.0:
        cache.weights.fill_(math.nan)  # not read
    before = cache.weights.double().cpu().numpy()
    q = randn(B, T, Hq, 128, seed=9)
    counts = [max(0, T - b) for b in range(B)]
    got = kv4_attention(q, cache, table, ints(lens), counts=ints(counts), decay=decay, return_lse=True)
    assert device_status() == 0
    w, dx = check_attention(got, q, cache, table, lens, counts)
    after, tab = cache.weights.double().cpu().numpy(), table.cpu().numpy()
    held = np.zeros(before.shape, bool)
    rows = T * Hq // H
    for b, n in enumerate(lens):
        i = np.arange(n)
        old = before[tab[b, i // page], :, i % page] if decay else 0.0
        want = decay * old + w[b]
        new = after[tab[b, i // page], :, i % page]
        # each weight e^(2 dx) off, then an fp32 sum of rows + 1 terms
        assert (np.abs(new - want) <= 2 * dx * w[b] + (rows + 3) * 2.0 ** -24 * want + 1e-37).all()
        held[tab[b, i // page], :, i % page] = True
    assert np.array_equal(after[~held], before[~held], equal_nan=True)


@pytest.mark.parametrize("T,Hq,group", [(1, 8, 64), (3, 16, 32), (40, 8, 128)])
def test_tracked_weights_without_room_for_the_scores(T, Hq, group):
    """A page table so long that the scores are worked out again: the same weights."""
    lens, H, page = [700, 41], 2, 256
    cache, table = filled(2, H, lens, page, group, seed=5)
    wide = torch.full((2, (1 << 23) // page), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = randn(2, T, Hq, 128, seed=9)
    counts = [T, T - 1 if T > 1 else 1]
    tab = table.cpu().numpy()
    for tb in (table, wide):
        cache.weights.fill_(2.0)
        got = kv4_attention(q, cache, tb, ints(lens), counts=ints(counts), decay=0.5, return_lse=True)
        assert device_status() == 0
        w, dx = check_attention(got, q, cache, table, lens, counts)
        after = cache.weights.double().cpu().numpy()
        for b, n in enumerate(lens):
            i = np.arange(n)
            want = 1.0 + w[b]
            err = np.abs(after[tab[b, i // page], :, i % page] - want)
            assert (err <= 2 * dx * w[b] + (T * Hq // H + 3) * 2.0 ** -24 * want).all()


def test_attention_strided_views_and_repeated_pages():
    """q and out as slices of wider tensors; two sequences that read the same pages."""
    cache, table = filled(1, 2, [200], 16, 64, seed=3)
    table = table.expand(2, -1).contiguous()
    wide = randn(2, 3, 3, 8, 256, seed=4)
    q = wide[:, :, 1, :, 128:]
    out = torch.zeros(2, 4, 3, 256, dtype=torch.bfloat16, device="cuda")[..., :128].transpose(1, 2)
    got = kv4_attention(q[:, :, :4], cache, table, ints([200, 77]), out=out, return_lse=True)
    want = kv4_attention(q[:, :, :4].contiguous(), cache, table, ints([200, 77]))
    assert torch.equal(got[0], want)
    check_attention(got, q[:, :, :4], cache, table, [200, 77], [3, 3])
    pad = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    pad[:, :table.shape[1]] = table
    assert torch.equal(kv4_attention(q[:, :, :4], cache, pad, ints([200, 77])), want)
    assert torch.equal(kv4_attention(q[:, :, :4], cache, pad[:, :table.shape[1]], ints([200, 77])), want)
    assert device_status() == 0


def test_bad_pages_and_lengths_are_reported_and_skipped():
    H, page = 2, 16
    cache, table = filled(2, H, [64, 64], page, 64, seed=3)
    q = randn(2, 1, 4, 128, seed=4)
    want = kv4_attention(q, cache, table, ints([64, 48]))
    bad = table.clone()
    bad[1, 3] = cache.pages.shape[0]
    got = kv4_attention(q, cache, bad, ints([64, 64]))
    assert device_status() == _lib.DEVICE_STATUS_KV4_BAD_PAGE
    assert torch.equal(got[0], want[0])
    # the tokens of the bad page count as absent
    assert (got[1].float() - want[1].float()).abs().max() <= 2.0 ** -7 * want[1].float().abs().max()
    reset_device_status()
    got = kv4_attention(q, cache, table, ints([1000, -5]))
    assert device_status() == _lib.DEVICE_STATUS_KV4_BAD_LENGTH
    assert torch.equal(got[0], want[0]) and (got[1] == 0).all()
    reset_device_status()
    before = cache.pages.clone()
    x = randn(2, 4, H, 128, seed=5)
    kv4_append(cache, x, x, bad, ints([64, 50]))  # past the table, and on the bad page
    assert device_status() == _lib.DEVICE_STATUS_KV4_BAD_PAGE
    assert torch.equal(cache.pages, before)
    reset_device_status()
    kv4_append(cache, x, x, table, ints([-2, -1000]))  # would reach slots 0 and 1
    assert device_status() == _lib.DEVICE_STATUS_KV4_BAD_LENGTH
    assert torch.equal(cache.pages, before)
    reset_device_status()
    kv4_append(cache, x, x, table, ints([3, 4]), counts=ints([-1, 0]))
    assert device_status() == _lib.DEVICE_STATUS_KV4_BAD_LENGTH
    assert torch.equal(cache.pages, before)
    reset_device_status()
    k, v = kv4_expand(cache, bad, ints([62, 46]), 4)
    assert device_status() == _lib.DEVICE_STATUS_KV4_BAD_PAGE
    assert (k[0, 2:] == 0).all() and (v[1, 2:] == 0).all() and (k[0, :2] != 0).any()
    reset_device_status()
    src = torch.full((2, H, 8), -1, dtype=torch.int32, device="cuda")
    src[0, 0, 0], src[1, 1, 2], src[1, 0, 3] = 3, 1000, 8
    bad[1, 0] = -7
    before = cache.pages.clone()
    kv4_evict_move(cache, bad, src)
    assert device_status() in (_lib.DEVICE_STATUS_KV4_BAD_SOURCE, _lib.DEVICE_STATUS_KV4_BAD_PAGE)
    assert torch.equal(cache.pages, before)


def test_pool_past_32_bit_offsets():
    """Pages whose byte offsets pass 2^32 and whose token indices pass 2^24."""
    page, group, H = 256, 128, 4
    pages = (5 << 30) // (H * 256 // 16 * plain.block_bytes(group))
    cache = KV4Cache.empty(pages, H, page_size=page, group=group)
    table = ints([[pages - 1, 3, pages - 2]])
    n = 600
    k, v, q = randn(1, n, H, 128, seed=1), randn(1, n, H, 128, seed=2), randn(1, 1, 8, 128, seed=3)
    kv4_append(cache, k, v, table, ints([0]))
    gk, gv = kv4_expand(cache, table, ints([0]), n)
    small = KV4Cache.empty(3, H, page_size=page, group=group)
    t2 = ints([[2, 0, 1]])
    kv4_append(small, k, v, t2, ints([0]))
    for a, b in zip((gk, gv), kv4_expand(small, t2, ints([0]), n)):
        assert torch.equal(a, b)
    assert torch.equal(kv4_attention(q, cache, table, ints([n]), decay=0.0),
                       kv4_attention(q, small, t2, ints([n]), decay=0.0))
    assert torch.equal(cache.weights[table[0].long()], small.weights[t2[0].long()])
    got = kv4_evict_select(cache, table, ints([n]), 300, recent=20)
    want = kv4_evict_select(small, t2, ints([n]), 300, recent=20)
    assert torch.equal(got[0], want[0])
    kv4_evict_move(cache, table, got[0])
    kv4_evict_move(small, t2, want[0])
    assert torch.equal(cache.pages[table[0].long()], small.pages[t2[0].long()])
    assert device_status() == 0


# ---------------------------------------------------------------- eviction
def weights_like(cache, kind, seed):
    gen = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(cache.weights.shape, generator=gen))
    if kind == "ties":
        w = torch.floor(w) / 4
    elif kind == "equal":
        w = torch.full_like(w, 0.25)
    elif kind == "special":
        u = torch.rand(w.shape, generator=gen)
        w[u < 0.2], w[u < 0.15], w[u < 0.1], w[u < 0.05] = math.nan, math.inf, -0.0, 0.0
        w[(u > 0.9)] *= -1
        w[(u > 0.97)] = 1e-42
    cache.weights.copy_(w)


def check_select(cache, table, lens, keep, recent, seen):
    src, new = kv4_evict_select(cache, table, ints(lens), keep, recent=recent,
                                seen=None if seen is None else ints(seen))
    w, pos, tab = (t.cpu().numpy() for t in (cache.weights, cache.positions, table))
    for b, n in enumerate(lens):
        for h in range(cache.heads):
            want, m = plain.select(w, pos, tab[b], n, page=cache.page_size, keep=keep, recent=recent,
                                   seen=n if seen is None else seen[b], h=h)
            assert np.array_equal(src[b, h].cpu().numpy(), want), (b, h)
        assert new[b].item() == m
    return src, new


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "special"])
@pytest.mark.parametrize("lens,keep,recent,page,H", [
    ([1], 1, 0, 16, 1), ([2], 1, 1, 16, 2), ([17, 16, 0], 16, 3, 16, 3), ([700, 3, 40], 33, 33, 64, 2),
    ([2049], 2048, 64, 64, 2), ([5000, 4096], 1500, 100, 256, 1), ([300], 299, 0, 32, 4),
    ([100], 300, 5, 128, 1), ([40001, 33000], 20000, 500, 64, 1),
])
def test_select(kind, lens, keep, recent, page, H):
    cache, table = pool(len(lens), H, max(lens), page, 64, seed=1)
    weights_like(cache, kind, seed=keep)
    gen = torch.Generator().manual_seed(3)
    cache.positions.copy_(torch.randint(0, 2 * max(lens), cache.positions.shape, generator=gen))
    check_select(cache, table, lens, keep, recent, None)
    check_select(cache, table, lens, keep, recent, [2 * n for n in lens])
    assert device_status() == 0


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "special"])
@pytest.mark.parametrize("lens,keep,recent,page", [
    ([239, 1, 0, 200, 100], 90, 20, 16),         # one row of slots a warp, or part of one
    ([1025, 1024, 1023, 2049, 511], 700, 9, 64),
    ([4096, 3000, 17, 4095, 2048], 2048, 64, 256),
])
def test_select_for_many_short_heads(kind, lens, keep, recent, page):
    cache, table = pool(len(lens), 40, max(lens), page, 64, seed=5)
    weights_like(cache, kind, seed=keep)
    gen = torch.Generator().manual_seed(6)
    cache.positions.copy_(torch.randint(0, 2 * max(lens), cache.positions.shape, generator=gen))
    check_select(cache, table, lens, keep, recent, [2 * n for n in lens])
    assert device_status() == 0


@pytest.mark.parametrize("kind", ["spread", "ties"])
@pytest.mark.parametrize("n,H", [(140_000, 1), (30_000, 160), (260_001, 2)])
def test_select_long_runs(kind, n, H):
    cache, table = pool(1, H, n, 256, 64, seed=2)
    weights_like(cache, kind, seed=4)
    gen = torch.Generator().manual_seed(7)
    cache.positions.copy_(torch.randint(0, 2 * n, cache.positions.shape, generator=gen))
    check_select(cache, table, [n - 3], n // 3, 100, [2 * n])
    assert device_status() == 0


@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
def test_select_from_a_table_too_long_for_shared_memory(kind):
    """A page table of 409,600 slots, of which 9000 are used."""
    cache, table = pool(1, 2, 9000, 256, 64, seed=2)
    weights_like(cache, kind, seed=7)
    wide = torch.full((1, 1600), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    check_select(cache, wide, [9000], 3000, 100, None)
    assert device_status() == 0


@pytest.mark.parametrize("group,page", [(32, 16), (64, 64), (128, 256)])
def test_move(group, page):
    lens, keep, H = [500, 333, 80], 100, 3
    cache, table = filled(3, H, lens, page, group, seed=2, fill=0)
    weights_like(cache, "spread", 5)
    src, new = check_select(cache, table, lens, keep, 10, None)
    tab = table.cpu().numpy()
    pages, pos, w = (t.cpu().numpy().copy() for t in (cache.pages, cache.positions, cache.weights))
    kv4_evict_move(cache, table, src)
    assert device_status() == 0
    want = pages.copy(), pos.copy(), w.copy()
    for b in range(3):
        for h in range(H):
            for d, s in enumerate(src[b, h].tolist()):
                if s < 0 or s == d:
                    continue
                pd, ps, sd, ss = tab[b, d // page], tab[b, s // page], d % page, s % page
                for value in (0, 1):
                    (a, x), (c, y) = plain.row_offset(sd, value, group), plain.row_offset(ss, value, group)
                    m = 4 * (128 // group)
                    want[0][pd, h, a:a + 64] = pages[ps, h, c:c + 64]
                    want[0][pd, h, x:x + m] = pages[ps, h, y:y + m]
                want[1][pd, h, sd], want[2][pd, h, sd] = pos[ps, h, ss], w[ps, h, ss]
    for got, ref in zip((cache.pages, cache.positions, cache.weights), want):
        assert np.array_equal(got.cpu().numpy(), ref)
    kv4_evict_move(cache, table, src)  # the same moves again change nothing
    assert np.array_equal(cache.pages.cpu().numpy(), want[0])


# ---------------------------------------------------------------- together
def test_a_run_of_steps_with_eviction():
    """A prompt, then steps of append, tracked attention and eviction at a budget: the cache's
    contents follow a plain copy of the tokens, and every step's outputs the definition."""
    B, H, Hq, page, group, keep, recent, T0 = 2, 2, 6, 16, 64, 40, 8, 70
    cache, table = pool(B, H, T0 + 8, page, group, seed=3, fill=0xff)
    lengths, seen = ints([0, 0]), ints([0, 0])
    counts = [T0, T0 - 13]
    k, v = randn(B, T0, H, 128, seed=1), randn(B, T0, H, 128, seed=2)
    kv4_append(cache, k, v, table, lengths, counts=ints(counts), seen=seen)
    lengths, seen = lengths + ints(counts), seen + ints(counts)
    tokens = [[[(p, k[b, p, h], v[b, p, h]) for p in range(counts[b])] for h in range(H)]
              for b in range(B)]
    for step in range(6):
        T = 1 + step % 3
        k, v = randn(B, T, H, 128, seed=10 + step), randn(B, T, H, 128, seed=50 + step)
        kv4_append(cache, k, v, table, lengths, seen=seen)
        for b in range(B):
            for h in range(H):
                tokens[b][h] += [(seen[b].item() + t, k[b, t, h], v[b, t, h]) for t in range(T)]
        lengths, seen = lengths + T, seen + T
        q = randn(B, T, Hq, 128, seed=90 + step)
        got = kv4_attention(q, cache, table, lengths, decay=0.9, return_lse=True)
        check_attention(got, q, cache, table, lengths.tolist(), [T] * B)
        src, new = check_select(cache, table, lengths.tolist(), keep, recent, seen.tolist())
        kv4_evict_move(cache, table, src)
        lengths = new
        for b in range(B):
            for h in range(H):
                tokens[b][h] = [tokens[b][h][s] for s in src[b, h].tolist() if s >= 0]
                latest = sorted(p for p, _, _ in tokens[b][h])[-recent:]
                assert latest == list(range(seen[b].item() - recent, seen[b].item()))
        n = int(lengths.max())
        gk, gv = kv4_expand(cache, table, ints([0, 0]), n, counts=lengths)
        tab, pos = table.cpu().numpy(), cache.positions.cpu().numpy()
        for b in range(B):
            for h in range(H):
                for i, (p, kk, vv) in enumerate(tokens[b][h]):
                    assert pos[tab[b, i // page], h, i % page] == p
                    for g, x in ((gk, kk), (gv, vv)):
                        want = plain.quantise(x.double().cpu().numpy(), group)[0]
                        assert torch.equal(g[b, i, h].cpu(), torch.as_tensor(want).to(torch.bfloat16))
    assert device_status() == 0


@pytest.mark.parametrize("lens,T,Hq,H,counts", [
    ([40, 300, 0], 3, 8, 2, [1, 0, 0]),          # one piece a unit
    ([5000, 4000], 40, 8, 2, [3, 40]),           # units cut; tiles without a row that is real
    ([2000, 1, 33], 7, 32, 8, [0, 1, 7]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_past_a_count_in_memory_used_before(lens, T, Hq, H, counts, causal):
    cache, table = filled(len(lens), H, lens, 64, 64, seed=3)
    q = randn(len(lens), T, Hq, 128, seed=4)
    for b, c in enumerate(counts):  # what padding holds is not for use
        q[b, c:] = float("nan")
    torch.use_deterministic_algorithms(True)  # new memory is filled with NaN
    try:
        assert torch.empty_like(q).isnan().all()
        got = kv4_attention(q, cache, table, ints(lens), counts=ints(counts), causal=causal,
                            return_lse=True)
    finally:
        torch.use_deterministic_algorithms(False)
    assert device_status() == 0
    for b, c in enumerate(counts):
        assert (got[0][b, c:] == 0).all() and (got[1][b, :, c:] == -math.inf).all()
    q.nan_to_num_(0.0)
    check_attention(got, q, cache, table, lens, counts, causal=causal)


def test_graph_capture_and_replay():
    B, H, Hq, n = 2, 2, 8, 500
    cache, table = filled(B, H, [n, n - 100], 64, 64, seed=1)
    k, v, q = randn(B, 1, H, 128, seed=2), randn(B, 1, H, 128, seed=3), randn(B, 1, Hq, 128, seed=4)
    lengths, seen = ints([n - 3, n - 103]), ints([n - 3, n - 103])
    out = torch.empty_like(q)

    def step():
        kv4_append(cache, k, v, table, lengths, seen=seen)
        now = lengths + 1
        kv4_attention(q, cache, table, now, decay=1.0, out=out)
        src, new = kv4_evict_select(cache, table, now, 450, recent=16, seen=seen)
        kv4_evict_move(cache, table, src)
        return src, new

    step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    start = [t.clone() for t in (cache.pages, cache.positions, cache.weights)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        src, new = step()
    for i in range(3):
        for t, x in zip((cache.pages, cache.positions, cache.weights), start):
            t.copy_(x)
        q.copy_(randn(B, 1, Hq, 128, seed=20 + i))
        k.copy_(randn(B, 1, H, 128, seed=30 + i))
        lengths.copy_(ints([n - 50 - i, 300]))
        g.replay()
        got = [t.clone() for t in (out, src, new, cache.pages, cache.positions, cache.weights)]
        for t, x in zip((cache.pages, cache.positions, cache.weights), start):
            t.copy_(x)
        out.zero_()
        src2, new2 = step()
        want = (out, src2, new2, cache.pages, cache.positions, cache.weights)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert device_status() == 0


def test_two_streams_at_once_and_repeated_runs_agree():
    cache, table = filled(4, 4, [900, 30, 2000, 1], 64, 64, seed=1)
    lens = ints([900, 30, 2000, 1])
    qs = [randn(4, 2, 16, 128, seed=s) for s in range(4)]
    want = [kv4_attention(q, cache, table, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(kv4_attention(qs[i % 4], cache, table, lens))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 4])


def test_python_surface_refuses():
    cache, table = filled(2, 2, [40, 30], 16, 64, seed=1)
    n = ints([40, 30])
    q = randn(2, 1, 4, 128)
    x = randn(2, 1, 2, 128)
    for call in (
            lambda: kv4_attention(q[:, :, :3], cache, table, n),
            lambda: kv4_attention(q.float(), cache, table, n),
            lambda: kv4_attention(q.cpu(), cache, table, n),
            lambda: kv4_attention(q[:1], cache, table, n),
            lambda: kv4_attention(q[..., :64], cache, table, n),
            lambda: kv4_attention(q.transpose(2, 3).contiguous().transpose(2, 3), cache, table, n),
            lambda: kv4_attention(q[:, :0], cache, table, n),
            lambda: kv4_attention(q, cache, table, n.long()),
            lambda: kv4_attention(q, cache, table, n[:1]),
            lambda: kv4_attention(q, cache, table.long(), n),
            lambda: kv4_attention(q, cache, table.cpu(), n),
            lambda: kv4_attention(q, cache, table[:, :0], n),
            lambda: kv4_attention(q, cache, table[:1].expand(2, -1), n),
            lambda: kv4_attention(q, cache, table, n, counts=n.cpu()),
            lambda: kv4_attention(q, cache, table, n, decay=-0.5),
            lambda: kv4_attention(q, cache, table, n, decay=math.nan),
            lambda: kv4_attention(q, cache, table, n, softmax_scale=0.0),
            lambda: kv4_attention(q, cache, table, n, out=q.half()),
            lambda: kv4_attention(q, cache, table, n, out=q),
            lambda: kv4_attention(q[:, :1].expand(2, 3, 4, 128), cache, table, n),
            lambda: kv4_append(cache, x, x.half(), table, n),
            lambda: kv4_append(cache, x, q, table, n),
            lambda: kv4_append(cache, x, x, table, n, seen=n[:1]),
            lambda: kv4_append(cache, randn(2 * 256 + 1)[1:].view(2, 1, 2, 128), x, table, n),
            lambda: kv4_expand(cache, table, n, 0),
            lambda: kv4_expand(cache, table, n, 4, dtype=torch.float32),
            lambda: kv4_expand(cache, table, n, 4, out=(x, x)),
            lambda: kv4_evict_select(cache, table, n, 0),
            lambda: kv4_evict_select(cache, table, n, 4, recent=5),
            lambda: kv4_evict_select(cache, table, n, 4, recent=-1),
            lambda: kv4_evict_move(cache, table, n),
            lambda: kv4_evict_move(cache, table, torch.zeros(2, 2, 4, device="cuda")),
            lambda: KV4Cache(cache.pages, cache.positions, cache.weights[:, :1], page_size=16,
                             group=64),
    ):
        with pytest.raises(RuntimeError):
            call()
    assert device_status() == 0
