"""GPU tests of the attention over the 4-bit cache for values, keys and queries of very different
sizes, and at a tolerance close to what fp32 sums give.

Reference: fp64, on what the cache's bytes stand for (tests/kv4_plain.py). Tolerances count
roundings (eps/2 relative to the value), for output o = sum_t w_t v_t over the seen tokens t:
  * the rounding to the output type;
  * a weight times its value scale is held as the sum of two bf16 numbers: the first is off by at
    most 2^-9 of it, the second by 2^-9 of that, so 2^-18, and a few fp32 roundings: 2^-17 of the
    sum of w |v|;
  * a score is a sum of 128 fp32 products, in any order, each partial sum rounded or cut (2^-23 of
    the sum of |q k|), then at most 8 more fp32 steps; the exponential is good to 2^-21: dx_t = 136
    * 2^-23 * sum |q k_t| * scale + 2^-21. It moves o by at most sum_t w_t dx_t (|v_t| + |o|);
  * partial sums of outputs and of weights: a chain of c tokens is c / 8 matrix products (two for
    16 tokens), each of which may cut twice, and at most 64 joins: (c / 4 + 64) * 2^-23 of the sum
    of w |v|;
  * what underflows: values are summed in units of 2^-24 of theirs, with bf16 steps of 2^-133 and
    codes up to 15, so n tokens leave at most n * 2^(-133 + 24 + 4 + 6) (weights reach 2^6).
"""
import math

import numpy as np
import pytest
import torch

from llm_fa_b200 import KV4Cache, device_status, kv4_append, kv4_attention, reset_device_status

from . import kv4_plain as plain

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


@pytest.fixture(autouse=True)
def _clean_status():
    reset_device_status()
    yield
    reset_device_status()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def normal(*shape, seed, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale


def hold(k, v, lens, page=64, group=64, dtype=torch.bfloat16):
    """A cache of k, v fp64 [B, n, H, 128], of which each sequence holds lens[b] tokens; what no
    token holds is 0xff (NaN pairs)."""
    B, n, H, _ = k.shape
    width = -(-n // page)
    cache = KV4Cache.empty(B * width + 1, H, page_size=page, group=group)
    cache.pages.fill_(0xff)
    table = torch.randperm(B * width + 1, generator=torch.Generator().manual_seed(n))[1:]
    table = table.reshape(B, width).to(torch.int32).cuda()
    kv4_append(cache, k.to(dtype).cuda(), v.to(dtype).cuda(), table, ints([0] * B), counts=ints(lens))
    assert device_status() == 0
    return cache, table


def check(got, q, cache, table, lens, *, chain=None, causal=True, scale=1 / math.sqrt(128),
          rows=slice(None)):
    """Compares o and lse of new tokens `rows` (all sequences have all of q's) and returns the
    fp64 weights that each token received and what errors of scores move them by, to first order.
    chain: tokens that one worker sums, at most (default: all)."""
    pages, tab = cache.pages.cpu().numpy(), table.cpu().numpy()
    B, T, Hq, _ = q.shape
    G = Hq // cache.heads
    o_got, lse_got = got[0].double()[:, rows], got[1].double()[:, :, rows]
    sums = []
    for b, n in enumerate(lens):
        k, v = (torch.as_tensor(np.stack([
            plain.read(pages, tab[b], n, cache.page_size, cache.group, h, side)
            for h in range(cache.heads)]), device="cuda") for side in (0, 1))  # [H, n, 128]
        qb = q[b].double()[rows].unflatten(1, (cache.heads, G)).permute(1, 0, 2, 3)  # [H, T, G, 128]
        x = qb @ k[:, None].transpose(-1, -2) * scale
        size = qb.abs() @ k[:, None].abs().transpose(-1, -2) * scale
        i = torch.arange(T, device="cuda")[rows]
        sees = torch.arange(n, device="cuda") < (n - (T - 1 - i) if causal else n + 0 * i)[:, None]
        sees = sees[None, :, None]
        x = torch.where(sees, x, -math.inf)
        w = torch.softmax(x, -1)
        held = torch.where(torch.isfinite(v), v, 0.0)[:, None]  # NaN only where no row looks
        o, mag = w @ held, w @ held.abs()
        dx = torch.where(sees, 136 * 2.0 ** -23 * size + 2.0 ** -21, 0.0)
        c = n if chain is None else chain
        tol = HALF[q.dtype] * o.abs() * (1 + 2.0 ** -7) + TINY[q.dtype] + n * 2.0 ** -99
        tol = tol + (2.0 ** -17 + (c / 4 + 64) * 2.0 ** -23) * mag
        tol = tol + (w * dx) @ held.abs() + (w * dx).sum(-1, keepdim=True) * o.abs()
        want = o.permute(1, 0, 2, 3).flatten(1, 2)
        err, tol = (o_got[b] - want).abs(), tol.permute(1, 0, 2, 3).flatten(1, 2)
        assert bool((err <= tol).all()), (b, (err / tol).max().item(), err.max().item())
        lse = torch.logsumexp(x, -1).permute(0, 2, 1).flatten(0, 1)
        ltol = (w * dx).sum(-1).permute(0, 2, 1).flatten(0, 1)
        ltol = ltol + (c / 4 + 64) * 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -22 * lse.abs()
        assert bool(((lse_got[b] - lse).abs() <= ltol).all()), b
        off = w * (dx + (w * dx).sum(-1, keepdim=True))
        sums.append((w.sum((1, 2)), off.sum((1, 2))))
    assert device_status() == 0
    return sums


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("low", [-3.38e38, -2.0e38, -1.0e36, 0.0])
def test_append_groups_whose_span_passes_fp32(group, low):
    """Finite groups are quantised as defined, however wide, and large ones attend."""
    x = normal(1, 40, 2, 128, seed=int(group)) * 1e37
    x[:, :, :, ::32], x[:, :, :, 1::32] = 3.38e38, low
    x = x.to(torch.bfloat16)
    cache, table = hold(x.double(), -x.double(), [40], group=group)
    pages, tab = cache.pages.cpu().numpy(), table.cpu().numpy()
    for h in range(2):
        for value, y in ((0, x), (1, -x)):
            want = plain.quantise(y[0, :, h].double().numpy(), group)[0]
            assert np.array_equal(plain.read(pages, tab[0], 40, 64, group, h, value), want)
    q = (normal(1, 1, 4, 128, seed=1) * 2.0 ** -124).to(torch.bfloat16).cuda()
    got = kv4_attention(q, cache, table, ints([40]), return_lse=True)
    inside = plain.read(pages, tab[0], 40, 64, group, 0, 1)
    if np.abs(inside).max() < 3.3e38:  # else an output may round to infinity
        check(got, q, cache, table, [40])


# 512 heads of 4 tiles each: a worker has several units, so a segment takes in whole sequences
MANY = dict(B=64, H=8, n=100)


def away(q, k, H, token, score):
    """Gives `token` of every sequence a key whose score is `score` for all rows of its head:
    q's first channel is 8 in every row, the others' first channels are 0 here."""
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[:, token] = 0.0
    k[:, token, :, 0] = score * math.sqrt(128) / 8.0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,power,token", [
    (torch.bfloat16, 16, 0), (torch.bfloat16, 24, 0), (torch.bfloat16, 34, 17), (torch.bfloat16, 60, 40),
    (torch.float16, 20, 0),
])
def test_large_values_of_a_token_that_has_no_weight(dtype, power, token, group):
    B, H, n = MANY.values()
    base = 1.0 if dtype == torch.bfloat16 else 2.0 ** -7
    q, k, v = normal(B, 1, 2 * H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    away(q, k, H, token, -300.0)
    v *= base
    v[:, token] *= 2.0 ** power
    if dtype == torch.float16:
        v.clamp_(-60000, 60000)
    cache, table = hold(k, v, [n] * B, group=group, dtype=dtype)
    q = q.to(dtype).cuda()
    got = kv4_attention(q, cache, table, ints([n] * B), return_lse=True)
    check(got, q, cache, table, [n] * B)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_a_tile_that_look_at_values_of_different_size(dtype):
    """Of a key head's rows, some give all their weight to a token with large values, some none;
    a group of small channels stands beside one of large channels."""
    B, H, n = MANY.values()
    q, k, v = normal(B, 1, 4 * H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    away(q, k, H, 3, 300.0)
    q[:, :, 0::2, 0] = -8.0  # even rows look away from token 3
    big = 2.0 ** 30 if dtype == torch.bfloat16 else 2.0 ** 13
    small = 2.0 ** -30 if dtype == torch.bfloat16 else 2.0 ** -9
    v[..., 32:64] *= small
    v[:, 3] *= big
    cache, table = hold(k, v, [n] * B, group=32, dtype=dtype)
    q = q.to(dtype).cuda()
    got = kv4_attention(q, cache, table, ints([n] * B), return_lse=True)
    check(got, q, cache, table, [n] * B)


def test_values_larger_than_any_that_a_later_maximum_leaves():
    """A token with large values whose weight is whole until a later token's score drops it."""
    B, H, n = MANY.values()
    q, k, v = normal(B, 1, H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    away(q, k, H, 0, 50.0)
    k[:, 64:, :, 0] = 150.0 * math.sqrt(128) / 8.0  # all later ones are 100 above it
    v[:, 0] *= 2.0 ** 40
    cache, table = hold(k, v, [n] * B)
    q = q.to(torch.bfloat16).cuda()
    got = kv4_attention(q, cache, table, ints([n] * B), return_lse=True)
    check(got, q, cache, table, [n] * B)


@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("kind", ["large", "nan"])
def test_values_of_tokens_that_early_rows_do_not_see(G, kind):
    """Causal among the new tokens: the last 32 of them, a tile of their own, hold values 2^30 times
    larger, or NaN."""
    B, H, n, T, seen = 64, 8, 160, 47, 15
    q, k, v = normal(B, T, G * H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    first = n - T + seen  # slots from here on are hidden from rows below `seen`
    if kind == "large":
        v[:, first:] *= 2.0 ** 30
    else:
        v[:, first:] = math.nan
        k[:, first:] *= 20  # and their scores are larger than any before
    cache, table = hold(k, v, [n] * B)
    q = q.to(torch.bfloat16).cuda()
    got = kv4_attention(q, cache, table, ints([n] * B), return_lse=True)
    check(got, q, cache, table, [n] * B, rows=slice(0, seen))
    if kind == "large":
        check(got, q, cache, table, [n] * B)
    else:
        assert bool(got[0][:, seen:].isnan().all())


@pytest.mark.parametrize("size", [2.0 ** 125, 2.0 ** 100, 2.0 ** -80])
def test_values_near_the_ends_of_the_type(size):
    B, H, n = 2, 2, 700
    q, k, v = normal(B, 1, 2 * H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    v = v.clamp(-3.5, 3.5) * size
    cache, table = hold(k, v, [n, 1])
    q = q.to(torch.bfloat16).cuda()
    got = kv4_attention(q, cache, table, ints([n, 1]), return_lse=True)
    check(got, q, cache, table, [n, 1])


@pytest.mark.parametrize("query,key", [
    (-105, 106), (-124, 123), (-130, 122), (-60, 60), (100, -101), (124, -114),
])
@pytest.mark.parametrize("decay", [None, 0.0])
def test_scores_of_ordinary_size_from_queries_and_keys_of_any(query, key, decay):
    """Powers of two whose product is ordinary, beside a row whose queries are ordinary and, for
    small keys, sees only scores near 0."""
    B, H, n, G = 2, 2, 300, 4
    q, k, v = normal(B, 1, G * H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    q = q.clamp(-3.5, 3.5) * 2.0 ** query
    k = k.clamp(-3.5, 3.5) * 2.0 ** key
    if key < 0:
        q[:, :, 1] *= 2.0 ** -query
    for group in (32, 128):
        cache, table = hold(k, v, [n] * B, group=group)
        qc = q.to(torch.bfloat16).cuda()
        got = kv4_attention(qc, cache, table, ints([n] * B), return_lse=True, decay=decay)
        sums = check(got, qc, cache, table, [n] * B)
        if decay is not None:
            # e^x - 1 <= 2 x up to 1.25, which errors of scores below 2^13 (dx < 0.2) stay under; then
            # G + 3 fp32 roundings and the sums' (n / 4 + 64) * 2^-23
            i = torch.arange(n, device="cuda")
            for b, (want, off) in enumerate(sums):
                w = cache.weights[table[b, i // 64].long(), :, i % 64].double().T
                tol = 2 * off + ((G + 3) * 2.0 ** -24 + (n / 4 + 64) * 2.0 ** -23) * want + 1e-30
                assert bool(((w - want).abs() <= tol).all())


@pytest.mark.parametrize("power", [20, 36, 50, 90])
@pytest.mark.parametrize("G", [4, 20])
def test_channels_of_a_query_of_very_different_size(power, G):
    """Half of the channels are large in queries and as small in keys: both halves count."""
    B, H, n = 2, 2, 300
    q, k, v = normal(B, 1, G * H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    q[..., :64] *= 2.0 ** power
    k[..., :64] *= 2.0 ** -power
    for group in (32, 64):
        cache, table = hold(k, v, [n] * B, group=group)
        qc = q.to(torch.bfloat16).cuda()
        got = kv4_attention(qc, cache, table, ints([n] * B), return_lse=True, decay=0.0)
        sums = check(got, qc, cache, table, [n] * B)
        for b, (want, off) in enumerate(sums):
            tol = 2 * off + ((G + 3) * 2.0 ** -24 + (n / 4 + 64) * 2.0 ** -23) * want + 1e-37
            assert bool(((weights_of(cache, table, b, n) - want.T).abs() <= tol.T).all())


def test_a_softmax_scale_far_from_one():
    B, H, n = 2, 2, 300
    q, k, v = normal(B, 1, 2 * H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    for power, scale in ((100, 2.0 ** -103), (-100, 2.0 ** 97), (-20, 2.0 ** 17), (110, 2.0 ** -113)):
        cache, table = hold(k, v, [n] * B)
        qc = (q * 2.0 ** power).to(torch.bfloat16).cuda()
        got = kv4_attention(qc, cache, table, ints([n] * B), return_lse=True, softmax_scale=scale)
        check(got, qc, cache, table, [n] * B, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,T,group", [(1, 1, 64), (4, 1, 32), (8, 1, 128), (16, 1, 64), (4, 5, 128)])
def test_precision_of_flat_weights(dtype, G, T, group):
    """Small scores, so that their error leaves that of the weights in sight."""
    B, H, n = MANY.values()
    q = normal(B, T, G * H, 128, seed=1, scale=0.01)
    k, v = normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    cache, table = hold(k, v, [n] * B, group=group, dtype=dtype)
    q = q.to(dtype).cuda()
    got = kv4_attention(q, cache, table, ints([n] * B), return_lse=True)
    check(got, q, cache, table, [n] * B)


# ---------------------------------------------------------------- large ones
def weights_of(cache, table, b, n):
    i = torch.arange(n, device="cuda")
    p = cache.page_size
    return cache.weights[table[b, i // p].long(), :, i % p].double()  # [n, heads]


@pytest.mark.parametrize("n,H,G,group,dtype", [
    (131072, 1, 4, 32, torch.bfloat16), (100001, 2, 2, 128, torch.float16), (40000, 1, 20, 64, torch.bfloat16),
])
def test_one_long_sequence_in_hundreds_of_pieces(n, H, G, group, dtype):
    q, k, v = normal(1, 1, G * H, 128, seed=1), normal(1, n, H, 128, seed=2), normal(1, n, H, 128, seed=3)
    v += 0.5  # so that outputs are not nearly nothing
    cache, table = hold(k, v, [n], group=group, dtype=dtype)
    q = q.to(dtype).cuda()
    got = kv4_attention(q, cache, table, ints([n]), return_lse=True, decay=0.0)
    # at least 8 workers on each of a GPU's 100 SMs or more
    chain = 32 * (n * H // 32 // 800 + 2)
    want, off = check(got, q, cache, table, [n], chain=chain)[0]
    err = (weights_of(cache, table, 0, n) - want.T).abs()
    tol = 2 * off + ((G + 3) * 2.0 ** -24 + (chain / 4 + 64) * 2.0 ** -23) * want + 1e-37
    assert bool((err <= tol.T).all())


@pytest.mark.parametrize("B,T,H,G", [(129, 1, 2, 1), (300, 2, 1, 3), (300, 1, 1, 20), (4096, 1, 1, 4)])
def test_batches_of_more_sequences_than_a_block_has_threads(B, T, H, G):
    gen = torch.Generator().manual_seed(B)
    lens = (T + torch.randint(0, 120, (B,), generator=gen)).tolist()
    n = max(lens)
    q, k, v = normal(B, T, G * H, 128, seed=1), normal(B, n, H, 128, seed=2), normal(B, n, H, 128, seed=3)
    cache, table = hold(k, v, lens, page=16)
    q = q.to(torch.bfloat16).cuda()
    lens[5] = 0  # what its pages hold is not for use
    got = kv4_attention(q, cache, table, ints(lens), return_lse=True, decay=0.0)
    assert bool((got[0][5] == 0).all()) and bool((got[1][5] == -math.inf).all())
    some = [b for b in (*range(0, B, max(1, B // 60)), *range(B - 4, B)) if b != 5]
    part = torch.tensor(some, device="cuda")
    sums = check([t[part] for t in got], q[part], cache, table[part], [lens[b] for b in some])
    for b, (want, off) in zip(some, sums):
        err = (weights_of(cache, table, b, lens[b]) - want.T).abs()
        tol = 2 * off + ((T * G + 3) * 2.0 ** -24 + (lens[b] / 4 + 64) * 2.0 ** -23) * want + 1e-37
        assert bool((err <= tol.T).all())
