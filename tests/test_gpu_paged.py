"""Paged caches and drafted tokens against plain restatements in 64 bits (numpy, one sequence at a time)."""
import itertools
import threading

import numpy as np
import pytest
import torch

from my_nn_engine_b200 import ffi, ops

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# half a step of the output's rounding
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def host(t):
    return t.detach().double().cpu().numpy()


def same(got, want):
    """Equal to the bit, without pages of numbers where it is not."""
    got, want = (x if isinstance(x, np.ndarray) else host(x) for x in (got, want))
    return got.shape == want.shape and int((got != want).sum()) == 0


def cache(rng, lengths, G, D, page, dt, spare=2, needed=None, fill=None):
    """Random pages in random order; a table with -1 behind the pages of a sequence (and where ``needed`` says that a page is not held)."""
    B, width = len(lengths), max([-(-n // page) for n in lengths] + [1]) + 1
    table = np.full((B, width), -1, np.int64)
    held = [(b, i) for b, n in enumerate(lengths) for i in range(-(-n // page)) if needed is None or needed(b, i)]
    order = rng.permutation(len(held) + spare)
    for (b, i), pg in zip(held, order):
        table[b, i] = pg
    shape = (len(held) + spare, G, page, D)
    k, v = torch.randn(shape, generator=torch.Generator().manual_seed(int(rng.integers(1 << 30)))), torch.randn(shape, generator=torch.Generator().manual_seed(int(rng.integers(1 << 30))))
    if fill is not None:  # rows that hold no position of any sequence
        owned = np.zeros(shape[0] * page, bool)
        for b, n in enumerate(lengths):
            for j in range(n):
                if table[b, j // page] >= 0:
                    owned[table[b, j // page] * page + j % page] = True
        for t in (k, v):
            t.permute(0, 2, 1, 3)[torch.from_numpy(~owned.reshape(-1, page))] = fill
    return k.to("cuda", DT[dt]), v.to("cuda", DT[dt]), torch.from_numpy(table).int().cuda()


def want_attention(q, k, v, table, lengths, counts, scale, window=0, sinks=0, cap=0.0):
    """The definition; also sum |p v| per output, which errors of the sums go by."""
    q, k, v, table = host(q), host(k), host(v), table.cpu().numpy()
    B, H, S, D = q.shape
    G, page = k.shape[1:3]
    out, mass = np.zeros((B, S, H, D)), np.zeros((B, S, H, D))
    for b, s in itertools.product(range(B), range(S)):
        at = lengths[b] - counts[b] + s
        if s >= counts[b] or at < 0:
            continue
        j = np.arange(at + 1)
        j = j[(window <= 0) | (at - j < window) | (j < sinks)]
        pages = table[b, j // page]
        j, pages = j[(pages >= 0) & (pages < k.shape[0])], pages[(pages >= 0) & (pages < k.shape[0])]
        if not len(j):
            continue
        for h in range(H):
            x = k[pages, h // (H // G), j % page] @ q[b, h, s] * scale
            x = cap * np.tanh(x / cap) if cap else x
            p = np.exp(x - x.max())
            p /= p.sum()
            vals = v[pages, h // (H // G), j % page]
            out[b, s, h], mass[b, s, h] = p @ vals, p @ np.abs(vals)
    return out, mass


def close_attention(got, want, mass, dt):
    """One rounding of the output.  Inside: a score is a sum of D <= 256 products whose magnitudes add up to some 10 (normal numbers, scale D^-0.5); its roundings of 2^-24
    are independent, so it is off by about 16 * 10 * 2^-24 = 2^-16.7, and so is each weight relative to itself (weights as two 16-bit parts: 2^-16).  The output moves
    by twice that times sum |p v|."""
    got = host(got)
    assert np.isfinite(got).all()
    bound = HALF[dt] * np.abs(want) + 2 * 2.0 ** -16 * mass + (2.0 ** -25 if dt == "f16" else 1e-30)
    worst = (np.abs(got - want) / np.maximum(bound, 1e-30)).max()
    assert worst <= 1.0, worst


def run_attention(seed, dt, lengths, H, G, D, page, S=1, counts=None, window=0, sinks=0, cap=0.0, needed=None, fill=None):
    rng = np.random.default_rng(seed)
    k, v, table = cache(rng, lengths, G, D, page, dt, needed=needed, fill=fill)
    q = torch.from_numpy(rng.standard_normal((len(lengths), H, S, D))).to("cuda", DT[dt])
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    c = torch.tensor(counts, dtype=torch.int32, device="cuda") if counts is not None else None
    got = ops.paged_attention(q, k, v, table, n, D ** -0.5, counts=c, window=window, sinks=sinks, softcap=cap)
    want, mass = want_attention(q, k, v, table, lengths, counts or [S] * len(lengths), D ** -0.5, window, sinks, cap)
    assert got.shape == want.shape and got.dtype == q.dtype
    close_attention(got, want, mass, dt)
    return got


# ---- attention -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (32, 8, 128), (4, 4, 80), (7, 1, 128), (16, 1, 64), (3, 3, 20), (6, 2, 33), (8, 2, 256), (4, 2, 192), (18, 1, 96), (2, 1, 8)])
def test_one_token_per_sequence(dt, H, G, D):
    for page, lengths in ((16, [1, 16, 17, 100, 0, 333]), (10, [5, 1, 29]), (1, [3, 40]), (64, [700, 64, 65]), (24, [23, 24, 25, 48])):
        run_attention(D + page, dt, lengths, H, G, D, page)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [16, 10, 128])
def test_long_and_short_sequences_in_one_batch(dt, page):
    """Pairs that lie in many CTAs, beside ones that lie in a CTA with others, and a sequence with nothing."""
    run_attention(page, dt, [9000, 1, 0, 130, 4097, 15, 2500, 0], 8, 2, 64, page)
    run_attention(page, dt, [20001], 4, 1, 128, page)
    run_attention(page, dt, [1] * 70 + [600] + [0] * 80 + [2] * 30, 4, 2, 64, page)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D", [(2, 2, 80), (3, 3, 33), (4, 2, 20), (8, 2, 36), (2, 1, 250), (12, 2, 72), (2, 2, 256), (18, 1, 100)])
def test_parts_of_every_number_of_rows(dt, H, G, D):
    """Pairs that lie in several CTAs, for one, two, four and more query heads per kv head and heads of odd sizes."""
    run_attention(D, dt, [3000, 7, 1501, 900], H, G, D, 16)
    run_attention(D, dt, [2000, 33], H, G, D, 10, S=2)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D,S", [(8, 2, 64, 2), (32, 8, 128, 5), (7, 1, 128, 3), (4, 4, 80, 8), (16, 2, 64, 8), (32, 1, 64, 5), (4, 2, 33, 4)])
def test_drafted_tokens(dt, H, G, D, S):
    lengths = [S, 40, 333, 1, 0, 700, 17]
    counts = [S, 1, S, 1, 0, min(S, 2), 0]
    run_attention(S, dt, lengths, H, G, D, 16, S, counts)
    run_attention(S + 1, dt, [max(n, S) for n in lengths], H, G, D, 24, S)


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("bf16", 128), ("f16", 40), ("f32", 64), ("f32", 33)])
def test_sequences_shorter_than_their_places(dt, D):
    """Without counts every place is a token: those of a sequence of fewer positions lie before its first one and see nothing."""
    for S in (3, 9):
        run_attention(S, dt, [0, 1, 2, S - 1, S, 700], 8, 2, D, 16, S)


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("bf16", 192), ("bf16", 256), ("bf16", 96), ("f32", 64)])
@pytest.mark.parametrize("group,S", [(1, 9), (5, 5), (8, 3), (8, 4), (7, 7), (8, 8), (9, 8), (4, 33)])
def test_numbers_of_rows_around_the_sizes_of_teams(dt, D, group, S):
    """9 to 132 query rows per kv head, over pairs that are cut and pairs that are not."""
    run_attention(group + S, dt, [1500, S, 77], 2 * group, 2, D, 16, S, [S, max(1, S - 2), 1])
    run_attention(group, dt, [S + 100, S], group, 1, D, 8, S, window=40, sinks=3)


def test_one_query_over_a_very_long_cache():
    """More CTAs than a pair has rows of parts in one go of the joining kernel."""
    for dt, D in (("bf16", 64), ("f32", 32)):
        run_attention(D, dt, [100003], 2, 1, D, 64)


def test_a_batch_larger_than_the_grid():
    rng = np.random.default_rng(3)
    lengths = [int(n) for n in rng.integers(0, 40, 700)]
    for width in (0, 70):  # a table that pairs are not cut for, and a wide one
        k, v, table = cache(rng, lengths, 1, 64, 16, "bf16")
        table = torch.nn.functional.pad(table, (0, width), value=-1).contiguous()
        q = torch.from_numpy(rng.standard_normal((700, 2, 1, 64))).to("cuda", torch.bfloat16)
        want, mass = want_attention(q, k, v, table, lengths, [1] * 700, 0.125)
        close_attention(ops.paged_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0.125), want, mass, "bf16")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (100, 33), (257, 16), (5000, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("S", [1, 4])
def test_window_and_first_tokens(dt, window, sinks, S):
    lengths = [4, 100, 101, 1000, 300, 17]
    for page in (16, 10):
        oldest = [n - S - window + 1 for n in lengths]
        run_attention(window % 1000 + sinks % 1000, dt, lengths, 8, 2, 64, page, S, window=window, sinks=sinks,
                      needed=lambda b, i: (i + 1) * page > oldest[b] or i * page < sinks, fill=float("nan"))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_capped_scores(dt):
    run_attention(3, dt, [1, 50, 700], 8, 2, 128, 16, cap=2.0)
    run_attention(3, dt, [5, 50, 700], 8, 2, 40, 16, S=3, cap=30.0, window=64, sinks=2)


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("f32", 64), ("bf16", 20)])
def test_what_is_not_seen_is_not_touched(dt, D):
    """NaN and infinity in rows behind the last position, in other sequences' spare pages, and in keys and values of later drafts."""
    for value in (float("nan"), float("inf")):
        run_attention(1, dt, [5, 17, 200, 0], 8, 2, D, 16, fill=value)
        run_attention(1, dt, [5, 17, 200, 1], 8, 2, D, 24, S=3, counts=[3, 2, 3, 1], fill=value)
    rng = np.random.default_rng(0)
    for window in (0, 20):
        k, v, table = cache(rng, [130], 2, D, 16, dt)
        q = torch.from_numpy(rng.standard_normal((1, 8, 4, D))).to("cuda", DT[dt])
        n = torch.tensor([130], dtype=torch.int32, device="cuda")
        clean = ops.paged_attention(q, k, v, table, n, 0.1, window=window)
        for j, first in ((129, 3), (128, 2)):  # only queries from `first` on see it
            for bad in (float("nan"), float("inf"), -float("inf")):
                k2, v2 = k.clone(), v.clone()
                k2[table[0, j // 16], :, j % 16] = bad
                v2[table[0, j // 16], :, j % 16] = bad
                got = ops.paged_attention(q, k2, v2, table, n, 0.1, window=window)
                assert torch.equal(got[:, :first], clean[:, :first])
                assert not torch.isfinite(got[:, first:]).any()


def test_entries_outside_the_cache_hold_no_rows():
    rng = np.random.default_rng(2)
    for dt, D in (("bf16", 64), ("f32", 20)):
        k, v, table = cache(rng, [100, 64], 2, D, 16, dt)
        table[0, 2], table[1, 0], table[0, 0] = 1 << 30, -7, k.shape[0]
        q = torch.from_numpy(rng.standard_normal((2, 4, 1, D))).to("cuda", DT[dt])
        n = torch.tensor([100, 64], dtype=torch.int32, device="cuda")
        want, mass = want_attention(q, k, v, table, [100, 64], [1, 1], 0.2)
        close_attention(ops.paged_attention(q, k, v, table, n, 0.2), want, mass, dt)
        table[:] = -1
        assert not ops.paged_attention(q, k, v, table, n, 0.2).any()
        # lengths and counts outside their ranges are taken as the nearest inside
        k, v, table = cache(rng, [64, 64], 2, D, 16, dt)
        table = table[:, :4].contiguous()
        over = ops.paged_attention(q, k, v, table, torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device="cuda"), 0.2)
        assert torch.equal(over[0], ops.paged_attention(q, k, v, table, torch.tensor([64, 0], dtype=torch.int32, device="cuda"), 0.2)[0]) and not over[1].any()


def test_pages_shared_by_sequences():
    """A common prefix: the table rows of two sequences name the same pages."""
    rng = np.random.default_rng(4)
    k, v, table = cache(rng, [100, 120], 2, 64, 16, "bf16")
    table[1, :6] = table[0, :6]
    q = torch.from_numpy(rng.standard_normal((2, 4, 1, 64))).to("cuda", torch.bfloat16)
    want, mass = want_attention(q, k, v, table, [100, 120], [1, 1], 0.125)
    close_attention(ops.paged_attention(q, k, v, table, torch.tensor([100, 120], dtype=torch.int32, device="cuda"), 0.125), want, mass, "bf16")


def test_rows_of_a_large_cache():
    """Element offsets past 2^31 in one cache tensor."""
    pages, G, page, D = 70000, 4, 64, 128  # 2.3e9 elements
    k = torch.empty(pages, G, page, D, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    rng = np.random.default_rng(6)
    table = torch.tensor([[69999, 3, 69000, -1]], dtype=torch.int32, device="cuda")
    for pg in (69999, 3, 69000):
        k[pg], v[pg] = (torch.from_numpy(rng.standard_normal((G, page, D))).cuda() for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((1, 8, 1, D))).to("cuda", torch.bfloat16)
    got = ops.paged_attention(q, k, v, table, torch.tensor([150], dtype=torch.int32, device="cuda"), 0.1)
    small = torch.tensor([[0, 1, 2, -1]], dtype=torch.int32, device="cuda")
    pick = [69999, 3, 69000]
    assert torch.equal(got, ops.paged_attention(q, k[pick].contiguous(), v[pick].contiguous(), small, torch.tensor([150], dtype=torch.int32, device="cuda"), 0.1))
    proj = torch.from_numpy(rng.standard_normal((1, 1, 16 * D))).to("cuda", torch.bfloat16)
    ops.paged_rotary_append(proj, torch.tensor([65], dtype=torch.int32, device="cuda"), table[:, [1, 0]].contiguous(), k, v, 8)
    assert torch.equal(k[69999, :, 0], proj.view(16, D)[8:12]) and torch.equal(v[69999, :, 0], proj.view(16, D)[12:])


def test_attention_into_a_given_tensor_and_unaligned_tensors():
    rng = np.random.default_rng(8)
    for dt in ("bf16", "f32"):
        lengths = [33, 260]
        k, v, table = cache(rng, lengths, 2, 64, 16, dt)
        q = torch.from_numpy(rng.standard_normal((2, 8, 1, 64))).to("cuda", DT[dt])
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        want, mass = want_attention(q, k, v, table, lengths, [1, 1], 0.125)
        shift = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
        out = shift(torch.full((2, 1, 8, 64), 7.0, device="cuda", dtype=DT[dt]))
        got = ops.paged_attention(shift(q), shift(k), shift(v), shift(table), shift(n), 0.125, out=out)
        assert got is out
        close_attention(got, want, mass, dt)


# ---- append --------------------------------------------------------------------------------------------------------------
def want_append(proj, lengths, counts, table, k, v, H, cos, sin, halves, norm, eps):
    proj, table, k, v = host(proj), table.cpu().numpy(), host(k), host(v)
    B, S, _ = proj.shape
    N, G, page, D = k.shape
    q = np.zeros((B, H, S, D))
    for b, s in itertools.product(range(B), range(S)):
        pos = lengths[b] - counts[b] + s
        if s >= counts[b] or pos < 0 or pos >= table.shape[1] * page or (cos is not None and pos >= cos.shape[0]):
            continue
        x = proj[b, s].reshape(H + 2 * G, D)
        y = x[:H + G].copy()
        if cos is not None:
            half = cos.shape[1]
            lo, hi = (slice(0, half), slice(half, 2 * half)) if halves else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
            c, a = host(cos)[pos], host(sin)[pos]
            y[:, lo], y[:, hi] = x[:H + G, lo] * c - x[:H + G, hi] * a, x[:H + G, hi] * c + x[:H + G, lo] * a
        if norm:
            y /= np.sqrt((y * y).mean(-1, keepdims=True) + eps)
        q[b, :, s] = y[:H]
        pg = table[b, pos // page]
        if 0 <= pg < N:
            k[pg, :, pos % page], v[pg, :, pos % page] = y[H:], x[H + G:]
    return q, k, v


def close_append(got, want, dt):
    """One rounding of the result; before it two products and a sum in f32 (of magnitudes up to 2^3 here), and with the norm a factor that is right to some
    2^-21: its sum, square root and quotient."""
    got = host(got)
    bound = HALF[dt] * np.abs(want) + 2.0 ** -21 * np.abs(want) + 2.0 ** -20
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,G,D,rot", [(8, 2, 64, 64), (32, 8, 128, 128), (4, 4, 80, 40), (6, 2, 33, 2), (3, 3, 20, 0), (8, 1, 256, 128), (2, 1, 96, 96)])
@pytest.mark.parametrize("halves,norm", [(True, False), (False, True), (True, True), (False, False)])
def test_append(dt, H, G, D, rot, halves, norm):
    rng = np.random.default_rng(D + rot)
    for page, S, lengths, counts in ((16, 1, [1, 17, 300, 0], None), (10, 3, [3, 21, 100, 0, 2], [3, 1, 2, 0, 2]), (24, 40, [40, 77, 41, 39], [40, 3, 40, 39])):
        k, v, table = cache(rng, lengths, G, D, page, dt)
        n = counts or [S] * len(lengths)
        cos, sin = (torch.from_numpy(f(rng.uniform(0, 7, (310, rot // 2)))).float().cuda() for f in (np.cos, np.sin)) if rot else (None, None)
        proj = torch.from_numpy(rng.standard_normal((len(lengths), S, (H + 2 * G) * D))).to("cuda", DT[dt])
        wq, wk, wv = want_append(proj, lengths, n, table, k, v, H, cos, sin, halves, norm, 1e-5)
        before = k.clone(), v.clone()
        q = ops.paged_rotary_append(proj, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, k, v, H, cos, sin,
                                    None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"), halves, norm, 1e-5)
        close_append(q, wq, dt)
        close_append(k, wk, dt)
        assert same(v, wv)
        untouched = wk == host(before[0])
        assert same(host(k)[untouched], wk[untouched])
        if not rot and not norm:
            assert same(k, wk) and same(q, wq)


def test_tokens_without_a_place_are_not_stored():
    """Positions below zero, behind the block table, behind the rotation table, and on entries that name no page."""
    rng = np.random.default_rng(5)
    k, v, table = cache(rng, [64, 64, 64, 64], 1, 16, 16, "f32")
    table = table[:, :4].contiguous()
    table[2, 1], table[2, 2] = -1, k.shape[0]
    lengths, counts = [2, 66, 48, 48], [3, 4, 40, 4]
    proj = torch.from_numpy(rng.standard_normal((4, 40, 3 * 16))).float().cuda()
    for cos in (None, torch.ones(46, 4, device="cuda")):
        k1, v1 = k.clone(), v.clone()
        wq, wk, wv = want_append(proj, lengths, counts, table, k, v, 1, cos, None if cos is None else cos * 0, True, False, 1e-6)
        q = ops.paged_rotary_append(proj, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, k1, v1, 1, cos, None if cos is None else cos * 0,
                                    counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        assert same(q, wq) and same(k1, wk) and same(v1, wv)


# ---- verification --------------------------------------------------------------------------------------------------------
def want_verify(target, draft, tokens, counts, accept, sample):
    target, tokens, accept, sample = host(target), tokens.cpu().numpy(), host(accept), host(sample)
    draft = host(draft) if draft is not None else None
    B, K1, V = target.shape
    out, taken = np.full((B, K1), -1), np.zeros(B, int)
    for b in range(B):
        n = 0
        while n < counts[b]:
            x = tokens[b, n]
            if not (0 <= x < V and accept[b, n] * (draft[b, n, x] if draft is not None else 1.0) < target[b, n, x]):
                break
            n += 1
        w = np.maximum(target[b, n], 0)
        if n < counts[b]:
            left = np.maximum(target[b, n] - (draft[b, n] if draft is not None else 0), 0)
            if draft is None and 0 <= tokens[b, n] < V:
                left[tokens[b, n]] = 0
            w = left if left.sum() > 0 else w
        out[b, :n], taken[b] = tokens[b, :n], n
        sums = np.cumsum(w)
        if sums[-1] > 0:
            over = np.nonzero((sums > sample[b] * sums[-1]) & (w > 0))[0]
            out[b, n] = over[0] if len(over) else np.nonzero(w)[0][-1]
    return out, taken


def draft_inputs(rng, B, K, V, dt, spread=0.7):
    z = rng.standard_normal((B, K + 1, V)) * 2
    soft = lambda x: np.exp(x) / np.exp(x).sum(-1, keepdims=True)
    target, near = soft(z), soft(z[:, :K] + spread * rng.standard_normal((B, K, V)))
    tokens = np.array([[rng.choice(V, p=near[b, i]) for i in range(K)] for b in range(B)], int).reshape(B, K)
    gpu = lambda x, t: torch.from_numpy(np.asarray(x)).to("cuda", t)
    accept, sample = (rng.integers(0, 1 << 24, n) / float(1 << 24) for n in ((B, K), (B,)))
    return gpu(target, DT[dt]), gpu(near, DT[dt]), gpu(tokens, torch.int32), gpu(accept, torch.float32), gpu(sample, torch.float32)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,K,V", [(1, 4, 32000), (9, 3, 1000), (40, 1, 77), (5, 8, 1), (3, 5, 50257), (2, 2, 128256), (4, 0, 513), (300, 2, 130), (3, 40, 64), (6, 3, 4096)])
@pytest.mark.parametrize("drawn", [True, False])
def test_verify_draft(dt, B, K, V, drawn):
    rng = np.random.default_rng(V + K)
    target, near, tokens, accept, sample = draft_inputs(rng, B, K, V, dt)
    for counts in (None, rng.integers(0, K + 1, B)):
        got, taken = ops.verify_draft(target, tokens, accept, sample, near if drawn else None, None if counts is None else torch.from_numpy(counts).int().cuda())
        want, n = want_verify(target, near if drawn else None, tokens, [K] * B if counts is None else counts, accept, sample)
        assert np.array_equal(taken.cpu().numpy(), n) and np.array_equal(got.cpu().numpy(), want)


def test_drafts_that_all_stand_and_drafts_that_all_fall():
    rng = np.random.default_rng(1)
    target, near, tokens, accept, sample = draft_inputs(rng, 6, 4, 900, "f32")
    got, taken = ops.verify_draft(target, tokens, accept * 0, sample, near)
    assert (taken == 4).all() and torch.equal(got[:, :4], tokens)
    zero = torch.zeros_like(target[:, 0]).scatter_(1, tokens[:, :1].long(), 1.0)
    target[:, 0] *= 1 - zero  # the first draft is impossible
    got, taken = ops.verify_draft(target, tokens, accept * 0, sample, near)
    want, n = want_verify(target, near, tokens, [4] * 6, accept * 0, sample)
    assert (taken == 0).all() and np.array_equal(got.cpu().numpy(), want) and (got[:, 1:] == -1).all()


def test_probabilities_that_leave_nothing():
    """Rows of zeros, rows that the draft covers, a single token with all the weight at either end, NaN, sample just below one."""
    V = 700
    target, draft = torch.zeros(8, 2, V, device="cuda"), torch.zeros(8, 1, V, device="cuda")
    tokens, accept = torch.full((8, 1), 5, dtype=torch.int32, device="cuda"), torch.full((8, 1), 0.5, device="cuda")
    sample = torch.full((8,), 1 - 2.0 ** -24, device="cuda")
    target[1, 0, 0] = 1.0                     # not the drafted token: everything left is token 0
    target[2, 0, V - 1] = 1.0
    target[3, 0, 3:6] = 0.25                  # accepted? 0.5 q < p with q = 0.5: no, 0.25 < 0.25 is false
    draft[3, 0, 3:6] = 0.5                    # and nothing is left of it: from the target itself
    target[4, 0, 5], draft[4, 0, 5] = 0.3, 0.5  # accepted; nothing behind
    target[5, 0], draft[5, 0, 5] = float("nan"), 1.0
    target[6, 0, 10], target[6, 0, 20] = 1.0, 2.0 ** -80
    target[7, 0, 5], draft[7, 0, 5] = float("inf"), 1.0
    target[7, 1, 9] = 1.0
    tokens[2, 0] = V
    tokens[1, 0] = -3
    got, taken = ops.verify_draft(target, tokens, accept, sample, draft)
    assert got.tolist() == [[-1, -1], [0, -1], [V - 1, -1], [5, -1], [5, -1], [-1, -1], [10, -1], [5, 9]]
    assert taken.tolist() == [0, 0, 0, 0, 1, 0, 0, 1]


def test_running_sums_are_held_in_64_bits():
    """One token with nearly all the weight and a hundred thousand behind it with some 2^-30 each: in f32 the running sum would stand still."""
    V = 120000
    target = torch.full((4, 1, V), 2.0 ** -30, device="cuda")
    target[:, 0, 0] = 1.0
    tokens, accept = torch.zeros(4, 0, dtype=torch.int32, device="cuda"), torch.zeros(4, 0, device="cuda")
    sample = torch.tensor([0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -15, 1 - 2.0 ** -14], device="cuda")
    got, taken = ops.verify_draft(target, tokens, accept, sample)
    want, _ = want_verify(target, None, tokens, [0] * 4, accept, sample)
    assert np.array_equal(got.cpu().numpy(), want) and want[1, 0] > 100000 and not taken.any()


# ---- streams, graphs, devices ---------------------------------------------------------------------------------------------
def step_inputs(rng, dt="bf16", B=5, H=8, G=2, D=64, S=3, page=16, V=2000):
    lengths = [3, 50, 333, 700, 4][:B]
    k, v, table = cache(rng, [n + 2 * S for n in lengths], G, D, page, dt)
    proj = torch.from_numpy(rng.standard_normal((B, S, (H + 2 * G) * D))).to("cuda", DT[dt])
    cos, sin = (torch.from_numpy(f(rng.uniform(0, 7, (1000, D // 2)))).float().cuda() for f in (np.cos, np.sin))
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    head = torch.from_numpy(rng.standard_normal((V, H * D))).float().cuda() * 0.3
    _, near, tokens, accept, sample = draft_inputs(rng, B, S - 1, V, "f32")
    return k, v, table, proj, cos, sin, n, head, near, tokens, accept, sample


def probabilities(o, head):
    # this library's product: graphs that replay side by side would share the workspace of torch's
    return torch.softmax(ops.dense_matmul(o.float().flatten(2).flatten(0, 1), head).view(*o.shape[:2], -1), -1)


def step(k, v, table, proj, cos, sin, n, head, near, tokens, accept, sample, H=8):
    """A step of drafted tokens: append, attention, probabilities, verification, and the lengths behind it."""
    S, D = proj.shape[1], k.shape[3]
    q = ops.paged_rotary_append(proj, n, table, k, v, H, cos, sin)
    o = ops.paged_attention(q, k, v, table, n, D ** -0.5)
    p = probabilities(o, head)
    out, taken = ops.verify_draft(p, tokens, accept, sample, near)
    return out, taken, n - S + 1 + taken


def test_a_step_of_drafted_tokens_and_the_next():
    rng = np.random.default_rng(11)
    H, G, D, S = 8, 2, 64, 3
    k, v, table, proj, cos, sin, n, head, near, tokens, accept, sample = step_inputs(rng)
    for _ in range(2):  # the second step overwrites what the first one's rejected drafts stored
        lengths = n.tolist()
        wq, wk, wv = want_append(proj, lengths, [S] * 5, table, k, v, H, cos, sin, True, False, 1e-6)
        out, taken, after = step(k, v, table, proj, cos, sin, n, head, near, tokens, accept, sample)
        close_append(k, wk, "bf16")
        assert same(v, wv)
        q = ops.paged_rotary_append(proj, n, table, k, v, H, cos, sin)
        o = ops.paged_attention(q, k, v, table, n, D ** -0.5)
        want, mass = want_attention(q, k, v, table, lengths, [S] * 5, D ** -0.5)
        close_attention(o, want, mass, "bf16")
        p = probabilities(o, head)
        w, m = want_verify(p, near, tokens, [S - 1] * 5, accept, sample)
        assert np.array_equal(out.cpu().numpy(), w) and np.array_equal(taken.cpu().numpy(), m)
        assert after.tolist() == [a - S + 1 + t for a, t in zip(lengths, m)]
        n = after + S
        proj = torch.from_numpy(rng.standard_normal(tuple(proj.shape))).to("cuda", torch.bfloat16)


def test_a_captured_step_replayed_beside_another():
    """Two graphs with buffers of their own, replayed on two streams at once, with lengths that change between replays."""
    rng = np.random.default_rng(12)
    inputs = [step_inputs(rng), step_inputs(rng)]
    graphs, outputs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    start = [(i[0].clone(), i[1].clone()) for i in inputs]
    for i in inputs:
        step(*i)
    torch.cuda.synchronize()
    for i in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outputs.append(step(*i))
        graphs.append(g)
    for add in (0, 2):
        for i in inputs:
            i[6].add_(add)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for i, out, (k0, v0) in zip(inputs, outputs, start):
            again = step(*i)
            for a, b in zip(out, again):
                assert torch.equal(a, b)
    del graphs, outputs


def test_calls_on_two_streams_and_repeated_calls_give_the_same_bits():
    rng = np.random.default_rng(13)
    for dt, D in (("bf16", 128), ("f32", 64)):
        lengths = [5000, 3, 800]
        k, v, table = cache(rng, lengths, 2, D, 16, dt)
        q = torch.from_numpy(rng.standard_normal((3, 8, 1, D))).to("cuda", DT[dt])
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        want = ops.paged_attention(q, k, v, table, n, 0.1)
        torch.cuda.synchronize()
        results, streams = [], [torch.cuda.Stream() for _ in range(3)]
        for i in range(12):
            with torch.cuda.stream(streams[i % 3]):
                results.append(ops.paged_attention(q, k, v, table, n, 0.1))
        torch.cuda.synchronize()
        assert all(torch.equal(r, want) for r in results)


def test_a_first_call_inside_a_capture():
    """Kernels, limits and sizes that no call before has asked for."""
    for dt, D, H, G, S in ((torch.float16, 192, 8, 2, 3), (torch.float32, 96, 2, 2, 1), (torch.bfloat16, 64, 8, 1, 7)):
        k = torch.randn(40, G, 16, D, device="cuda", dtype=dt)
        table = torch.full((2, 120), -1, dtype=torch.int32, device="cuda")
        table[:, :20] = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
        q, n = torch.randn(2, H, S, D, device="cuda", dtype=dt), torch.tensor([300, 41], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.paged_attention(q, k, k, table, n, 0.1)
        g.replay()
        assert torch.equal(out, ops.paged_attention(q, k, k, table, n, 0.1))
        del g


def test_calls_from_several_threads():
    rng = np.random.default_rng(14)
    k, v, table = cache(rng, [1500, 3, 800], 2, 64, 16, "bf16")
    q, n = torch.from_numpy(rng.standard_normal((3, 8, 1, 64))).to("cuda", torch.bfloat16), torch.tensor([1500, 3, 800], dtype=torch.int32, device="cuda")
    want = ops.paged_attention(q, k, v, table, n, 0.1)
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(ops.paged_attention(q, k, v, table, n, 0.1), want):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ---- refusals ------------------------------------------------------------------------------------------------------------
def test_windows_beyond_32_bits_are_the_whole_past():
    rng = np.random.default_rng(9)
    k, v, table = cache(rng, [100], 1, 64, 16, "bf16")
    q, n = torch.from_numpy(rng.standard_normal((1, 2, 1, 64))).to("cuda", torch.bfloat16), torch.tensor([100], dtype=torch.int32, device="cuda")
    whole = ops.paged_attention(q, k, v, table, n, 0.1)
    assert torch.equal(ops.paged_attention(q, k, v, table, n, 0.1, window=2 ** 32 + 5, sinks=2 ** 33), whole)
    assert torch.equal(ops.paged_attention(q, k, v, table, n, 0.1, window=-1), whole)


def test_a_batch_in_which_nobody_has_a_token():
    k = torch.randn(4, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    table, n, c = torch.zeros(3, 200, dtype=torch.int32, device="cuda"), torch.full((3,), 9, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for dt in (torch.bfloat16, torch.float32):
        out = torch.full((3, 2, 4, 64), 7.0, device="cuda", dtype=dt)
        assert not ops.paged_attention(torch.full((3, 4, 2, 64), float("nan"), device="cuda", dtype=dt), k.to(dt), k.to(dt), table, n, 1.0, counts=c, out=out).any()
    k2, v2 = k.clone(), k.clone()
    q = ops.paged_rotary_append(torch.full((3, 2, 8 * 64), float("nan"), device="cuda", dtype=torch.bfloat16), n, table, k2, v2, 4, counts=c)
    assert not q.any() and torch.equal(k2, k) and torch.equal(v2, k)


def test_empty_batches():
    k = torch.zeros(2, 1, 16, 64, device="cuda", dtype=torch.bfloat16)
    table, n = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    assert ops.paged_attention(torch.zeros(0, 4, 1, 64, device="cuda", dtype=torch.bfloat16), k, k, table, n, 1.0).shape == (0, 1, 4, 64)
    assert ops.paged_rotary_append(torch.zeros(0, 2, 6 * 64, device="cuda", dtype=torch.bfloat16), n, table, k, k, 4).shape == (0, 4, 2, 64)
    out, taken = ops.verify_draft(torch.zeros(0, 3, 50, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, 2, device="cuda"), n.float())
    assert out.shape == (0, 3) and taken.shape == (0,)
    none = torch.zeros(0, 1, 16, 64, device="cuda", dtype=torch.bfloat16)  # a cache without pages
    table, n = torch.full((2, 1), 0, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    assert not ops.paged_attention(torch.ones(2, 4, 1, 64, device="cuda", dtype=torch.bfloat16), none, none, table, n, 1.0).any()
    for dt in (torch.float32, torch.float16):
        q = torch.ones(2 * 4 * 64 + 1, device="cuda", dtype=dt)[1:].view(2, 4, 1, 64)
        assert not ops.paged_attention(q, none.to(dt), none.to(dt), table, n, 1.0, out=torch.ones(2, 1, 4, 64, device="cuda", dtype=dt)).any()
    assert not ops.paged_rotary_append(torch.ones(2, 1, 6 * 64, device="cuda", dtype=torch.bfloat16), n, table, none, none, 4).eq(0).any()


def test_host_tensors_are_refused():
    k = torch.zeros(2, 1, 16, 64)
    table, n = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(torch.zeros(1, 4, 1, 64), k, k, table, n, 1.0)
    with pytest.raises(ValueError, match="tensors on"):
        ops.paged_attention(torch.zeros(1, 4, 1, 64, device="cuda"), k, k, table, n, 1.0)
    with pytest.raises(ValueError, match="contiguous"):
        ops.paged_attention(torch.zeros(1, 2, 4, 64, device="cuda").transpose(1, 2), k.cuda(), k.cuda(), table.cuda(), n.cuda(), 1.0)
