"""Weights of paged attention that are far apart: one key that leads, tails that are the whole output, weights read off one by one."""
import numpy as np
import pytest
import torch

from my_nn_engine_b200 import ops
from test_gpu_paged import DT, HALF, cache, host, want_attention

pytestmark = pytest.mark.gpu


def led(dt, n, lead, at, H, G, D, S, page, scale=1.0, counts=None):
    """One sequence per entry of ``lead``, of n positions: the score of position ``at`` (of each query; -1: the last position that all see) is ``lead``, that of all others 0, to the
    bit; the leading key's value is 0, the others' are 500 to 1500.  So the output is the tail alone."""
    rng = np.random.default_rng(n + D)
    B = len(lead)
    k, v, table = cache(rng, [n] * B, G, D, page, dt)
    k.zero_()
    v.copy_(torch.from_numpy(rng.uniform(500, 1500, tuple(v.shape))))
    at = n - S if at < 0 else at
    for b, x in enumerate(lead):
        pg = int(table[b, at // page])
        k[pg, :, at % page, 0] = x
        v[pg, :, at % page] = 0
        assert (k[pg, :, at % page, 0].float() == x).all()
    q = torch.zeros(B, H, S, D, device="cuda", dtype=DT[dt])
    q[..., 0] = 1.0 / scale
    lengths = torch.full((B,), n, dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, k, v, table, lengths, scale, counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"))
    want, mass = want_attention(q, k, v, table, [n] * B, counts or [S] * B, scale)
    return got, want, mass


def close_led(got, want, mass, dt):
    """One rounding of the output (f16: or half of its smallest step).  A 16-bit cache holds a weight to 2^-16 of itself, or, among the up to 32 positions that it is worked on with, to 2^-38 of the
    largest weight there is, which is at most 1; the sums of some thousand positive terms in f32, in groups of fewer than 200, to 2^-16."""
    got = host(got)
    bound = HALF[dt] * np.abs(want) + 2 * 2.0 ** -16 * mass + 32 * 1500 * 2.0 ** -38 + (2.0 ** -25 if dt == "f16" else 0)
    assert np.isfinite(got).all()
    worst = np.abs(got - want) / bound
    assert (worst <= 1.0).all(), [float(x.max()) for x in worst]


LEADS = [0.0, 10.0, 12.0, 14.0, 16.0, 17.5, 18.0, 20.0, 23.0]


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("group,D", [(1, 64), (4, 128), (12, 64), (12, 128), (20, 128), (40, 64), (8, 192), (12, 256), (24, 256), (60, 192), (3, 40)])
@pytest.mark.parametrize("n", [40, 256, 4096])
def test_a_tail_behind_a_key_that_leads(dt, group, D, n):
    """Pairs that lie in one CTA and pairs that are cut, for every number of warps that share rows; the key that leads comes first, in the middle and last."""
    for at in (0, n // 2 + 5, -1):
        close_led(*led(dt, n, LEADS, at, 2 * group, 2, D, 1, 16), dt)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("S,D", [(3, 64), (5, 128), (9, 192)])
def test_a_tail_behind_a_key_that_leads_drafts(dt, S, D):
    for at in (0, 33, -1):
        close_led(*led(dt, 300, LEADS, at, 8, 2, D, S, 24), dt)
        close_led(*led(dt, 2100, LEADS, at, 8, 2, D, S, 24, counts=[S, 1, 2, S, 0, S, 1, S, S]), dt)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D,H,n", [(64, 2, 64), (128, 8, 100), (256, 20, 256), (40, 1, 33), (64, 40, 50)])
@pytest.mark.parametrize("spread", [1.0, 8.0])
def test_weights_one_by_one(dt, D, H, n, spread):
    """Values that are unit vectors give the weights themselves; scores are multiples of 2^-4 up to ``spread`` and exact.  Beside the output's rounding a weight is off by its
    exponential's 2^-22, that of up to five factors that bring it to another maximum, and the sum's roundings: 64 of 2^-24 in all; a 16-bit cache adds 2^-16."""
    rng = np.random.default_rng(n)
    k, v, table = cache(rng, [n], 1, D, 16, dt)
    k.zero_()
    v.zero_()
    x = rng.integers(-16 * spread, 16 * spread + 1, n) / 16.0
    for j in range(n):
        pg = int(table[0, j // 16])
        k[pg, 0, j % 16, 0], v[pg, 0, j % 16, j % D] = x[j], 1.0
    q = torch.zeros(1, H, 1, D, device="cuda", dtype=DT[dt])
    q[..., 0] = 1.0
    got = host(ops.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0))
    want, _ = want_attention(q, k, v, table, [n], [1], 1.0)
    bound = (HALF[dt] + 64 * 2.0 ** -24 + (2.0 ** -16 if dt != "f32" else 0)) * want + (2.0 ** -25 if dt == "f16" else 0) + (2.0 ** -38 if dt != "f32" else 0)
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("H,G,D,S", [(8, 2, 64, 1), (4, 4, 80, 1), (32, 8, 128, 5), (6, 2, 33, 1), (8, 2, 256, 3)])
def test_scores_that_are_far_apart(dt, H, G, D, S):
    """Queries ten times as large: few keys have nearly all the weight.  A score is a sum of D products in some order, whose partial sums are within three times the root of
    the products' squares, A; D roundings of 2^-24 of those, independent, add up to 3 A sqrt(D) 2^-24, and four times that is allowed for the largest of all."""
    rng = np.random.default_rng(D)
    lengths = [S, 40, 333, 1500]
    k, v, table = cache(rng, lengths, G, D, 16, dt)
    q = torch.from_numpy(10 * rng.standard_normal((4, H, S, D))).to("cuda", DT[dt])
    got = host(ops.paged_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), D ** -0.5))
    want, mass = want_attention(q, k, v, table, lengths, [S] * 4, D ** -0.5)
    A = D ** -0.5 * np.sqrt((host(q) ** 2).max()) * np.sqrt((host(k) ** 2).sum(-1).max())
    weight = 2.0 ** -24 * (12 * A * np.sqrt(D) + 64) + (2.0 ** -16 if dt != "f32" else 0)
    bound = HALF[dt] * np.abs(want) + 2 * weight * mass + (2.0 ** -25 if dt == "f16" else 1e-30)
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cap,spread", [(0.5, 4.0), (30.0, 20.0), (1e3, 30.0), (1e4, 30.0), (1e4, 6000.0), (1e30, 8.0), (1e-3, 8.0)])
@pytest.mark.parametrize("D,H", [(64, 1), (128, 20)])
def test_capped_weights_one_by_one(dt, cap, spread, D, H):
    """Caps far from the scores and close to them.  A capped score is right to 2^-21 of itself (argument, hyperbolic tangent and product), which moves each weight and the sum by
    as much; else as ``test_weights_one_by_one``."""
    rng = np.random.default_rng(int(spread) + D)
    n = 60
    k, v, table = cache(rng, [n], 1, D, 16, dt)
    k.zero_()
    v.zero_()
    step = 4.0 if spread > 1000 else 1 / 16  # scores that all types hold
    x = np.round(rng.uniform(-spread, spread, n) / step) * step if spread < 1000 else 5632.0 + 32 * rng.integers(0, 3, n)
    for j in range(n):
        pg = int(table[0, j // 16])
        k[pg, 0, j % 16, 0], v[pg, 0, j % 16, j % D] = x[j], 1.0
    x = np.array([float(k[int(table[0, j // 16]), 0, j % 16, 0]) for j in range(n)])
    q = torch.zeros(1, H, 1, D, device="cuda", dtype=DT[dt])
    q[..., 0] = 1.0
    got = host(ops.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0, softcap=cap))
    want, _ = want_attention(q, k, v, table, [n], [1], 1.0, cap=float(np.float32(cap)))
    score = np.abs(cap * np.tanh(x / cap)).max() * 2.0 ** -21
    bound = (HALF[dt] + 64 * 2.0 ** -24 + (2.0 ** -16 if dt != "f32" else 0) + 2 * score) * want + (2.0 ** -25 if dt == "f16" else 0) + (2.0 ** -38 if dt != "f32" else 0)
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()
