"""Paged attention with many query rows per kv head: prompts and chunks of them, behind tables that pairs are cut for."""
import pytest
import torch

from my_nn_engine_b200 import ffi, ops
from test_gpu_paged import DT, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [40, 64, 128, 192, 256])
@pytest.mark.parametrize("group", [1, 4, 8])
def test_scratch_is_bounded_whatever_the_number_of_tokens(D, group):
    """Eight parts of 64 rows of 256 numbers, their maxima and sums per CTA that is resident: 78.3 MB on 148 SMs."""
    torch.cuda.init()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for S in (1, 5, 17, 100, 512, 777, 2048, 65536 // group):
        n = ffi.lib().mynn_b200_paged_attention_workspace_bytes(6, S, 8 * group, 8, D, 16, 2000)
        assert n <= sms * 8 * (64 * 258 * 4 + 16), (S, n)
        assert S > 512 or n > 0


@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("bf16", 192), ("f32", 64), ("f32", 20)])
@pytest.mark.parametrize("H,G,S", [(4, 1, 50), (8, 1, 150), (6, 2, 333), (8, 1, 601)])
def test_prompts(dt, D, H, G, S):
    """4 to 76 blocks of 64 rows, 25 to 601 of eight: cut pairs, whole ones in fewer CTAs than blocks, several waves."""
    run_attention(S + D, dt, [S + 1400, S, S // 2, 0], H, G, D, 16, S, [S, S - 1, S // 2, 0])


def test_a_chunk_behind_a_window():
    run_attention(5, "bf16", [2500, 700], 8, 2, 128, 24, 260, [260, 130], window=300, sinks=5)
    run_attention(6, "f32", [1500, 300], 4, 2, 64, 24, 130, [130, 1], window=100, sinks=5)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 3])
def test_windows_of_nearly_all_positions_there_can_be(dt, S):
    """The last position a length can have, over a table of 64: what is seen of it follows from the window to the position.  Both sides are rounded once, so they differ by a step at most."""
    k, v = torch.randn(4, 2, 16, 64, device="cuda").to(DT[dt]), torch.randn(4, 2, 16, 64, device="cuda").to(DT[dt])
    table, q = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), torch.randn(1, 4, S, 64, device="cuda").to(DT[dt])
    last = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda")
    for first in (0, 1, 17, 50, 63):  # the first position that the oldest query sees
        near = torch.tensor([64], dtype=torch.int32, device="cuda")
        got = ops.paged_attention(q, k, v, table, last, 0.1, window=2 ** 31 - 1 - S - first + 1)
        want = torch.cat([ops.paged_attention(q[:, :, s:s + 1].contiguous(), k, v, table, near, 0.1, window=64 - first - s) if first + s < 64 else torch.zeros_like(got[:, :1]) for s in range(S)], 1)
        assert torch.allclose(got.float(), want.float(), rtol=2.0 ** -7 if dt == "bf16" else 1e-5, atol=1e-5) and got[:, 0].any()
    assert torch.equal(ops.paged_attention(q, k, v, table, last, 0.1, window=2 ** 31 - 1), ops.paged_attention(q, k, v, table, last, 0.1))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_windows_below_32_bits_are_none_and_first_positions_below_zero_are_refused(dt):
    k, table = torch.randn(4, 2, 16, 64, device="cuda").to(DT[dt]), torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    q, n = torch.randn(1, 4, 1, 64, device="cuda").to(DT[dt]), torch.tensor([64], dtype=torch.int32, device="cuda")
    whole = ops.paged_attention(q, k, k, table, n, 0.1)
    for window in (-1, -2 ** 31, 5 - 2 ** 32, 5 - 2 ** 40):
        assert torch.equal(ops.paged_attention(q, k, k, table, n, 0.1, window=window), whole)
    for sinks in (-1, 4 - 2 ** 32, 4 - 2 ** 40):
        with pytest.raises(RuntimeError, match="first positions"):
            ops.paged_attention(q, k, k, table, n, 0.1, window=5, sinks=sinks)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("width", [100, 3])
def test_idle_sequences_among_prompts_are_zeros(dt, width):
    """Fewer CTAs than sequences, several blocks of rows: every element of an idle sequence is written by one of them."""
    B, S, H, G, D = 40, 700, 4, 1, 64
    counts = [S if b == 7 else 0 for b in range(B)]
    k = torch.randn(50, G, 16, D, device="cuda").to(DT[dt])
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    table[7, :min(width, 44)] = torch.arange(min(width, 44), dtype=torch.int32, device="cuda")
    q = torch.randn(B, H, S, D, device="cuda").to(DT[dt])
    n, c = torch.full((B,), 700, dtype=torch.int32, device="cuda"), torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = torch.full((B, S, H, D), float("nan"), device="cuda", dtype=DT[dt])
    ops.paged_attention(q, k, k, table, n, 0.1, counts=c, out=out)
    assert torch.isfinite(out).all() and out[7].any() and not out[:7].any() and not out[8:].any()


@pytest.mark.parametrize("dt,D,group", [("f16", 128, 4), ("bf16", 64, 2), ("f16", 64, 8), ("f32", 64, 4)])
@pytest.mark.parametrize("scale", [0.1, 0.6])
def test_other_queries_leave_a_query_its_bits(dt, D, group, scale):
    """Keys that only the last query sees, infinite or so large that its weights are all but one, over many batches: the first queries' outputs do not change by a bit."""
    g = torch.Generator("cuda").manual_seed(D)
    B, G, S, n = 48, 2, 4, 130
    table = torch.randperm(B * 9, generator=g, device="cuda").int().view(B, 9)
    lengths = torch.full((B,), n, dtype=torch.int32, device="cuda")
    for _ in range(4):
        k, v = (torch.randn(B * 9, G, 16, D, generator=g, device="cuda").to(DT[dt]) for _ in range(2))
        q = torch.randn(B, G * group, S, D, generator=g, device="cuda").to(DT[dt])
        q[..., 0] = 1.0
        clean = ops.paged_attention(q, k, v, table, lengths, scale)
        for bad in (float("inf"), float("nan"), 300.0, -300.0):
            k2 = k.clone()
            k2[table[:, (n - 1) // 16].long(), :, (n - 1) % 16, 0] = bad
            assert torch.equal(ops.paged_attention(q, k2, v, table, lengths, scale)[:, :S - 1], clean[:, :S - 1])
