"""What the operators over paged caches refuse, before anything touches a device."""
import ctypes

import pytest
import torch

from my_nn_engine_b200 import ffi, ops

P = ctypes.c_void_p(256)


def attention(B=1, S=1, Hq=4, Hkv=2, D=64, page=16, pages=4, width=2, dtype=ffi.BF16, sinks=0, ws=None):
    return ffi.lib().mynn_b200_paged_attention(None, P, P, P, P, P, P, None, 1.0, 0.0, 0, sinks, B, S, Hq, Hkv, D, page, pages, width, dtype, ws, 0)


def append(B=1, S=1, Hq=4, Hkv=2, D=64, rot=64, page=16, pages=4, width=2, positions=9, dtype=ffi.BF16, tables=P):
    return ffi.lib().mynn_b200_paged_rotary_append(None, P, P, P, P, tables, tables, P, None, P, B, S, Hq, Hkv, D, rot, 1, 0, 1e-6, page, pages, width, positions, dtype)


def verify(B=1, K=2, V=100, dtype=ffi.F32, tokens=P):
    return ffi.lib().mynn_b200_verify_draft(None, P, P, P, None, tokens, None, P, P, B, K, V, dtype)


@pytest.mark.parametrize("bad", [dict(B=-1), dict(S=0), dict(Hq=0), dict(Hkv=0), dict(Hq=5), dict(D=0), dict(page=0), dict(width=0), dict(pages=-1), dict(sinks=-1), dict(dtype=7)])
def test_attention_refuses_bad_arguments(bad):
    assert attention(**bad) == ffi.E_ARG and "paged_attention" in ffi.last_error()


@pytest.mark.parametrize("bad", [dict(D=257), dict(page=1 << 20, width=1 << 12), dict(S=1 << 17), dict(pages=1 << 24, page=64, Hkv=2)])
def test_attention_refuses_sizes_beyond_its_limits(bad):
    assert attention(**bad) == ffi.E_UNSUPPORTED and "paged_attention" in ffi.last_error()


@pytest.mark.parametrize("bad", [dict(B=-1), dict(S=0), dict(Hq=0), dict(Hkv=0), dict(D=0), dict(rot=-2), dict(rot=66), dict(rot=3), dict(page=0), dict(pages=-1), dict(width=0),
                                 dict(positions=-1), dict(dtype=7), dict(tables=None)])
def test_append_refuses_bad_arguments(bad):
    assert append(**bad) == ffi.E_ARG and "paged_rotary_append" in ffi.last_error()


@pytest.mark.parametrize("bad", [dict(D=1025), dict(page=1 << 20, width=1 << 12), dict(B=1 << 20, S=1 << 20)])
def test_append_refuses_sizes_beyond_its_limits(bad):
    assert append(**bad) == ffi.E_UNSUPPORTED and "paged_rotary_append" in ffi.last_error()


@pytest.mark.parametrize("bad,code", [(dict(B=-1), ffi.E_ARG), (dict(K=-1), ffi.E_ARG), (dict(V=0), ffi.E_ARG), (dict(dtype=9), ffi.E_ARG), (dict(tokens=None), ffi.E_ARG),
                                      (dict(K=1025), ffi.E_UNSUPPORTED), (dict(B=65536), ffi.E_UNSUPPORTED), (dict(V=(1 << 30) + 1), ffi.E_UNSUPPORTED)])
def test_verification_refuses(bad, code):
    assert verify(**bad) == code and "verify_draft" in ffi.last_error()


def test_empty_batches_touch_nothing():
    assert attention(B=0) == ffi.OK and append(B=0) == ffi.OK and verify(B=0) == ffi.OK
    assert ffi.lib().mynn_b200_paged_attention_workspace_bytes(0, 1, 4, 2, 64, 16, 2) == 0
    assert ffi.lib().mynn_b200_paged_attention_workspace_bytes(1, 1, 5, 2, 64, 16, 2) == 0


def test_shapes_and_types_are_checked_in_python():
    q, k = torch.zeros(2, 4, 1, 64), torch.zeros(3, 2, 16, 64)
    table, n = torch.zeros(2, 5, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for args, what in (((q, k, k[:, :1], table, n), "one shape"), ((q, k.half(), k.half(), table, n), "dtype"), ((q, k, k, table[:1], n), "block_table"),
                       ((q, k, k, table.long(), n), "block_table"), ((q, k, k, table, n[:1]), "lengths"), ((q, k, k, table, n.float()), "lengths"),
                       ((q, k[..., :32], k[..., :32], table, n), "heads of"), ((q, k, k, table[0], n), "block_table")):
        with pytest.raises((ValueError, TypeError), match=what):
            ops.paged_attention(*args, 1.0)
    with pytest.raises(ValueError, match="counts"):
        ops.paged_attention(q, k, k, table, n, 1.0, counts=n[:1])
    proj = torch.zeros(2, 3, 8 * 64)
    for kw, what in ((dict(heads=5), "columns"), (dict(heads=4, cos=torch.zeros(9, 32)), "cos and sin"), (dict(heads=4, cos=torch.zeros(9, 32), sin=torch.zeros(9, 31)), "cos and sin"),
                     (dict(heads=4, cos=torch.zeros(9, 32).half(), sin=torch.zeros(9, 32).half()), "cos and sin")):
        with pytest.raises(ValueError, match=what):
            ops.paged_rotary_append(proj, n, table, k, k, **kw)
    target, tokens, accept, sample = torch.zeros(2, 4, 50), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3), torch.zeros(2)
    for args, kw, what in (((target, tokens.long(), accept, sample), {}, "tokens"), ((target, tokens[:, :2], accept, sample), {}, "tokens"),
                           ((target, tokens, accept.double(), sample), {}, "accept"), ((target, tokens, accept, sample[:1]), {}, "accept"),
                           ((target, tokens, accept, sample), dict(draft=target), "draft"), ((target, tokens, accept, sample), dict(draft=target[:, :3].half()), "draft"),
                           ((target, tokens, accept, sample), dict(counts=tokens), "counts")):
        with pytest.raises(ValueError, match=what):
            ops.verify_draft(*args, **kw)
