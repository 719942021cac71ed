"""Configuration and host-side refusals of the expert and 8-bit operators (CPU only)."""
import dataclasses

import pytest
import torch

from llm_infer_rust_amd import experts, int8
from llm_infer_rust_amd._native import NativeError, lib
from llm_infer_rust_amd.kv_cache import ModelError
from llm_infer_rust_amd.model import Qwen3Config

A, B, C, D = 0x10000, 0x20000, 0x30000, 0x40000  # 16-byte aligned, never dereferenced


def err(r):
    assert r is not None
    return r.decode()


def test_expert_configuration():
    cfg = dataclasses.replace(Qwen3Config.qwen3_0_6b(), num_experts=64, num_experts_per_tok=4,
                              moe_intermediate_size=256)
    cfg.validate()
    Qwen3Config.qwen3_8b().validate()
    for bad in (dict(num_experts_per_tok=0), dict(num_experts_per_tok=65),
                dict(moe_intermediate_size=0), dict(num_experts=1025), dict(num_experts=-1)):
        with pytest.raises(ModelError):
            dataclasses.replace(cfg, **bad).validate()


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 16, dtype=torch.bfloat16)
    ids, w = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1)
    for call in (lambda: int8.quantize_rows(x), lambda: int8.Int8Weight.quantize(x),
                 lambda: int8.Int8Weight(torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)),
                 lambda: experts.route_experts(x, 2),
                 lambda: experts.expert_mlp(x, ids, w, torch.zeros(1, 32, 16, dtype=x.dtype),
                                            torch.zeros(1, 16, 16, dtype=x.dtype))):
        with pytest.raises(NativeError):
            call()


def test_entries_refuse_bad_arguments_before_launching():
    f = lib()
    q = f.mi355x_quantize_rows
    assert q(None, 16, None, 16, None, 0, 16, 0, None) is None  # no rows: nothing to do
    assert "null" in err(q(None, 16, B, 16, C, 1, 16, 0, None))
    assert "shape" in err(q(A, 15, B, 16, C, 2, 16, 0, None))
    assert "shape" in err(q(A, 16, B, 17, C, 2, 16, 0, None))
    assert "shape" in err(q(A, 16, B, 16, C, 2, 16, 3, None))
    assert "misaligned" in err(q(A, 16, B + 4, 16, C, 2, 16, 0, None))

    ws = f.mi355x_linear_int8_workspace_bytes
    assert ws(1, 64, 4096, 256) == 0 and ws(0, 64, 64, 256) == 0
    assert ws(40, 64, 100, 256) >= 40 * 128 + 160
    assert ws(40, 64, int8.MAX_K + 1, 256) == -1 and ws(-1, 64, 64, 256) == -1
    # K split in parts where the tiles would leave most compute units idle
    assert ws(64, 4096, 12288, 256) >= 64 * 12288 + 2 * 64 * 4096 * 4
    need = ws(40, 64, 100, 256)

    def lin(x=A, ldx=100, w=B, ldw=112, s=C, out=D, ldo=64, m=40, n=64, k=100, silu=False, wsp=A,
            size=need, dt=0):
        return f.mi355x_linear_int8(x, ldx, w, ldw, s, out, ldo, m, n, k, silu, wsp, size, 256, dt,
                                    None)
    assert lin(m=0) is None
    assert "null" in err(lin(x=None)) and "null" in err(lin(wsp=None))
    assert "too small" in err(lin(size=need - 1))
    for bad in (dict(ldw=100), dict(ldw=120), dict(ldx=99), dict(ldo=63), dict(k=int8.MAX_K + 1),
                dict(n=63, silu=True), dict(dt=2), dict(m=-1), dict(n=0),
                dict(ldw=1 << 26, n=64)):
        assert "shape" in err(lin(**bad)), bad
    assert "misaligned" in err(lin(w=B + 8))

    def route(x=A, ld=8, t=4, e=8, k=2, dt=0):
        return f.mi355x_route_experts(x, ld, B, C, t, e, k, True, dt, None)
    assert route(t=0) is None
    assert "null" in err(route(x=None))
    for bad in (dict(e=1025, ld=1025), dict(k=9), dict(k=0), dict(ld=7), dict(dt=3), dict(t=-1),
                dict(e=200, ld=200, k=65)):
        assert "shape" in err(route(**bad)), bad

    size = f.mi355x_expert_mlp_workspace_bytes
    assert size(0, 2, 8, 64, 32, 64, False, 256) >= 0
    assert size(4, 2, 8, 60, 32, 64, False, 256) == -1 and size(4, 2, 8, 60, 32, 64, True, 256) > 0
    assert size(4, 65, 8, 64, 32, 64, False, 256) == -1 and size(4, 2, 1025, 64, 32, 64, False, 256) == -1
    assert size(4, 2, 8, 64, 32, 63, False, 256) == -1
    # the slots of one pass bound the workspace, however many tokens there are
    assert size(1 << 22, 8, 8, 64, 32, 64, False, 256) < 131072 * (32 + 64 + 64) * 4
    need = size(40, 2, 8, 64, 32, 64, False, 256)

    def mlp(x=A, ldx=64, ids=B, gu=C, ldg=64, gs=None, dn=D, ldd=32, ds=None, t=40, k=2, e=8,
            h=64, i=32, wsp=A, n=need, dt=0, ldo=64):
        return f.mi355x_expert_mlp(x, ldx, ids, B, gu, ldg, gs, dn, ldd, ds, C, ldo, t, k, e, h, i,
                                   wsp, n, 256, dt, None)
    assert mlp(t=0) is None
    assert "null" in err(mlp(ids=None)) and "null" in err(mlp(wsp=None))
    assert "too small" in err(mlp(n=need - 1))
    assert "one kind" in err(mlp(gs=A)) and "one kind" in err(mlp(ds=A))
    for bad in (dict(ldx=63), dict(ldx=68), dict(ldg=63), dict(ldd=36), dict(h=60), dict(i=30),
                dict(k=0), dict(e=0), dict(dt=2), dict(ldo=63), dict(t=-1)):
        assert "shape" in err(mlp(**bad)), bad
    assert "4 GiB" in err(mlp(h=131072, i=131072, ldx=131072, ldo=131072, ldg=131072, ldd=131072))
    assert "misaligned" in err(mlp(x=A + 8)) and "misaligned" in err(mlp(gu=C + 8))
