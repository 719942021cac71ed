"""Every form that the 8-bit and expert products take by size: what is chosen (on the host), and the
results of the forms that the other tests' sizes do not reach. The sizes are chosen for 256 compute
units; a change of the estimates that moves one to another form fails here without a GPU.

Bounds as in test_gpu_int8.py and, column by column, test_gpu_experts_columns.py.
"""
import ctypes

import pytest
import torch

import test_gpu_experts as older
import test_gpu_int8 as older8
from llm_infer_rust_amd import experts, int8
from llm_infer_rust_amd._native import check as ok, lib
from test_gpu_experts_columns import SHAPES as COLUMNS, bounds16, bounds8
from test_gpu_int8 import check

VEC, ROWS, TILES = 0, 1, 2
T64, T128, T128_TWO, T256X128, T256 = range(5)


def linear_plan(t, n, k):
    plan = (ctypes.c_int32 * 3)()
    assert lib().mi355x_linear_int8_plan(t, n, k, 256, plan)
    return tuple(plan)


def expert_plan(t, e, k, h, i, i8):
    plan = (ctypes.c_int32 * 4)()
    assert lib().mi355x_expert_mlp_plan(t, k, e, h, i, h, i8, 256, plan)
    return tuple(plan)


# Vector math past its first 4,096 columns (a batch of its loop) and its first 16,384 (rows that are
# read twice to be quantised), up to the longest that it takes, and just past that.
VECTOR = [(1, 66, 4112), (1, 130, 12288), (1, 34, 20001), (1, 34, 32768), (2, 66, 4112),
          (2, 130, 12288), (2, 34, 5003), (2, 34, 16384)]
# The rows kernel past the four steps a wave that it starts with, with ragged ends.
FEW_ROWS = [(3, 4100, 4096), (9, 8200, 12288), (16, 6146, 4096), (5, 8200, 5003), (16, 66, 2500),
            (2, 8200, 16400)]
# One row and few rows whose K is cut in parts on tiles.
PARTS = [(1, 34, 32780), (2, 34, 16400), (3, 130, 4096)]


@pytest.mark.parametrize("shapes,kind", [(VECTOR, VEC), (FEW_ROWS, ROWS), (PARTS, TILES)])
def test_linear_choice(shapes, kind):
    for s in shapes:
        assert linear_plan(*s)[0] == kind, s


def test_linear_tiles_of_the_other_tests():
    met = {linear_plan(*s) for s in older8.SHAPES + older8.LARGE}
    for form in ((VEC, T64, 1), (ROWS, T64, 1), (TILES, T64, 1), (TILES, T64, 2), (TILES, T64, 4),
                 (TILES, T64, 8), (TILES, T128, 1), (TILES, T128, 2), (TILES, T128_TWO, 1),
                 (TILES, T256X128, 1), (TILES, T256, 1)):
        assert form in met, form


def test_plans_of_empty_and_invalid_shapes():
    plan = (ctypes.c_int32 * 4)()
    assert not lib().mi355x_linear_int8_plan(0, 8, 8, 256, plan)
    assert not lib().mi355x_linear_int8_plan(1, 8, int8.MAX_K + 1, 256, plan)
    assert not lib().mi355x_linear_int8_plan(1, 8, 8, 256, None)
    assert not lib().mi355x_expert_mlp_plan(0, 2, 8, 64, 64, 64, False, 256, plan)
    assert not lib().mi355x_expert_mlp_plan(1, 2, 8, 60, 64, 60, False, 256, plan)
    assert not lib().mi355x_expert_mlp_plan(1, 2, 8, 64, 64, 64, False, 256, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,k", VECTOR + FEW_ROWS + PARTS)
@pytest.mark.parametrize("silu", [False, True])
def test_linear_int8(gpu, dtype, t, n, k, silu):
    g = torch.Generator(device=gpu).manual_seed(t + n + k)
    x = torch.randn(t, k, generator=g, device=gpu).to(dtype)
    x[:, k - 1] *= 8.0  # the row's largest value at its end
    weight = int8.Int8Weight.quantize(torch.randn(n, k, generator=g, device=gpu) * k ** -0.5)
    check(int8.linear_int8(x, weight, silu_mul=silu), x, weight, silu)


# Slots one by one: the down product with 16, 32 and 64 lanes a slot (its weight row up to 768, 1,536
# and more bytes), more slots a token than it takes at once, K past a pass of its loop, gate_up past
# its first 4,096 bytes.
ONE_BY_ONE = [(1, 8, 2, 264, 384), (2, 8, 2, 264, 768), (1, 6, 3, 136, 1040), (1, 5, 2, 4104, 2056),
              (1, 8, 8, 2056, 768), (1, 16, 12, 64, 64), (3, 32, 16, 72, 40), (2, 16, 12, 136, 1040),
              (1, 16, 9, 72, 1544), (3, 6, 5, 64, 768)]
ONE_BY_ONE_8 = ONE_BY_ONE + [(1, 4, 2, 5001, 1041), (2, 5, 2, 333, 2057), (1, 2, 2, 20001, 67),
                             (1, 16, 13, 65, 1537), (1, 2, 2, 64, 16001)]
# Grouped: (shape, 16 bits, 8 bits), each gate_up tile, down tile and parts of K.
GROUPED = [((40, 6, 2, 104, 2056), (T64, T64, 4), (T64, T64, 2)),
           ((90, 2, 2, 72, 4104), (T64, T64, 4), (T64, T64, 4)),
           ((60, 4, 2, 264, 1288), (T64, T64, 2), (T64, T64, 1)),
           ((77, 8, 2, 264, 520), (T64, T64, 1), (T64, T64, 1)),
           ((1200, 2, 2, 72, 1032), (T128_TWO, T64, 2), (T128_TWO, T64, 1)),
           ((1200, 2, 2, 2056, 72), (T64, T128_TWO, 1), (T64, T128_TWO, 1)),
           ((2500, 6, 2, 1032, 520), (T128_TWO, T128_TWO, 1), (T128_TWO, T128_TWO, 1)),
           ((2100, 5, 2, 2056, 72), (T64, T256, 1), (T64, T256, 1)),
           ((4100, 5, 2, 1032, 520), (T256, T256, 1), (T256, T256, 1)),
           ((3000, 3, 2, 512, 1024), (T256, T64, 1), (T256, T64, 1)),
           ((3000, 3, 2, 2056, 128), (T64, T256, 1), (T64, T256, 1))]


def test_expert_choice():
    for s in ONE_BY_ONE:
        assert expert_plan(*s, False)[0] == 1, s
    for s in ONE_BY_ONE_8:
        assert expert_plan(*s, True)[0] == 1, s
    for s, bits16, bits8 in GROUPED:
        assert expert_plan(*s, False) == (0, *bits16), s
        assert expert_plan(*s, True) == (0, *bits8), s
    # all of them run in the other tests, but for those of K in two parts, which run here
    met = set(older.SHAPES + older.LARGE + COLUMNS)
    assert {s for s, _, _ in GROUPED} - met == {(60, 4, 2, 264, 1288)}


def problem(t, e, k, h, i, dtype, gpu):
    g = torch.Generator(device=gpu).manual_seed(t + h + i)
    x = torch.randn(t, h, generator=g, device=gpu).to(dtype)
    ids = torch.rand(t, e, generator=g, device=gpu).argsort(1)[:, :k].to(torch.int32).contiguous()
    w = torch.rand(t, k, generator=g, device=gpu)
    gu = (torch.randn(e, 2 * i, h, generator=g, device=gpu) * h ** -0.5).to(dtype)
    dn = (torch.randn(e, h, i, generator=g, device=gpu) * i ** -0.5).to(dtype)
    return x, ids, w, gu, dn


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,h,i", ONE_BY_ONE + [(60, 4, 2, 264, 1288)])
def test_expert_mlp(gpu, dtype, t, e, k, h, i):
    p = problem(t, e, k, h, i, dtype, gpu)
    out, bound = bounds16(*p)
    err = (experts.expert_mlp(*p).double() - out).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k,h,i", ONE_BY_ONE_8 + [(60, 4, 2, 264, 1288)])
def test_expert_mlp_int8(gpu, dtype, t, e, k, h, i):
    x, ids, w, gu, dn = problem(t, e, k, h, i, dtype, gpu)
    gu, dn = int8.Int8Weight.quantize(gu), int8.Int8Weight.quantize(dn)
    out, bound = bounds8(x, ids, w, gu, dn)
    err = (experts.expert_mlp(x, ids, w, gu, dn).double() - out).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


# 8-bit weight rows of whole 16-byte words that end inside a 128-byte step, which the C entry takes:
# one by one, and every tile of either product, K whole and in parts.
TAILS = [((2, 8, 2, 150, 150), (1, T64, T64, 1)), ((77, 8, 2, 150, 150), (0, T64, T64, 1)),
         ((90, 2, 2, 72, 4104), (0, T64, T64, 4)), ((1200, 2, 2, 150, 1032), (0, T128_TWO, T64, 1)),
         ((1200, 2, 2, 2056, 150), (0, T64, T128_TWO, 1)), ((2100, 5, 2, 150, 1032), (0, T256, T64, 1)),
         ((2100, 5, 2, 2056, 150), (0, T64, T256, 1)), ((4100, 5, 2, 1030, 520), (0, T256, T256, 1))]


def test_tail_choice():
    for s, plan in TAILS:
        assert expert_plan(*s, True) == plan, s


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,i", [s for s, _ in TAILS])
def test_expert_weight_rows_of_whole_16_byte_words(gpu, t, e, k, h, i):
    """The padding of any value: the same result as with rows of whole steps."""
    g = torch.Generator(device=gpu).manual_seed(t)
    x, ids, w, _, _ = problem(t, e, k, h, 8, torch.bfloat16, gpu)
    ldg, ldd = -(-h // 16) * 16, -(-i // 16) * 16
    gv = torch.randint(-128, 128, (e, 2 * i, ldg), generator=g, device=gpu, dtype=torch.int8)
    dv = torch.randint(-128, 128, (e, h, ldd), generator=g, device=gpu, dtype=torch.int8)
    gs = torch.rand(e, 2 * i, generator=g, device=gpu) * (0.02 / h ** 0.5)
    ds = torch.rand(e, h, generator=g, device=gpu) * 0.01
    want = experts.expert_mlp(x, ids, w, int8.Int8Weight(gv[..., :h], gs),
                              int8.Int8Weight(dv[..., :i], ds))
    assert bool(want.isfinite().all()) and bool((want != 0).any())
    out = torch.empty_like(want)
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    need = lib().mi355x_expert_mlp_workspace_bytes(t, k, e, h, i, h, True, cus)
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    ok(lib().mi355x_expert_mlp(
        x.data_ptr(), h, ids.data_ptr(), w.data_ptr(), gv.data_ptr(), ldg, gs.data_ptr(),
        dv.data_ptr(), ldd, ds.data_ptr(), out.data_ptr(), h, t, k, e, h, i, ws.data_ptr(), need,
        cus, 0, torch.cuda.current_stream().cuda_stream), "expert_mlp")
    torch.cuda.synchronize()
    assert torch.equal(out, want)
