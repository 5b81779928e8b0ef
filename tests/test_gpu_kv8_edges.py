"""8-bit KV cache on the GPU at the ends of its ranges: large counts, values far from one, tensors that do not fit a call."""
import math

import numpy as np
import pytest

import kv8_ref as R
import lastro_b200 as LB

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv8 import Gpu, bounds, check_attend, ctx, f64, filled, ints, rows, same_values  # noqa: E402, F401


def code_of(f, *a, **kw):
    with pytest.raises(LB.LastroError) as e:
        f(*a, **kw)
    assert "kv8" in str(e.value)
    return e.value.code


# ---- counts -------------------------------------------------------------------------------------------------------------
def test_append_with_a_bound_far_above_its_rows(ctx):
    """max_new is an upper bound: one that times the heads passes 32 bits changes nothing"""
    kv, d, pages = 64, 64, 1 << 23
    gpu, ref, rng = filled(ctx, "e4m3", kv, d, [20], max_pages=2)
    wide = torch.full((1, pages), 2 ** 30, dtype=torch.int32, device="cuda")
    wide[:, :2] = gpu.table
    c = LB.Kv8Cache(ctx, "e4m3", 1, kv, d, gpu.num_pages, pages, gpu.k, gpu.v, gpu.ks, gpu.vs, wide, gpu.status)
    k, v = (rows(rng, 30, kv, d, "bf16") for _ in "kv")
    out = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.append(ints([20]), ints([0, 30]), 1 << 29, LB.rows_of(k), LB.rows_of(v), out)
    ref.append(0, f64(k), f64(v))
    assert out.tolist() == [50] and gpu.status.item() == 0
    same_values(gpu, ref, [50])


def test_append_of_more_rows_than_can_be_counted_is_refused(ctx):
    kv, pages = 64, 1 << 24
    gpu, _, _ = filled(ctx, "e4m3", kv, 64, [20], max_pages=1)
    table, out = torch.zeros(1, pages, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    c = LB.Kv8Cache(ctx, "e4m3", 1, kv, 64, gpu.num_pages, pages, gpu.k, gpu.v, gpu.ks, gpu.vs, table, gpu.status)
    x = torch.zeros(64, device="cuda")
    one = LB.Rows(x.data_ptr(), LB.DTYPE_F32, 2 ** 31 - 1, 0, 0)  # one row given 2^31 - 1 times
    assert code_of(c.append, ints([0]), ints([0, 1]), 1 << 30, one, one, out) == LB.E_UNSUPPORTED
    torch.cuda.synchronize()
    assert gpu.status.item() == 0


# ---- shared memory ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("news", [1, 12])
def test_copies_that_follow_the_list_closely(ctx, news):
    """many short sequences: the list is written several times over where the first copies go; every repeat gives the same"""
    lens = (np.arange(1500) * 7 % 61 + 12).tolist()
    gpu, ref, rng = filled(ctx, "int8", 1, 64, lens)
    check_attend(gpu, ref, rng, lens, [news] * len(lens), 2, "bf16")
    q = [rows(rng, news, 2, 64, "bf16") for _ in lens]
    first = gpu.attend(lens, q, 0.125, mass=True)
    for _ in range(30):
        again = gpu.attend(lens, q, 0.125, mass=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
