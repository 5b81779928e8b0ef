"""The 8-bit KV cache's host side: what is refused without a GPU, and the plain 64-bit form the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import kv8_ref as R
import lastro_b200 as LB


def test_calls_without_a_context_are_refused():
    L = LB.lib()
    d, r = LB.Kv8Desc(), LB.Rows()
    n = C.c_size_t()
    assert L.lastro_kv8_append(None, d, None, None, 1, r, r, None, None, 0) == LB.E_ARG
    assert L.lastro_kv8_attend_workspace(None, d, 1, 1, 0, C.byref(n)) == LB.E_ARG
    assert L.lastro_kv8_attend(None, d, None, None, 1, 1, r, 1.0, r, None, None, 0, None, 0) == LB.E_ARG
    assert L.lastro_kv8_evict(None, d, d, None, 1, 1, None, 0, None, None, None, 0) == LB.E_ARG
    assert L.lastro_kv8_read(None, d, None, None, 1, None, None, LB.DTYPE_BF16) == LB.E_ARG


def test_formats_and_row_types_are_checked_on_the_host():
    torch = pytest.importorskip("torch")
    with pytest.raises(LB.LastroError):
        LB.Kv8Cache(None, "fp4", 1, 1, 64, 1, 1, 0, 0, 0, 0, 0)
    t = torch.zeros(4, 2, 64)
    r = LB.rows_of(t[:, :, :64])
    assert (r.rows, r.row_stride, r.head_stride, r.dtype) == (4, 128, 64, LB.DTYPE_F32)
    assert LB.rows_of(t.bfloat16().transpose(0, 1)).row_stride == 64
    for bad in (t.half(), t[0], t[:, :, ::2], t.transpose(1, 2)):
        with pytest.raises(LB.LastroError):
            LB.rows_of(bad)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_scale_is_the_smallest_power_of_two_that_holds_the_block(fmt):
    q = R.QMAX[fmt]
    for a, want in ((0.0, 2.0 ** -126), (q, 1.0), (np.nextafter(q, 1e9), 2.0), (q / 2, 0.5), (q * 2.0 ** 30, 2.0 ** 30)):
        assert R.scale_for(float(a), fmt) == want
    assert np.isnan(R.scale_for(float("inf"), fmt))


def test_e4m3_grid_matches_the_hardware_type():
    torch = pytest.importorskip("torch")
    x = torch.cat([torch.linspace(-448, 448, 4001), torch.linspace(-0.05, 0.05, 4001)]).double()
    assert np.array_equal(R.quantise(x.numpy(), "e4m3"), x.to(torch.float8_e4m3fn).double().numpy())


def test_a_block_moved_to_a_smaller_scale_keeps_its_values():
    rng = np.random.default_rng(0)
    for fmt in R.QMAX:
        s = R.Side(64, fmt)
        s.append(rng.standard_normal((40, 64)) * 5)
        keep = np.arange(3, 33, 2)
        assert np.abs(s.gather(keep).values() - s.values()[keep]).max() <= 2.0 ** -4 * np.abs(s.values()).max()
        again = s.gather(np.arange(16))
        assert np.array_equal(again.values(), s.values()[:16])
