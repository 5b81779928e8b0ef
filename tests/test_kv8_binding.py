"""The 8-bit KV cache's Python binding without a GPU: what it sees of rows and tensors before a call is made."""
import pytest

import lastro_b200 as LB

torch = pytest.importorskip("torch")


class NoCall:
    """a context that no call may reach"""
    h = None

    def check(self, rc):
        raise AssertionError(f"the call was made ({rc})")


def refusal(f, *a, **kw):
    with pytest.raises(LB.LastroError) as e:
        f(*a, **kw)
    assert e.value.code == LB.E_ARG
    return str(e.value)


def test_rows_keep_their_heads_and_size():
    t = torch.zeros(5, 3, 64)
    same, fewer, smaller = (LB.rows_of(x).shape for x in (t.bfloat16(), t[:, :2], t[:, :, :32]))
    assert LB.rows_of(t).shape == same and len({same, fewer, smaller, LB.rows_of(torch.zeros(5, 3, 128)).shape}) == 4
    assert LB.Rows().shape == 0  # rows given as an address say nothing


def test_rows_of_another_shape_do_not_reach_the_call():
    c = LB.Kv8Cache(NoCall(), "e4m3", 2, 2, 64, 4, 2, 0, 0, 0, 0, 0)
    k = LB.rows_of(torch.zeros(2, 2, 64))  # right but for being on the host
    for rows in (k, LB.rows_of(torch.zeros(2, 1, 64)), LB.rows_of(torch.zeros(2, 2, 32))):
        assert "kv8_append" in refusal(c.append, 16, 16, 1, rows, rows, 32)
        assert "kv8_attend" in refusal(c.attend, 16, 16, 1, 2, rows, 1.0, rows, 16, 1)


def test_tensors_on_the_host_do_not_reach_the_call():
    c = LB.Kv8Cache(NoCall(), "int8", 2, 2, 64, 4, 2, 0, 0, 0, 0, 0)
    r, lens, mass = LB.Rows(), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64)
    assert "lens" in refusal(c.append, lens, 16, 1, r, r, 32)
    assert "mass_in" in refusal(c.attend, 16, 16, 1, 2, r, 1.0, r, 16, 1, mass_in=mass, mass_stride=64)
    assert "workspace" in refusal(c.attend, 16, 16, 1, 2, r, 1.0, r, torch.zeros(1, dtype=torch.uint8), 1)
    assert "kept" in refusal(c.evict, c, 16, 4, 1, 16, 64, torch.zeros(2, 2, 4, dtype=torch.int32), 32)
    assert "k_out" in refusal(c.read, 16, 16, 1, torch.zeros(2, 1, 2, 64), None, "f32")
    for i, t in enumerate((torch.zeros(4 * 2 * 64 * 64, dtype=torch.uint8), torch.zeros(4 * 2 * 4))):
        a = [0] * 5
        a[2 * i] = t
        assert "cache" in refusal(LB.Kv8Cache, NoCall(), "int8", 2, 2, 64, 4, 2, *a)
