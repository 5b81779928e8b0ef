"""8-bit KV cache on the GPU (lastro_kv8_append / attend / evict / read) against the plain 64-bit form (kv8_ref)."""
import math

import numpy as np
import pytest

import kv8_ref as R
import lastro_b200 as LB

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ctx():
    c = LB.Context(0, LB.LEGACY_STREAM)
    yield c
    c.close()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Gpu:
    """A cache whose buffers hold garbage (NaN codes, NaN scales, page numbers outside the pool) wherever nothing was
    written, its pages taken from the pool in random order."""

    def __init__(self, ctx, fmt, n_seqs, kv, d, max_pages, seed=0, num_pages=None):
        self.num_pages = num_pages or n_seqs * max_pages + 3
        self.fmt, self.kv, self.d, self.n_seqs = fmt, kv, d, n_seqs
        self.k, self.v = (torch.full((self.num_pages, kv, R.PAGE, d), 0x7f, dtype=torch.uint8, device="cuda") for _ in "kv")
        self.ks, self.vs = (torch.full((self.num_pages, kv, R.PAGE // R.BLOCK), math.nan, device="cuda") for _ in "kv")
        perm = np.random.default_rng(seed).permutation(self.num_pages)[:n_seqs * max_pages]
        self.table = ints(perm.reshape(n_seqs, max_pages).tolist())
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.c = LB.Kv8Cache(ctx, fmt, n_seqs, kv, d, self.num_pages, max_pages, self.k, self.v, self.ks, self.vs,
                             self.table, self.status)

    def append(self, lens, k_rows, v_rows, **kw):
        """k_rows, v_rows: per sequence [n_b, kv, d]; returns the new lengths"""
        off = np.concatenate([[0], np.cumsum([r.shape[0] for r in k_rows])])
        k, v = (torch.cat(list(r)) for r in (k_rows, v_rows))
        out = torch.full((self.n_seqs,), -7, dtype=torch.int32, device="cuda")
        self.c.append(ints(lens), ints(off.tolist()), max(1, max(r.shape[0] for r in k_rows)), LB.rows_of(k), LB.rows_of(v),
                      out, **kw)
        return out

    def attend(self, lens, q_rows, scale, mass_in=None, mass=False, stride=None, out=None):
        off = np.concatenate([[0], np.cumsum([r.shape[0] for r in q_rows])])
        q = torch.cat(list(q_rows))
        heads, most = q.shape[1], max(1, max(r.shape[0] for r in q_rows))
        out = torch.full_like(q, math.nan) if out is None else out
        stride = stride or max(1, int(max(lens)))
        m = torch.full((self.n_seqs, self.kv, stride), -5.0, device="cuda") if mass else None
        n = self.c.attend_workspace(heads, most, mass)
        work = torch.full((n,), 0xff, dtype=torch.uint8, device="cuda")
        self.c.attend(ints(lens), ints(off.tolist()), most, heads, LB.rows_of(q), scale, LB.rows_of(out), work, n,
                      mass_in=mass_in, mass_out=m, mass_stride=stride if mass else 0)
        return out, m

    def values(self, lens, n=None, dtype="f32"):
        n = n or max(1, int(max(lens)))
        k, v = (torch.full((self.n_seqs, n, self.kv, self.d), math.nan, dtype=DT[dtype], device="cuda") for _ in "kv")
        self.c.read(ints(lens), ints([0] * self.n_seqs), n, k, v, dtype)
        return k.double().cpu().numpy(), v.double().cpu().numpy()


def rows(rng, n, heads, d, dtype, scale=1.0):
    x = rng.standard_normal((n, heads, d)) * scale * np.exp(0.5 * rng.standard_normal(d))
    return torch.tensor(x, dtype=torch.float32).to(DT[dtype]).cuda()


def f64(t):
    return t.double().cpu().numpy()


def same_values(gpu, ref, lens):
    k, v = gpu.values(lens)
    for b, n in enumerate(lens):
        for h in range(ref.kv_heads):
            for got, w in ((k, "k"), (v, "v")):
                want = ref.side[b][h][w].values()
                assert want.shape[0] == n
                assert np.array_equal(got[b, :n, h], want, equal_nan=True), (b, h, w)
                assert not got[b, n:, h].any()


def filled(ctx, fmt, kv, d, lens, dtype="bf16", seed=0, max_pages=None, scale=1.0):
    """a GPU cache and its plain form holding the same random rows"""
    rng = np.random.default_rng(seed)
    max_pages = max_pages or max(1, -(-(max(lens) + 40) // R.PAGE))
    gpu, ref = Gpu(ctx, fmt, len(lens), kv, d, max_pages, seed), R.Cache(len(lens), kv, d, fmt)
    k, v = ([rows(rng, n, kv, d, dtype, scale) for n in lens] for _ in "kv")
    gpu.append([0] * len(lens), k, v)
    for b in range(len(lens)):
        ref.append(b, f64(k[b]), f64(v[b]))
    return gpu, ref, rng


# ---- append -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt,kv,d,dtype", [("e4m3", 2, 64, "bf16"), ("int8", 3, 64, "f32"), ("e4m3", 1, 128, "f32"),
                                            ("int8", 2, 128, "bf16")])
def test_append_in_steps_matches_the_plain_cache(ctx, fmt, kv, d, dtype):
    """lengths on and around block and page edges, no rows for some sequences, scales that grow from step to step"""
    rng = np.random.default_rng(1)
    lens = [0, 0, 0, 0, 0, 0]
    gpu, ref = Gpu(ctx, fmt, 6, kv, d, 4), R.Cache(6, kv, d, fmt)
    for step, news in enumerate(([0, 1, 15, 16, 17, 65], [1, 1, 1, 1, 1, 0], [3, 63, 2, 33, 1, 100], [1, 0, 40, 1, 15, 16],
                                 [1, 1, 1, 1, 1, 1])):
        k, v = ([rows(rng, n, kv, d, dtype, 2.0 ** (step - 1)) for n in news] for _ in "kv")
        out = gpu.append(lens, k, v)
        for b in range(6):
            ref.append(b, f64(k[b]), f64(v[b]))
        lens = [n + m for n, m in zip(lens, news)]
        assert out.tolist() == lens
        same_values(gpu, ref, lens)
    assert gpu.status.item() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_takes_strided_and_unaligned_rows(ctx, fmt, dtype):
    rng = np.random.default_rng(2)
    kv, d, n = 2, 64, 21
    x = rows(rng, n, 3 * kv, d, dtype)
    fused = (x[:, kv:2 * kv], x[:, 2 * kv:])  # slices of one projection row
    heads_first = tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in fused)
    flat = torch.zeros(2, n * kv * d + 8, dtype=DT[dtype], device="cuda")
    odd = tuple(flat[i, 1:1 + n * kv * d].view(n, kv, d).copy_(t) for i, t in enumerate(fused))  # not 16-byte aligned
    broadcast = tuple(t[:, :1].expand(n, kv, d) for t in fused)  # one head's rows given to every head
    one_row = tuple(t[:1].expand(n, kv, d) for t in fused)
    for k, v in (fused, heads_first, odd, broadcast, one_row):
        gpu, ref = Gpu(ctx, fmt, 1, kv, d, 1), R.Cache(1, kv, d, fmt)
        out = torch.zeros(1, dtype=torch.int32, device="cuda")
        gpu.c.append(ints([0]), ints([0, n]), n, LB.rows_of(k), LB.rows_of(v), out)
        ref.append(0, f64(k), f64(v))
        same_values(gpu, ref, [n])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_of_extreme_values(ctx, fmt):
    """zeros, subnormals, the largest finite values, and values that are not finite: their block reads as NaN, stays so,
    and no other block does"""
    d, kv = 64, 1
    base = torch.randn(48, kv, d, generator=torch.Generator().manual_seed(3))
    for fill in (0.0, 1e-45, 1e-39, 1.2e-38, 3e38, -3.2e38):
        x = base.clone()
        x[20:24] = fill
        x[32:48] = fill
        gpu, ref = Gpu(ctx, fmt, 1, kv, d, 1), R.Cache(1, kv, d, fmt)
        gpu.append([0], [x.cuda()], [x.flip(0).cuda()])
        ref.append(0, f64(x), f64(x.flip(0)))
        same_values(gpu, ref, [48])
    for bad in (math.nan, math.inf, -math.inf):
        x = base.clone()
        x[17, 0, 63] = bad
        gpu, ref = Gpu(ctx, fmt, 1, kv, d, 2), R.Cache(1, kv, d, fmt)
        for lo, hi in ((0, 20), (20, 48)):  # the block is added to after it turned NaN
            gpu.append([lo], [x[lo:hi].cuda()], [base[lo:hi].cuda()])
            ref.append(0, f64(x[lo:hi]), f64(base[lo:hi]))
        assert np.isnan(ref.side[0][0]["k"].values()[16:32]).all()
        same_values(gpu, ref, [48])


def test_append_starts_the_mass_of_new_slots_at_zero(ctx):
    gpu, _, rng = filled(ctx, "e4m3", 2, 64, [5, 0, 17])
    mass = torch.ones(3, 2, 40, device="cuda")
    gpu.append([5, 0, 17], *(([rows(rng, n, 2, 64, "bf16") for n in (2, 0, 20)]) for _ in "kv"), mass=mass, mass_stride=40)
    want = torch.ones(3, 2, 40)
    want[0, :, 5:7] = 0
    want[2, :, 17:37] = 0
    assert torch.equal(mass.cpu(), want)


def test_read_gives_bf16_exactly_and_any_range(ctx):
    for fmt in R.QMAX:
        gpu, ref, _ = filled(ctx, fmt, 2, 128, [70, 3])
        k32, _ = gpu.values([70, 3])
        k16, _ = gpu.values([70, 3], dtype="bf16")
        assert np.array_equal(k16, k32)
        k = torch.full((2, 9, 2, 128), 7.0, device="cuda")
        gpu.c.read(ints([70, 3]), ints([66, 1]), 9, k, None, "f32")
        want = np.zeros((2, 9, 2, 128))
        want[0, :4], want[1, :2] = k32[0, 66:70], k32[1, 1:3]
        assert np.array_equal(f64(k), want)


# ---- attention --------------------------------------------------------------------------------------------------------
# Tolerances, from the arithmetic.  A score is a sum of d products accumulated in f32: its error is at most
# d * 2^-23 * (sum |q_j k_j| * scale) =: e (a unit in the last place per addition), f32 rows add their two-term split,
# 2^-21 of the same sum.  Weights then carry a relative error of at most 2e + 2^-20 (both the weight and the sum it is
# divided by; the exponential's own error and the sums' rounding are in the second term), outputs that times max |v|.
# bf16 outputs add 2^-8 of themselves (half a unit of an 8-bit significand), and 2^-11 of max |v| for weights rounded to 11 bits.
def bounds(dtype, d, big, vmax):
    e = (d * 2.0 ** -23 + 2.0 ** -21) * big
    w = 2 * e + 2.0 ** -20
    return w, w * vmax + (2.0 ** -11 * vmax if dtype == "bf16" else 0.0)


def check_attend(gpu, ref, rng, lens, news, heads, dtype, with_mass=True, qscale=1.0, layout=None, stride=None):
    d, kv = gpu.d, gpu.kv
    scale = d ** -0.5
    q = [rows(rng, n, heads, d, dtype, qscale) for n in news]
    if layout:
        q = layout(q)
    stride = stride or max(1, max(lens))
    mass_in = torch.rand(len(lens), kv, stride, generator=torch.Generator().manual_seed(9)).cuda() if with_mass else None
    out, mass = gpu.attend(lens, q, scale, mass_in, with_mass, stride)
    out, at = f64(out), 0
    for b, (n, m) in enumerate(zip(lens, news)):
        want, wm, big = ref.attend(b, f64(q[b]), scale)
        vmax = max((np.abs(ref.side[b][h]["v"].values()).max(initial=0.0) for h in range(kv)))
        rel, tol = bounds(dtype, d, big, vmax)
        err = np.abs(out[at:at + m] - want)
        assert (err <= tol + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0.0)).all(), (b, err.max(initial=0), tol)
        at += m
        if with_mass:
            base = f64(mass_in[b, :, :n])
            got = f64(mass[b])
            assert (np.abs(got[:, :n] - (base + wm)) <= rel * wm + 2.0 ** -22 * (base + wm)).all(), b
            assert (got[:, n:] == -5.0).all()
    assert gpu.status.item() == 0


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 129, 500]


@pytest.mark.parametrize("fmt,kv,group,d,dtype", [
    ("e4m3", 2, 3, 64, "bf16"), ("int8", 2, 3, 64, "f32"), ("e4m3", 1, 1, 64, "f32"), ("int8", 1, 8, 64, "bf16"),
    ("e4m3", 3, 4, 128, "bf16"), ("int8", 1, 2, 128, "bf16"), ("e4m3", 1, 20, 128, "f32"), ("int8", 2, 1, 128, "f32")])
def test_single_token_attention(ctx, fmt, kv, group, d, dtype):
    """one query for each sequence, lengths around every edge; a sequence of length 0 sees nothing and gives zeros"""
    gpu, ref, rng = filled(ctx, fmt, kv, d, LENS)
    check_attend(gpu, ref, rng, LENS, [1] * len(LENS), kv * group, dtype)
    check_attend(gpu, ref, rng, LENS, [1] * len(LENS), kv * group, dtype, with_mass=False)


@pytest.mark.parametrize("fmt,kv,group,d,dtype,most", [
    ("e4m3", 2, 3, 64, "bf16", 32), ("int8", 1, 4, 64, "f32", 7), ("e4m3", 1, 2, 128, "f32", 33), ("int8", 2, 4, 128, "bf16", 17),
    ("int8", 1, 1, 64, "bf16", 150), ("e4m3", 1, 20, 64, "bf16", 11)])
def test_multi_position_attention_is_causal(ctx, fmt, kv, group, d, dtype, most):
    """ragged numbers of queries, none for some sequences, more queries than slots (the first see nothing)"""
    lens = [0, 1, 40, 64, 65, 200, 161]
    news = [min(most, n) for n in (3, 4, 0, 64, 17, 150, 16)]
    gpu, ref, rng = filled(ctx, fmt, kv, d, lens)
    check_attend(gpu, ref, rng, lens, news, kv * group, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_over_a_long_context(ctx, dtype):
    """a context split over many CTAs beside short ones"""
    lens = [9001, 1, 130]
    gpu, ref, rng = filled(ctx, "e4m3", 2, 64, lens)
    check_attend(gpu, ref, rng, lens, [1, 1, 1], 6, dtype)
    check_attend(gpu, ref, rng, lens, [5, 1, 2], 6, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_with_peaked_and_flat_weights(ctx, dtype):
    """scores spread over hundreds (one slot takes all) and nearly equal ones"""
    lens = [300, 77]
    for scale, q in ((8.0, 8.0), (1e-3, 1.0)):
        gpu, ref, rng = filled(ctx, "int8", 1, 64, lens, scale=scale)
        check_attend(gpu, ref, rng, lens, [2, 1], 2, dtype, qscale=q)


def test_query_and_output_strides(ctx):
    lens, kv, d, heads = [100, 33], 2, 64, 4
    gpu, ref, rng = filled(ctx, "e4m3", kv, d, lens)
    for dtype in ("bf16", "f32"):
        q = rows(rng, 3, heads, d, dtype)
        plain, _ = gpu.attend(lens, [q[:2], q[2:]], 0.125)
        wide = torch.zeros(3, 3 * heads, d, dtype=DT[dtype], device="cuda")
        wide[:, heads:2 * heads] = q
        hf = q.transpose(0, 1).contiguous().transpose(0, 1)
        odd = torch.zeros(3 * heads * d + 1, dtype=DT[dtype], device="cuda")[1:].view(3, heads, d).copy_(q)
        work = torch.empty(gpu.c.attend_workspace(heads, 2, False), dtype=torch.uint8, device="cuda")
        for src in (wide[:, heads:2 * heads], hf, odd, q[:, :1].expand(3, heads, d)):
            for dst in (torch.zeros_like(wide)[:, :heads], torch.zeros_like(hf), torch.zeros_like(odd)):
                gpu.c.attend(ints(lens), ints([0, 2, 3]), 2, heads, LB.rows_of(src), 0.125, LB.rows_of(dst), work, work.numel())
                if src.stride(1) == 0:
                    assert torch.equal(dst[:, 0], plain[:, 0])
                else:
                    assert torch.equal(dst, plain)


def test_rows_that_are_not_finite_stay_apart(ctx):
    """a query with NaN or infinity gives NaN and touches no other query's output"""
    gpu, ref, rng = filled(ctx, "e4m3", 1, 64, [90, 20])
    for dtype in ("bf16", "f32"):
        for bad in (math.nan, math.inf):
            q = rows(rng, 6, 3, 64, dtype)
            plain, _ = gpu.attend([90, 20], [q[:4], q[4:]], 0.125)
            q[2, 1, 5] = bad
            out, _ = gpu.attend([90, 20], [q[:4], q[4:]], 0.125)
            assert out[2, 1].isnan().all()
            out[2, 1] = plain[2, 1]
            assert torch.equal(out, plain)


def test_a_nan_block_reaches_only_the_queries_that_see_it(ctx):
    """the same cache with and without an infinity in slot 63: queries that see its block 48..63 give NaN, those of a
    length that ends before it give the same bits"""
    for fmt in R.QMAX:
        rng = np.random.default_rng(5)
        q = rows(rng, 8, 2, 64, "f32")
        k, v = (rows(rng, 32, 1, 64, "f32") for _ in "kv")
        clean, _, _ = filled(ctx, fmt, 1, 64, [32])
        clean.append([32], [k], [v])
        for which in (0, 1):
            x = [k.clone(), v.clone()]
            x[which][31, 0, 7] = math.inf
            bad, _, _ = filled(ctx, fmt, 1, 64, [32])
            bad.append([32], [x[0]], [x[1]])
            assert not clean.attend([64], [q], 0.125)[0].isnan().any()
            assert bad.attend([64], [q], 0.125)[0].isnan().all()
            assert torch.equal(bad.attend([48], [q], 0.125)[0], clean.attend([48], [q], 0.125)[0])
            # queries 0..3 (slots 44..47) end before the block, 4..7 (slots 48..51) see it
            part, _ = bad.attend([52], [q], 0.125)
            assert torch.equal(part[:4], clean.attend([52], [q], 0.125)[0][:4]) and part[4:].isnan().all()


@pytest.mark.parametrize("scale", [-1.0, -math.inf, math.inf, 0.0, -3e38, 1e-40, math.nan])
@pytest.mark.parametrize("group,new", [(2, 1), (5, 3)])
def test_what_was_never_written_does_not_matter(ctx, scale, group, new):
    """any scale and any code in blocks and slots past a sequence's length"""
    lens = [3, 17, 40, 64, 81]
    for code in (0x7f, 0xff, 0x80, 0x00):
        for fmt in R.QMAX:
            gpu, rng = Gpu(ctx, fmt, 5, 1, 64, 2), np.random.default_rng(6)
            for t in (gpu.ks, gpu.vs):
                t.fill_(scale)
            for t in (gpu.k, gpu.v):
                t.fill_(code)
            ref = R.Cache(5, 1, 64, fmt)
            k, v = ([rows(rng, n, 1, 64, "f32") for n in lens] for _ in "kv")
            gpu.append([0] * 5, k, v)
            for b in range(5):
                ref.append(b, f64(k[b]), f64(v[b]))
            check_attend(gpu, ref, rng, lens, [new] * 5, group, "f32")
            same_values(gpu, ref, lens)


def test_mass_accumulates_in_place_and_over_steps(ctx):
    lens = [65, 20]
    gpu, ref, rng = filled(ctx, "int8", 2, 64, lens)
    q = [rows(rng, 2, 4, 64, "f32") for _ in lens]
    _, one = gpu.attend(lens, q, 0.125, mass=True)
    work = torch.empty(gpu.c.attend_workspace(4, 2, True), dtype=torch.uint8, device="cuda")
    out = torch.empty(4, 4, 64, device="cuda")
    both = one.clone()
    gpu.c.attend(ints(lens), ints([0, 2, 4]), 2, 4, LB.rows_of(torch.cat(q)), 0.125, LB.rows_of(out), work, work.numel(),
                 mass_in=both, mass_out=both, mass_stride=65)
    for b, n in enumerate(lens):
        assert torch.equal(both[b, :, :n], one[b, :, :n] + one[b, :, :n])
        assert abs(float(one[b, :, :n].double().sum()) - 2 * 4) < 1e-4  # every query and head hands out 1
        assert torch.equal(both[b, :, n:], one[b, :, n:])


def test_the_same_call_gives_the_same_bits(ctx):
    lens = [3000, 700, 64, 1]
    gpu, _, rng = filled(ctx, "e4m3", 2, 128, lens)
    q = [rows(rng, 1, 8, 128, "bf16") for _ in lens]
    first = gpu.attend(lens, q, 0.1, mass=True)
    for _ in range(5):
        again = gpu.attend(lens, q, 0.1, mass=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_pools_beyond_two_gigabytes(ctx):
    """pages whose codes start past 2^32 bytes"""
    kv, d, pages = 8, 128, 70000
    gpu = Gpu.__new__(Gpu)
    gpu.fmt, gpu.kv, gpu.d, gpu.n_seqs, gpu.num_pages = "e4m3", kv, d, 1, pages
    gpu.k, gpu.v = (torch.empty(pages * kv * R.PAGE * d, dtype=torch.uint8, device="cuda") for _ in "kv")
    gpu.ks, gpu.vs = (torch.empty(pages * kv * 4, device="cuda") for _ in "kv")
    gpu.table, gpu.status = ints([[pages - 1, 0, pages - 2]]), torch.zeros(1, dtype=torch.int32, device="cuda")
    gpu.c = LB.Kv8Cache(ctx, "e4m3", 1, kv, d, pages, 3, gpu.k, gpu.v, gpu.ks, gpu.vs, gpu.table, gpu.status)
    ref, rng = R.Cache(1, kv, d, "e4m3"), np.random.default_rng(4)
    k, v = (rows(rng, 150, kv, d, "bf16") for _ in "kv")
    gpu.append([0], [k], [v])
    ref.append(0, f64(k), f64(v))
    same_values(gpu, ref, [150])
    check_attend(gpu, ref, rng, [150], [1], 16, "bf16")


def test_more_sequences_than_a_block_has_threads(ctx):
    """the list of work is found in several steps; sequences without queries or slots among them"""
    rng = np.random.default_rng(12)
    lens = rng.integers(0, 40, 700).tolist()
    lens[255], lens[256], lens[511], lens[512] = 64, 1, 0, 130
    news = [min(n, int(m)) for n, m in zip(lens, rng.integers(0, 3, 700))]
    gpu, ref, rng = filled(ctx, "int8", 1, 64, lens)
    check_attend(gpu, ref, rng, lens, news, 2, "f32")  # few rows
    check_attend(gpu, ref, rng, lens, [4 * n for n in news], 5, "bf16")  # many rows, also more queries than slots


@pytest.mark.parametrize("kv,group,d,dtype,new", [(1, 4, 128, "bf16", 1), (1, 2, 64, "f32", 3), (1, 9, 64, "bf16", 1), (1, 12, 128, "bf16", 3)])
def test_one_long_sequence_in_many_parts(ctx, kv, group, d, dtype, new):
    """more parts of one unit than a warp has lanes"""
    lens = [40001]
    gpu, ref, rng = filled(ctx, "e4m3", kv, d, lens)
    check_attend(gpu, ref, rng, lens, [new], kv * group, dtype)
    check_attend(gpu, ref, rng, lens, [new], kv * group, dtype, with_mass=False)


def test_weights_rebuilt_from_k_when_scores_are_not_kept(ctx):
    """a page table so long that the scores of every slot it could name would pass the workspace's bound"""
    kv, d, heads, pages = 8, 64, 64, 70000
    gpu, ref, rng = filled(ctx, "e4m3", kv, d, [300])
    scores = lambda: gpu.c.attend_workspace(heads, 1, True) - gpu.c.attend_workspace(heads, 1, False)  # noqa: E731
    assert scores() > kv * 300 * heads // kv * 4
    wide = torch.full((1, pages), 2 ** 30, dtype=torch.int32, device="cuda")
    wide[:, :gpu.table.shape[1]] = gpu.table
    gpu.c = LB.Kv8Cache(ctx, "e4m3", 1, kv, d, gpu.num_pages, pages, gpu.k, gpu.v, gpu.ks, gpu.vs, wide, gpu.status)
    assert scores() < 2 ** 12
    check_attend(gpu, ref, rng, [300], [1], heads, "f32")
    check_attend(gpu, ref, rng, [300], [1], heads, "bf16", stride=301)


@pytest.mark.parametrize("group,new", [(3, 1), (5, 4)])
def test_scales_of_either_sign_and_zero(ctx, group, new):
    lens = [100, 33]
    gpu, ref, rng = filled(ctx, "int8", 1, 64, lens)
    q = [rows(rng, new, group, 64, "f32") for _ in lens]
    for scale in (-0.125, 0.0, -0.0, 1e-30):
        out, mass = gpu.attend(lens, q, scale, mass=True, stride=101)
        for b, n in enumerate(lens):
            want, wm, big = ref.attend(b, f64(q[b]), scale)
            vmax = max(np.abs(ref.side[b][0]["v"].values()).max(), 0.0)
            rel, tol = bounds("f32", 64, big, vmax)
            assert (np.abs(f64(out[b * new:(b + 1) * new]) - want) <= tol).all()
            assert (np.abs(f64(mass[b, :, :n]) - wm) <= rel * wm + 2.0 ** -22 * wm).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("group,new", [(2, 1), (6, 3)])
def test_values_of_very_different_size(ctx, dtype, group, new):
    """V blocks from 1e-30 to 1e30, the large ones far out of the attention, zeros where it looks: weights stay in range"""
    n, d = 128, 64
    rng = np.random.default_rng(8)
    k = np.zeros((n, 1, d))
    v = rng.standard_normal((n, 1, d))
    k[:, 0, 0] = np.repeat([0.0, -300.0, 1.0, -300.0, 2.0, 0.5, -300.0, 3.0], 16)
    v *= np.repeat([1.0, 1e30, 1e-4, 1e38, 1e-30, 2.0, 1e20, 0.0], 16)[:, None, None]
    k, v = (torch.tensor(x, dtype=torch.float32) for x in (k, v))
    gpu, ref = Gpu(ctx, "e4m3", 1, 1, d, 2), R.Cache(1, 1, d, "e4m3")
    gpu.append([0], [k.cuda()], [v.cuda()])
    ref.append(0, f64(k), f64(v))
    q = torch.zeros(new, group, d)
    q[:, :, 0] = 1.0
    q[:, :, 1:] = torch.tensor(rng.standard_normal((new, group, d - 1)))
    q = q.to(DT[dtype]).cuda()
    out, mass = gpu.attend([n], [q], 1.0, mass=True)
    want, wm, big = ref.attend(0, f64(q), 1.0)
    # what each query sees: the far blocks' weights are e^-300 = 0 against values of at most 1e38; the blocks near 1 rule
    rel, tol = bounds(dtype, d, big, 10.0)
    assert (np.abs(f64(out) - want) <= tol + 2.0 ** -8 * np.abs(want)).all()
    assert (np.abs(f64(mass[0]) - wm) <= rel * wm + 1e-12).all()


# ---- eviction ---------------------------------------------------------------------------------------------------------
def check_evict(ctx, gpu, ref, lens, mass, budget, recent, stride_out=None):
    n, kv, d = len(lens), gpu.kv, gpu.d
    dst = Gpu(ctx, gpu.fmt, n, kv, d, -(-budget // R.PAGE), seed=11)
    kept = torch.full((n, kv, budget), -9, dtype=torch.int32, device="cuda")
    out = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    so = stride_out or budget
    mo = torch.full((n, kv, so), -5.0, device="cuda") if mass is not None else None
    gpu.c.evict(dst.c, ints(lens), budget, recent, mass, mass.shape[2] if mass is not None else 0, kept, out, mo, so if mo is not None else 0)
    assert out.tolist() == [min(x, budget) for x in lens]
    kept = kept.cpu().numpy()
    for b, x in enumerate(lens):
        m = f64(mass[b, :, :x]) if mass is not None else np.zeros((kv, x))
        for h, want in enumerate(ref.evict(b, m, budget, recent)):
            assert np.array_equal(kept[b, h, :len(want)], want), (b, h)
            assert (kept[b, h, len(want):] == -1).all()
            if mass is not None:
                assert np.array_equal(f64(mo[b, h, :len(want)]), m[h, want], equal_nan=True)
                assert (mo[b, h, len(want):] == -5.0).all()
    same_values(dst, ref, [min(x, budget) for x in lens])
    assert dst.status.item() == 0 and gpu.status.item() == 0
    return dst


@pytest.mark.parametrize("fmt,kv,d,budget,recent", [("e4m3", 2, 64, 33, 5), ("int8", 1, 128, 64, 0), ("int8", 3, 64, 100, 100),
                                                    ("e4m3", 1, 128, 1, 0), ("e4m3", 1, 64, 17, 16)])
def test_eviction_keeps_the_heaviest_and_the_latest(ctx, fmt, kv, d, budget, recent):
    """lengths below, at and above the budget; masses with many ties"""
    lens = [0, 1, 16, 33, 34, 100, 101, 300]
    gpu, ref, rng = filled(ctx, fmt, kv, d, lens)
    mass = torch.tensor(rng.integers(0, 6, (len(lens), kv, 301)) / 4.0, dtype=torch.float32).cuda()
    check_evict(ctx, gpu, ref, lens, mass, budget, recent, stride_out=budget + 3)


def test_eviction_by_unusual_masses(ctx):
    """negative values, both zeros, infinities and NaN"""
    lens = [200]
    for seed in range(3):
        gpu, ref, rng = filled(ctx, "e4m3", 1, 64, lens, seed=seed)
        mass = torch.tensor(rng.choice([0.0, -0.0, 1.0, -1.0, 1e-40, -1e-40, 3e38, math.inf, -math.inf, math.nan], (1, 1, 200)),
                            dtype=torch.float32).cuda()
        check_evict(ctx, gpu, ref, lens, mass, 50 + 40 * seed, 10)


def test_eviction_of_equal_masses_and_without_mass(ctx):
    lens = [2500, 40]
    gpu, ref, _ = filled(ctx, "int8", 1, 64, lens)
    check_evict(ctx, gpu, ref, lens, torch.ones(2, 1, 2500, device="cuda"), 1111, 111)
    gpu, ref, _ = filled(ctx, "int8", 1, 64, lens)
    check_evict(ctx, gpu, ref, lens, None, 1111, 1111)  # the latest slots only


@pytest.mark.parametrize("length,budget,recent", [(40000, 5000, 100), (131072, 70001, 1), (8193, 8192, 0)])
def test_eviction_from_long_contexts(ctx, length, budget, recent):
    """the selection alone, on sequences longer than one CTA's pass"""
    rng = np.random.default_rng(7)
    mass = torch.tensor(np.floor(np.exp(rng.standard_normal((1, 2, length))) * 16) / 16, dtype=torch.float32).cuda()
    gpu = Gpu(ctx, "int8", 1, 2, 64, -(-length // R.PAGE))
    gpu.k.random_(0, 256), gpu.v.random_(0, 256), gpu.ks.fill_(0.5), gpu.vs.fill_(2.0)
    gpu.k[gpu.k == 128], gpu.v[gpu.v == 128] = 0, 0
    dst = Gpu(ctx, "int8", 1, 2, 64, -(-budget // R.PAGE), seed=3)
    kept = torch.zeros(1, 2, budget, dtype=torch.int32, device="cuda")
    out = torch.zeros(1, dtype=torch.int32, device="cuda")
    gpu.c.evict(dst.c, ints([length]), budget, recent, mass, length, kept, out)
    cand = length - recent
    k, _ = gpu.values([length])
    got, _ = dst.values([budget])
    for h in range(2):
        order = torch.sort(mass[0, h, :cand], descending=True, stable=True).indices[:budget - recent].sort().values
        want = torch.cat([order.cpu(), torch.arange(cand, length)])
        assert torch.equal(kept[0, h].cpu().long(), want)
        assert np.array_equal(got[0, :, h], k[0, want.numpy(), h])


@pytest.mark.parametrize("length,shift", [(150001, 0), (200000, 1), (30000, 1), (3000, 3)])
def test_eviction_with_masses_at_any_address(ctx, length, shift):
    """mass rows off 16-byte boundaries, and more slots than a cluster's shared memory holds the keys of"""
    rng = np.random.default_rng(length)
    flat = torch.tensor(rng.standard_normal(length + shift), dtype=torch.float32).cuda()
    mass = flat[shift:].view(1, 1, length)
    gpu = Gpu(ctx, "e4m3", 1, 1, 64, -(-length // R.PAGE))
    gpu.k.random_(0, 127), gpu.v.random_(0, 127), gpu.ks.fill_(1.0), gpu.vs.fill_(0.25)
    budget, recent = length // 3, 77
    dst = Gpu(ctx, "e4m3", 1, 1, 64, -(-budget // R.PAGE), seed=3)
    kept, out = torch.zeros(1, 1, budget, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    mo = torch.zeros(1, 1, budget, device="cuda")
    gpu.c.evict(dst.c, ints([length]), budget, recent, mass, length, kept, out, mo, budget)
    order = torch.sort(mass[0, 0, :length - recent], descending=True, stable=True).indices[:budget - recent].sort().values
    want = torch.cat([order, torch.arange(length - recent, length, device="cuda")])
    assert torch.equal(kept[0, 0].long(), want) and torch.equal(mo[0, 0], mass[0, 0, want])
    k, _ = gpu.values([length])
    got, _ = dst.values([budget])
    assert np.array_equal(got[0, :, 0], k[0, want.cpu().numpy(), 0])


def test_a_bounded_cache_decodes_on(ctx):
    """append, attend and evict in turn, as a decode loop with a budget runs them, each step against the plain form"""
    for fmt, dtype in (("e4m3", "f32"), ("int8", "bf16")):
        kv, d, heads, budget = 2, 64, 6, 48
        lens = [40, 60, 3]
        gpu, ref, rng = filled(ctx, fmt, kv, d, lens, dtype, max_pages=2)
        mass = torch.zeros(3, kv, 128, device="cuda")
        for step in range(12):
            k, v = ([rows(rng, 1, kv, d, dtype) for _ in lens] for _ in "kv")
            out = gpu.append(lens, k, v, mass=mass, mass_stride=128)
            for b in range(3):
                ref.append(b, f64(k[b]), f64(v[b]))
            lens = out.tolist()
            check_attend(gpu, ref, rng, lens, [1, 1, 1], heads, dtype, with_mass=False)
            q = [rows(rng, 1, heads, d, dtype) for _ in lens]
            _, new = gpu.attend(lens, q, 0.125, mass_in=mass, mass=True, stride=128)
            mass = torch.where(torch.arange(128, device="cuda") < ints(lens)[:, None, None], new, mass)
            if max(lens) > 62:
                gpu = check_evict(ctx, gpu, ref, lens, mass, budget, 8, stride_out=budget)
                lens = [min(n, budget) for n in lens]
                wide = Gpu(ctx, fmt, 3, kv, d, 2, seed=step)  # the same pages in a cache with room for more
                for dst, src in ((wide.k, gpu.k), (wide.v, gpu.v), (wide.ks, gpu.ks), (wide.vs, gpu.vs)):
                    dst[:src.shape[0]] = src
                wide.table[:, :1] = gpu.table
                wide.table[:, 1] = ints([6, 7, 8])
                gpu = wide
                mass = torch.zeros(3, kv, 128, device="cuda")


def test_the_bounded_decode_example(ctx):
    """without evictions a bounded cache decodes like a large one; with them it runs on in the same memory"""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "bounded_decode.py")
    spec = importlib.util.spec_from_file_location("bounded_decode", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    for fmt in R.QMAX:
        large, c = ex.decode(3, 150, 256, 64, 16, fmt)
        assert c.evictions == 0
        small, c = ex.decode(3, 150, 96, 64, 16, fmt)
        assert c.evictions == 2 and c.longest == 64 + (150 - 96 - 32) and c.slots == 128
        assert torch.equal(small[:, :96], large[:, :96])
        # after 150 steps of 16 heads the kept slots hold at most the weight handed out since the start
        total = c.mass[0][:, :, :c.longest].double().sum(-1)
        assert (total <= 150 * 2 + 1e-3).all() and (total > 0).all()


# ---- streams, refusals, bad data on the device ------------------------------------------------------------------------
def test_a_context_on_its_own_stream(ctx):
    side = torch.cuda.Stream()
    c2 = LB.Context(0, side.cuda_stream)
    with torch.cuda.stream(side):
        gpu, ref, rng = filled(c2, "e4m3", 2, 64, [100, 7])
        check_attend(gpu, ref, rng, [100, 7], [1, 1], 4, "bf16")
    side.synchronize()
    c2.close()


def test_calls_are_captured_into_a_graph(ctx):
    side = torch.cuda.Stream()
    c2 = LB.Context(0, side.cuda_stream)
    lens = [70, 5]
    with torch.cuda.stream(side):
        gpu, _, rng = filled(c2, "int8", 2, 64, lens)
        q = torch.cat([rows(rng, 1, 4, 64, "bf16") for _ in lens])
        ln, off = ints(lens), ints([0, 1, 2])
        work = torch.zeros(gpu.c.attend_workspace(4, 1, True), dtype=torch.uint8, device="cuda")
        out, mass = torch.zeros_like(q), torch.zeros(2, 2, 70, device="cuda")

        def call():
            gpu.c.attend(ln, off, 1, 4, LB.rows_of(q), 0.125, LB.rows_of(out), work, work.numel(), mass_out=mass, mass_stride=70)

        call()
        want = out.clone(), mass.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call()
        out.zero_(), mass.zero_()
        g.replay()
        side.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(mass, want[1])
    c2.close()


def test_refusals(ctx):
    gpu, _, rng = filled(ctx, "e4m3", 2, 64, [20, 20])
    q = rows(rng, 2, 4, 64, "bf16")
    k = rows(rng, 2, 2, 64, "bf16")
    out, lens, off = torch.zeros_like(q), ints([20, 20]), ints([0, 1, 2])
    n = gpu.c.attend_workspace(4, 1, False)
    work = torch.zeros(n + 16, dtype=torch.uint8, device="cuda")
    lo = torch.zeros(2, dtype=torch.int32, device="cuda")
    kept = torch.zeros(2, 2, 16, dtype=torch.int32, device="cuda")
    mass = torch.zeros(2, 2, 20, device="cuda")
    ro = LB.rows_of

    def cache(**kw):
        a = dict(fmt="e4m3", n_seqs=2, kv_heads=2, head_dim=64, num_pages=gpu.num_pages, max_pages=1, k=gpu.k, v=gpu.v,
                 k_scale=gpu.ks, v_scale=gpu.vs, page_table=gpu.table) | kw
        return LB.Kv8Cache(ctx, *a.values())

    def refused(code, f, *a, **kw):
        with pytest.raises(LB.LastroError) as e:
            f(*a, **kw)
        assert e.value.code == code and "kv8" in str(e.value)

    att = dict(lens=lens, q_off=off, max_new=1, heads=4, q=ro(q), scale=0.1, out=ro(out), workspace=work, workspace_bytes=n)
    for kw in (dict(lens=None), dict(q_off=None), dict(max_new=-1), dict(heads=3), dict(heads=0), dict(scale=math.nan),
               dict(scale=math.inf), dict(workspace=None), dict(workspace_bytes=n - 1), dict(workspace=work.data_ptr() + 1),
               dict(out=ro(out.float())), dict(out=ro(out[:1])), dict(q=LB.Rows()), dict(mass_in=mass, mass_stride=20),
               dict(mass_out=mass, mass_stride=0), dict(max_new=0)):
        refused(LB.E_ARG, gpu.c.attend, **(att | kw))
    app = dict(lens=lens, new_off=off, max_new=1, k=ro(k), v=ro(k), lens_out=lo)
    for kw in (dict(lens=None), dict(new_off=None), dict(lens_out=None), dict(lens_out=lens), dict(max_new=-1),
               dict(k=LB.Rows()), dict(mass=mass, mass_stride=0)):
        refused(LB.E_ARG, gpu.c.append, **(app | kw))
    evi = dict(dst=gpu.c, lens=lens, budget=16, recent=4, mass=mass, mass_stride=20, kept=kept, lens_out=lo)
    for kw in (dict(budget=0), dict(budget=65), dict(recent=17), dict(recent=-1), dict(mass=None), dict(mass_stride=0),
               dict(kept=None), dict(lens_out=lens), dict(lens=None), dict(mass_out=mass, mass_out_stride=20),
               dict(mass_out=torch.zeros(2, 2, 16, device="cuda"), mass_out_stride=15), dict(dst=cache(fmt="int8"))):
        refused(LB.E_ARG, gpu.c.evict, **(evi | kw))
    rd = dict(lens=lens, pos0=lens, n=1, k_out=k, v_out=None, dtype="bf16")
    for kw in (dict(lens=None), dict(n=-1), dict(pos0=None), dict(k_out=k.data_ptr() + 2), dict(dtype="f16")):
        with pytest.raises(LB.LastroError):
            gpu.c.read(**(rd | kw))
    for code, kw in ((LB.E_ARG, dict(n_seqs=0)), (LB.E_ARG, dict(kv_heads=0)), (LB.E_UNSUPPORTED, dict(head_dim=80)),
                     (LB.E_ARG, dict(num_pages=0)), (LB.E_ARG, dict(max_pages=0)), (LB.E_ARG, dict(k=None)),
                     (LB.E_ARG, dict(v_scale=None)), (LB.E_ARG, dict(page_table=None)), (LB.E_ARG, dict(k=gpu.k.data_ptr() + 8)),
                     (LB.E_UNSUPPORTED, dict(max_pages=1 << 25))):
        c = cache(**kw)
        refused(code, c.append, **app)
        refused(code, c.attend, **att)
        refused(code, c.read, **rd)
        refused(code, c.attend_workspace, 4, 1, False)
        refused(code, c.evict, **(evi | dict(dst=gpu.c)))
    gpu.c.attend(**att)  # still usable
    torch.cuda.synchronize()


def test_misaligned_addresses_are_refused(ctx):
    gpu, _, rng = filled(ctx, "e4m3", 1, 64, [20])
    q, k = rows(rng, 1, 2, 64, "f32"), rows(rng, 1, 1, 64, "f32")
    out, lens, off = torch.zeros_like(q), ints([20]), ints([0, 1])
    n = gpu.c.attend_workspace(2, 1, True)
    work, mass = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(1, 1, 64, device="cuda")
    spare, kept = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, 16, dtype=torch.int32, device="cuda")
    odd = lambda t: t.data_ptr() + 2  # noqa: E731
    ro = LB.rows_of
    att = dict(lens=lens, q_off=off, max_new=1, heads=2, q=ro(q), scale=0.1, out=ro(out), workspace=work, workspace_bytes=n,
               mass_in=mass, mass_out=mass, mass_stride=64)
    app = dict(lens=lens, new_off=off, max_new=1, k=ro(k), v=ro(k), lens_out=spare, mass=mass, mass_stride=64)
    evi = dict(dst=gpu.c, lens=lens, budget=16, recent=4, mass=mass, mass_stride=64, kept=kept, lens_out=spare)
    for f, args, names in ((gpu.c.attend, att, ("lens", "q_off", "mass_in", "mass_out")), (gpu.c.append, app, ("lens", "new_off", "lens_out", "mass")),
                           (gpu.c.evict, evi, ("lens", "kept", "lens_out", "mass"))):
        for name in names:
            with pytest.raises(LB.LastroError) as e:
                f(**(args | {name: odd(args[name])}))
            assert e.value.code == LB.E_ARG
    for a in ((odd(lens), lens), (lens, odd(lens))):
        with pytest.raises(LB.LastroError):
            gpu.c.read(*a, 1, k, None, "f32")
    with pytest.raises(LB.LastroError):
        gpu.c.append(**(app | dict(v=ro(k.bfloat16()))))


def test_calls_without_rows(ctx):
    """no query and no new row: lengths and masses are handed on"""
    gpu, _, _ = filled(ctx, "int8", 2, 64, [70, 5])
    n = gpu.c.attend_workspace(6, 0, True)
    work, mass = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.rand(2, 2, 80, device="cuda")
    out = torch.full_like(mass, -5.0)
    r = LB.Rows(work.data_ptr(), LB.DTYPE_F32, 0, 64, 64)
    gpu.c.attend(ints([70, 5]), ints([0, 0, 0]), 0, 6, r, 0.1, r, work, n, mass_in=mass, mass_out=out, mass_stride=80)
    assert torch.equal(out[0, :, :70], mass[0, :, :70]) and torch.equal(out[1, :, :5], mass[1, :, :5])
    assert (out[0, :, 70:] == -5.0).all() and (out[1, :, 5:] == -5.0).all()
    for most in (0, 3, 40):  # room for queries, none there
        n = gpu.c.attend_workspace(6, most, True)
        work = torch.zeros(n, dtype=torch.uint8, device="cuda")
        again = torch.full_like(mass, -5.0)
        gpu.c.attend(ints([70, 5]), ints([0, 0, 0]), most, 6, r, 0.1, r, work, n, mass_in=mass, mass_out=again, mass_stride=80)
        assert torch.equal(again, out)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    gpu.c.append(ints([70, 5]), ints([0, 0, 0]), 0, r, r, lens)
    assert lens.tolist() == [70, 5] and gpu.status.item() == 0
    gpu.c.append(ints([-3, 5]), ints([0, 0, 0]), 0, r, r, lens)
    assert lens.tolist() == [-3, 5] and gpu.status.item() == LB.KV8_BAD_LENGTH


def test_bad_device_data_is_reported_and_skipped(ctx):
    """page numbers outside the pool, lengths and offsets that do not fit: the other sequences' results stand"""
    lens, kv, d, heads = [100, 90, 30], 2, 64, 4
    gpu, ref, rng = filled(ctx, "e4m3", kv, d, lens, max_pages=3)
    q = [rows(rng, 1, heads, d, "f32") for _ in lens]
    good, gm = gpu.attend(lens, q, 0.125, mass=True, stride=192)
    table = gpu.table.clone()
    for page in (-1, gpu.num_pages, 2 ** 31 - 1):
        gpu.table[1, 1] = page
        out, mass = gpu.attend(lens, q, 0.125, mass=True, stride=192)
        assert gpu.status.item() == LB.KV8_BAD_PAGE
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2]) and not out.isnan().any()
        assert torch.equal(mass[0], gm[0]) and torch.equal(mass[2], gm[2])
        gpu.status.zero_()
        new = [rows(rng, n, kv, d, "f32") for n in (1, 1, 1)]
        before = [(t, t.clone()) for t in (gpu.k, gpu.v, gpu.ks, gpu.vs)]
        gpu.append([100, 90, 30], new, new)
        assert gpu.status.item() == LB.KV8_BAD_PAGE
        for t, was in before:
            t.copy_(was)
        gpu.status.zero_()
        gpu.table.copy_(table)
    for bad in ([-1, 90, 30], [193, 90, 30]):
        out, _ = gpu.attend(bad, q, 0.125, stride=192)
        assert gpu.status.item() == LB.KV8_BAD_LENGTH
        assert torch.equal(out[1:], good[1:])
        gpu.status.zero_()
    qq = torch.cat(q)
    out = torch.full_like(qq, 3.0)
    work = torch.zeros(gpu.c.attend_workspace(heads, 1, False), dtype=torch.uint8, device="cuda")
    for off in ([0, 2, 2, 3], [-1, 1, 2, 3], [0, 1, 0, 3], [0, 1, 2, 9]):
        gpu.c.attend(ints(lens), ints(off), 1, heads, LB.rows_of(qq), 0.125, LB.rows_of(out), work, work.numel())
        assert gpu.status.item() == LB.KV8_BAD_OFFSET
        gpu.status.zero_()
    new = rows(rng, 3, kv, d, "f32")
    lo = torch.zeros(3, dtype=torch.int32, device="cuda")
    k0, s0 = gpu.k.clone(), gpu.ks.clone()
    gpu.c.append(ints([192, 90, 30]), ints([0, 1, 1, 1]), 1, LB.rows_of(new), LB.rows_of(new), lo)  # past the page table
    assert gpu.status.item() == LB.KV8_BAD_LENGTH and lo.tolist() == [192, 90, 30]
    assert torch.equal(gpu.k, k0) and torch.equal(gpu.ks.nan_to_num(), s0.nan_to_num())
