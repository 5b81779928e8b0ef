"""8-bit KV cache on the GPU at the ends of its ranges: large counts, values far from one, tensors that do not fit a call."""
import math

import numpy as np
import pytest

import kv8_ref as R
import lastro_b200 as LB

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv8 import DT, Gpu, bounds, check_attend, ctx, f64, filled, ints, rows, same_values  # noqa: E402, F401


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


def test_attention_of_more_rows_than_can_be_counted_is_refused(ctx):
    """rows times heads right up to 2^31; the bound alone, with few rows, is taken"""
    gpu, ref, rng = filled(ctx, "e4m3", 1, 64, [20], max_pages=1)
    q, most = rows(rng, 3, 1, 64, "f32"), 2 ** 31 - 1
    out = torch.zeros_like(q)
    work = torch.zeros(gpu.c.attend_workspace(1, most, False), dtype=torch.uint8, device="cuda")
    many = [LB.Rows(x.data_ptr(), LB.DTYPE_F32, most, 0, 0) for x in (q, out)]
    call = dict(lens=ints([20]), q_off=ints([0, 3]), max_new=most, heads=1, scale=0.125, workspace=work, workspace_bytes=work.numel())
    assert code_of(gpu.c.attend, **call, q=many[0], out=many[1]) == LB.E_UNSUPPORTED
    gpu.c.attend(**call, q=LB.rows_of(q), out=LB.rows_of(out))
    want, _, big = ref.attend(0, f64(q), 0.125)
    assert (np.abs(f64(out) - want) <= bounds("f32", 64, big, np.abs(ref.side[0][0]["v"].values()).max())[1]).all()


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


# ---- calls right behind one another ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt,dtype,new", [("e4m3", "bf16", 1), ("int8", "f32", 6)])
def test_a_chain_of_calls_passes_its_results_on_the_device(ctx, fmt, dtype, new):
    """append, attend, evict, read, with lengths, masses and kept slots that stay on the device and nothing between the
    launches; again and again over the same buffers"""
    kv, d, heads, budget, recent, room = 2, 64, 4, 40, 8, 128
    lens = [100, 57, 41, 3]
    rng = np.random.default_rng(21)
    src, dst = Gpu(ctx, fmt, 4, kv, d, 2), Gpu(ctx, fmt, 4, kv, d, 1, seed=5)
    first = [[rows(rng, n, kv, d, dtype) for n in lens] for _ in "kv"]
    off0, off = ints(np.concatenate([[0], np.cumsum(lens)]).tolist()), ints([new * i for i in range(5)])
    zero, l0, l1, l2 = ints([0] * 4), ints([-1] * 4), ints([-1] * 4), ints([-1] * 4)
    mass, mass2 = (torch.zeros(4, kv, n, device="cuda") for n in (room, budget))
    kept = torch.zeros(4, kv, budget, dtype=torch.int32, device="cuda")
    out = torch.zeros(4 * new, heads, d, dtype=torch.bfloat16 if dtype == "bf16" else torch.float32, device="cuda")
    k, v = (torch.zeros(4, budget, kv, d, device="cuda") for _ in "kv")
    work = torch.zeros(src.c.attend_workspace(heads, new, True), dtype=torch.uint8, device="cuda")
    keep_alive = [torch.cat(x) for x in first]
    all0 = [LB.rows_of(x) for x in keep_alive]
    for step in range(8):
        q = [rows(rng, new, heads, d, dtype) for _ in lens]
        kn, vn = ([rows(rng, new, kv, d, dtype) for _ in lens] for _ in "kv")
        qc, kc, vc = (torch.cat(x) for x in (q, kn, vn))
        torch.cuda.synchronize()
        src.c.append(zero, off0, max(lens), *all0, l0, mass, room)
        src.c.append(l0, off, new, LB.rows_of(kc), LB.rows_of(vc), l1, mass, room)
        src.c.attend(l1, off, new, heads, LB.rows_of(qc), 0.125, LB.rows_of(out), work, work.numel(), mass_in=mass, mass_out=mass,
                     mass_stride=room)
        src.c.evict(dst.c, l1, budget, recent, mass, room, kept, l2, mass2, budget)
        dst.c.read(l2, zero, budget, k, v, "f32")
        ref = R.Cache(4, kv, d, fmt)
        got, gm, at = f64(out), f64(mass), 0
        assert l1.tolist() == [n + new for n in lens] and l2.tolist() == [min(n + new, budget) for n in lens]
        for b, n in enumerate(lens):
            ref.append(b, f64(first[0][b]), f64(first[1][b]))
            ref.append(b, f64(kn[b]), f64(vn[b]))
            want, wm, big = ref.attend(b, f64(q[b]), 0.125)
            vmax = max(np.abs(ref.side[b][h]["v"].values()).max() for h in range(kv))
            rel, tol = bounds(dtype, d, big, vmax)
            assert (np.abs(got[at:at + new] - want) <= tol + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0.0)).all()
            assert (np.abs(gm[b, :, :n + new] - wm) <= rel * wm + 2.0 ** -22 * wm).all()
            at += new
            for h, keep in enumerate(ref.evict(b, gm[b, :, :n + new], budget, recent)):
                assert kept[b, h, :len(keep)].tolist() == keep.tolist()
                for w, x in (("k", k), ("v", v)):
                    assert np.array_equal(f64(x[b, :len(keep), h]), ref.side[b][h][w].values())
    assert src.status.item() == 0 and dst.status.item() == 0


# ---- tensors that do not fit a call -----------------------------------------------------------------------------------------
def test_tensors_that_do_not_fit_are_refused(ctx):
    """of another type, place, layout or size than the call will read or write"""
    n, kv, d, heads, room = 3, 2, 64, 4, 40
    gpu, ref, rng = filled(ctx, "e4m3", kv, d, [20, 30, 5])
    q, k = rows(rng, n, heads, d, "bf16"), rows(rng, n, kv, d, "bf16")
    out, lens, off, lo = torch.zeros_like(q), ints([20, 30, 5]), ints([0, 1, 2, 3]), ints([0, 0, 0])
    mass, kept = torch.zeros(n, kv, room, device="cuda"), torch.zeros(n, kv, 16, dtype=torch.int32, device="cuda")
    size = gpu.c.attend_workspace(heads, 1, True)
    work = torch.zeros(size, dtype=torch.uint8, device="cuda")
    kr, vr = (torch.zeros(n, 8, kv, d, device="cuda") for _ in "kv")
    ro = LB.rows_of
    bad_ints = [lens.long(), lens.float(), lens.cpu(), lens[:2], ints([20, 0, 30, 0, 5, 0])[::2]]
    bad_mass = [mass.double(), mass.half(), mass.cpu(), mass[:2], mass[:, :1], mass[:, :, :39].contiguous(), mass.transpose(0, 1),
                torch.zeros(n, kv, 2 * room, device="cuda")[:, :, ::2], mass.flatten()[:-1]]
    good_mass = [mass, mass.flatten(), torch.zeros(n, kv, room, device="cuda")[:, :, :33]]

    def rows_like(x):
        return [ro(x[:, :1]), ro(x[:, :, :32].contiguous()), ro(torch.cat([x, x], 2)), ro(torch.cat([x, x], 1)), ro(x.cpu())]

    att = dict(lens=lens, q_off=off, max_new=1, heads=heads, q=ro(q), scale=0.125, out=ro(out), workspace=work, workspace_bytes=size,
               mass_in=mass, mass_out=mass, mass_stride=room)
    app = dict(lens=lens, new_off=off, max_new=1, k=ro(k), v=ro(k), lens_out=lo, mass=mass, mass_stride=room)
    dst = Gpu(ctx, "e4m3", n, kv, d, 1)
    evi = dict(dst=dst.c, lens=lens, budget=16, recent=4, mass=mass, mass_stride=room, kept=kept, lens_out=lo,
               mass_out=torch.zeros(n, kv, 16, device="cuda"), mass_out_stride=16)
    rd = dict(lens=lens, pos0=lo, n=8, k_out=kr, v_out=vr, dtype="f32")
    many = [kept.long(), kept[:, :, :15].contiguous(), kept.cpu(), kept.transpose(0, 1)]
    outs = [kr.bfloat16(), kr[:, :7].contiguous(), kr.cpu(), kr.transpose(1, 2)]
    for f, good, bad in (
            (gpu.c.attend, att, dict(lens=bad_ints, q_off=bad_ints + [off[:3]], q=rows_like(q), out=rows_like(out), mass_in=bad_mass,
                                     mass_out=bad_mass, workspace=[work[:-1], work.cpu(), work.view(-1, 1)[::2]])),
            (gpu.c.append, app, dict(lens=bad_ints, new_off=bad_ints + [off[:3]], lens_out=bad_ints, k=rows_like(k), v=rows_like(k),
                                     mass=bad_mass)),
            (gpu.c.evict, evi, dict(lens=bad_ints, kept=many, lens_out=bad_ints, mass=bad_mass, mass_out=[mass[:, :, :15].contiguous()])),
            (gpu.c.read, rd, dict(lens=bad_ints, pos0=bad_ints, k_out=outs, v_out=outs))):
        for name, values in bad.items():
            for x in values:
                assert code_of(f, **(good | {name: x})) == LB.E_ARG, (name, x)
    for x in good_mass:
        gpu.c.attend(**(att | dict(mass_in=x, mass_out=x)))
        gpu.c.append(**(app | dict(mass=x, max_new=0, new_off=ints([0] * 4))))
        gpu.c.evict(**(evi | dict(mass=x)))
    gpu.c.read(**rd)
    buffers = dict(k=gpu.k, v=gpu.v, k_scale=gpu.ks, v_scale=gpu.vs, page_table=gpu.table, status=gpu.status)
    make = lambda b: LB.Kv8Cache(ctx, "e4m3", n, kv, d, gpu.num_pages, gpu.table.shape[1], **b)  # noqa: E731
    make(buffers)
    for name, t in buffers.items():
        for x in (t.cpu(), t.flatten()[:-1], t.double()) + ((t.transpose(0, 1),) if t.ndim > 1 and name != "page_table" else ()):
            if name in "kv" and x.dtype == torch.float64:
                continue  # codes may be of any type, they are bytes
            assert code_of(make, buffers | {name: x}) == LB.E_ARG, name
    torch.cuda.synchronize()
    assert gpu.status.item() == 0


# ---- threads --------------------------------------------------------------------------------------------------------------
THREADS = """
import sys, threading
sys.path[:0] = %r
import torch
import lastro_b200 as LB

SIZES = [256, 135, 250, 140, 2048, 258, 1500, 300] * 3  # pages: what the selection's launches take, of either kind
sys.setswitchinterval(1e-6)
torch.zeros(1, device="cuda")


class Evict:
    def __init__(self, pages):
        self.ctx = LB.Context(0)
        g = dict(device="cuda")
        n, self.n = 2 * pages, pages * 64
        self.k, self.v = torch.zeros((2, n, 1, 64, 64), dtype=torch.uint8, **g).unbind()
        self.s = torch.ones((n, 1, 4), **g)
        self.table = torch.arange(n, dtype=torch.int32, **g).view(2, 1, pages)
        self.src, self.dst = (LB.Kv8Cache(self.ctx, "int8", 1, 1, 64, n, pages, self.k, self.v, self.s, self.s.clone(), t) for t in self.table)
        self.mass = torch.arange(self.n, device="cuda").float().view(1, 1, -1)
        self.lens, self.out = (torch.tensor([x], dtype=torch.int32, **g) for x in (self.n, 0))
        self.kept = torch.zeros((1, 1, 100), dtype=torch.int32, **g)

    def __call__(self):
        self.src.evict(self.dst, self.lens, 100, 10, self.mass, self.n, self.kept, self.out)


calls = [Evict(p) for p in SIZES]
torch.cuda.synchronize()
together, errors = threading.Barrier(len(calls)), []


def first(c):
    together.wait()
    try:
        c()
    except LB.LastroError as e:
        errors.append(str(e))


threads = [threading.Thread(target=first, args=(c,)) for c in calls]
[t.start() for t in threads]
[t.join() for t in threads]
for c in calls + calls[::-1]:
    first.__globals__["together"] = threading.Barrier(1)
    first(c)
torch.cuda.synchronize()
for c in calls:
    if c.out.item() != 100 or c.kept[0, 0].tolist() != list(range(c.n - 100, c.n)):
        errors.append("kept %%s" %% c.kept[0, 0, :4].tolist())
sys.exit("; ".join(errors) or 0)
"""


def test_first_calls_from_several_threads(ctx):
    """each with a context and a cache of another size: a launch's shared memory must not be what another thread asked for"""
    import os
    import subprocess
    import sys
    for _ in range(2):
        r = subprocess.run([sys.executable, "-c", THREADS % [os.path.dirname(os.path.dirname(LB.__file__))]], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-2000:]


# ---- outputs in the queries' place ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_outputs_over_the_queries(ctx, dtype):
    """out may be q itself unless q is read again for the weights, which is refused, as is q's address in another layout"""
    lens, kv, d = [300, 65, 9001], 2, 64
    gpu, _, rng = filled(ctx, "e4m3", kv, d, lens)
    for group, new, mass in ((3, 1, True), (3, 1, False), (2, 3, True), (2, 20, False), (1, 12, False), (3, 4, True), (1, 40, True)):
        q, heads = [rows(rng, new, kv * group, d, dtype) for _ in lens], kv * group
        want = gpu.attend(lens, q, 0.125, mass=mass)
        both = torch.cat(q)
        m = torch.full_like(want[1], -5.0) if mass else None
        work = torch.zeros(gpu.c.attend_workspace(heads, new, mass), dtype=torch.uint8, device="cuda")
        call = dict(lens=ints(lens), q_off=ints([0, new, 2 * new, 3 * new]), max_new=new, heads=heads, q=LB.rows_of(both), scale=0.125,
                    out=LB.rows_of(both), workspace=work, workspace_bytes=work.numel(), mass_out=m, mass_stride=max(lens) if mass else 0)
        if mass and group * new > 8:
            assert code_of(gpu.c.attend, **call) == LB.E_ARG
            continue
        gpu.c.attend(**call)
        assert torch.equal(both, want[0]) and (not mass or torch.equal(m, want[1]))
    turned = torch.cat(q).transpose(0, 1).contiguous().transpose(0, 1)
    call |= dict(q=LB.rows_of(turned), out=LB.rows_of(torch.empty(0, device="cuda").to(turned.dtype).set_(turned.untyped_storage(), 0, turned.shape)),
                 mass_out=None, mass_stride=0)
    assert code_of(gpu.c.attend, **call) == LB.E_ARG


# ---- values and scores far from one -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt,dtype,group,new", [("e4m3", "f32", 3, 1), ("int8", "bf16", 3, 1), ("int8", "f32", 9, 1), ("e4m3", "bf16", 4, 9),
                                                 ("e4m3", "f32", 2, 17)])
@pytest.mark.parametrize("size", [1e-30, 1e-33, 3e-36, 1e-37])
def test_small_values_throughout(ctx, fmt, dtype, group, new, size):
    """V near the smallest normal f32: the outputs are as large, and as exact, as for values near one.  Beside the usual terms
    the weights' second f16 terms lose what is below 2^-24 of the heaviest weight, for each slot, and outputs are multiples
    of 2^-149."""
    lens, kv, d = [500, 1, 70], 2, 64
    rng = np.random.default_rng(31)
    gpu, ref = Gpu(ctx, fmt, 3, kv, d, 9), R.Cache(3, kv, d, fmt)
    k, v = [rows(rng, n, kv, d, dtype) for n in lens], [rows(rng, n, kv, d, "f32", size).to(DT[dtype]) for n in lens]
    gpu.append([0] * 3, k, v)
    for b in range(3):
        ref.append(b, f64(k[b]), f64(v[b]))
    same_values(gpu, ref, lens)
    q, at = [rows(rng, min(new, n), kv * group, d, dtype) for n in lens], 0
    out = f64(gpu.attend(lens, q, 0.125)[0])
    for b, n in enumerate(lens):
        want, _, big = ref.attend(b, f64(q[b]), 0.125)
        vmax = max(np.abs(ref.side[b][h]["v"].values()).max() for h in range(kv))
        _, tol = bounds(dtype, d, big, vmax)
        tol += n * 2.0 ** -24 * vmax + 2.0 ** -149
        got = out[at:at + len(q[b])]
        assert (np.abs(got - want) <= tol + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0.0)).all(), (b, np.abs(got - want).max(), tol)
        at += len(q[b])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("group,new", [(3, 1), (9, 1), (4, 9)])
@pytest.mark.parametrize("score", [2.0 ** 20, 2.0 ** 27, 2.0 ** 40, 1e35])
def test_scores_far_from_zero(ctx, dtype, group, new, score):
    """every slot has the same score, far from zero on either side: the same bits for all, so every weight is the same and an
    output is the mean of the values it sees, whatever their scales are"""
    lens, kv, d = [9001, 33], 1, 64
    rng = np.random.default_rng(33)
    k = torch.zeros(max(lens), kv, d)
    k[:, :, 0] = score
    for size in (1.0, 1e4, 1e-6):
        gpu, ref = Gpu(ctx, "int8", 2, kv, d, 141), R.Cache(2, kv, d, "int8")
        v = [rows(rng, n, kv, d, "f32", size) for n in lens]
        gpu.append([0, 0], [k[:n].cuda() for n in lens], v)
        for b in range(2):
            ref.append(b, f64(k[:lens[b]]), f64(v[b]))
        q = [rows(rng, new, group, d, dtype) for _ in lens]
        for x in q:
            x[:, :, 0] = torch.tensor([1.0, -1.0])[torch.arange(group) % 2].to(x)
        out = f64(gpu.attend(lens, q, 1.0)[0])
        for b, n in enumerate(lens):
            x = ref.side[b][0]["v"].values()
            for i in range(new):
                want = x[:n - new + i + 1].mean(0)
                tol = np.abs(x).max() * (2.0 ** -20 + (2.0 ** -11 if dtype == "bf16" else 0.0)) + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0.0)
                assert (np.abs(out[b * new + i] - want) <= tol).all(), (size, b, i)


# ---- weights ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("group,new", [(2, 3), (1, 8), (3, 7), (2, 40)])
def test_weights_of_rows_that_are_not_finite_stay_apart(ctx, dtype, group, new):
    """a query that holds NaN or infinity gives NaN to the slots it sees and nothing to the others; what a page outside the
    pool would hold gets nothing"""
    lens, kv, d = [100, 50], 1, 64
    gpu, _, rng = filled(ctx, "e4m3", kv, d, lens)
    q = [rows(rng, new, group, d, dtype) for _ in lens]
    _, clean = gpu.attend(lens, q, 0.125, mass=True)
    for bad in (math.nan, math.inf):
        x = [t.clone() for t in q]
        x[0][1, 0, 5] = bad
        _, mass = gpu.attend(lens, x, 0.125, mass=True)
        see = lens[0] - new + 2  # slots that query 1 sees
        assert mass[0, :, :see].isnan().all() and torch.equal(mass[0, :, see:], clean[0, :, see:])
        assert torch.equal(mass[1], clean[1])
    assert gpu.status.item() == 0
    gpu.table[0, 0] = -1
    _, mass = gpu.attend(lens, x, 0.125, mass=True)
    assert (mass[0, :, :64] == 0).all() and torch.equal(mass[1], clean[1]) and gpu.status.item() == LB.KV8_BAD_PAGE


@pytest.mark.parametrize("group,new", [(3, 1), (2, 4), (3, 7)])
@pytest.mark.parametrize("score", [0.0, 1e5, 2.0 ** 23, 1e9, -1e5, -1e9, -1e30])
def test_weights_of_scores_far_from_zero(ctx, group, new, score):
    """every slot has the same score: each gets the same weight, and a row hands out 1"""
    lens, kv, d = [5000, 40], 1, 64
    k = torch.zeros(max(lens), kv, d, device="cuda")
    k[:, :, 0] = score
    gpu = Gpu(ctx, "int8", 2, kv, d, 79)
    gpu.append([0, 0], [k[:n] for n in lens], [k[:n] for n in lens])
    q = torch.zeros(new, group, d, device="cuda")
    q[:, :, 0] = 1.0
    _, mass = gpu.attend(lens, [q, q], 1.0, mass=True)
    for b, n in enumerate(lens):
        want = sum(group * (torch.arange(n) < n - new + i + 1).double() / (n - new + i + 1) for i in range(new))
        assert (np.abs(f64(mass[b, 0, :n]) - want.numpy()) <= 2.0 ** -20 * want.numpy()).all()


# ---- prompts -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt,kv,group,d,dtype", [("e4m3", 2, 3, 64, "bf16"), ("int8", 1, 4, 128, "f32"), ("int8", 1, 1, 64, "bf16")])
def test_attention_over_a_prompt(ctx, fmt, kv, group, d, dtype):
    """hundreds of queries a sequence, some of them all of its slots, with and without the weights"""
    lens, news = [700, 513, 64, 900], [700, 257, 64, 1]
    gpu, ref, rng = filled(ctx, fmt, kv, d, lens)
    check_attend(gpu, ref, rng, lens, news, kv * group, dtype)
    check_attend(gpu, ref, rng, lens, news, kv * group, dtype, with_mass=False)
