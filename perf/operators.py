"""Workloads of the 8-bit KV cache operators: append, attention, eviction.

Each operator in two forms that take the same state: ``run`` with ``own`` true makes the calls a user makes
(``lastro_b200.Kv8Cache``), with ``own`` false it computes the same from elementary torch operations in 32 bits.

The cache: pages of 64 slots, blocks of 16; codes [num_pages, kv_heads, 64, d] (one byte: e4m3 or int8), scales
[num_pages, kv_heads, 4] (f32 powers of two); value = code * scale; page_table [n_seqs, max_pages] (-1: no page).
"""
import os
import sys

import torch

own = False

PAGE, BLOCK = 64, 16
QMAX = {"e4m3": 448.0, "int8": 127.0}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ----------------------------------------------------------------------------------------------------------
# batch sequences whose lengths run from ctx - spread to ctx; kv KV heads of `group` query heads each, head dimension d;
# `new` tokens per sequence this step (every fourth sequence half of them); fmt the cache's format, dtype the rows'.
def _append(batch, ctx, spread, new, kv, group, d, fmt, dtype):
    return dict(op="append", batch=batch, ctx=ctx, spread=spread, new=new, kv=kv, group=group, d=d, fmt=fmt,
                dtype=dtype)


def _attend(batch, ctx, spread, new, kv, group, d, fmt, dtype, mass):
    return dict(op="attend", batch=batch, ctx=ctx, spread=spread, new=new, kv=kv, group=group, d=d, fmt=fmt,
                dtype=dtype, mass=mass)


def _evict(batch, ctx, spread, budget, recent, kv, d, fmt):
    return dict(op="evict", batch=batch, ctx=ctx, spread=spread, budget=budget, recent=recent, kv=kv, d=d,
                fmt=fmt)


def listed():
    return [
        # one layer of one decode step of the 3B model for 64 sequences around 1024 tokens of context
        {"name": "append-decode"} | _append(64, 1024, 63, 1, 8, 3, 64, "e4m3", "bf16"),
        # a prompt chunk of several sequences, each on top of an odd-sized context
        {"name": "append-prompt"} | _append(8, 1333, 200, 4097, 8, 4, 128, "int8", "bf16"),
        # one layer of the batch-1 decode step at context 2048 (the 3B model's heads, the model's f32 activations)
        {"name": "attend-single"} | _attend(1, 2048, 0, 1, 8, 3, 64, "e4m3", "f32", False),
        # freshly started chats: contexts of 1 to 65 tokens, one query head to a KV head
        {"name": "attend-short"} | _attend(96, 65, 64, 1, 8, 1, 64, "int8", "f32", True),
        # the 64-sequence batch at context 1024
        {"name": "attend-batch"} | _attend(64, 1024, 63, 1, 8, 3, 64, "e4m3", "bf16", False),
        # few sequences, long contexts, the weights accumulated for a later eviction
        {"name": "attend-long"} | _attend(4, 65537, 9000, 1, 8, 3, 64, "e4m3", "bf16", True),
        # a multi-position step: 32 positions of each sequence
        {"name": "attend-positions"} | _attend(8, 2048, 77, 32, 8, 3, 64, "int8", "bf16", True),
        # ragged batch with wider heads, weights accumulated, f32 rows
        {"name": "attend-ragged"} | _attend(24, 8191, 8000, 1, 8, 4, 128, "int8", "f32", True),
        # the largest: a full serving batch, wide heads
        {"name": "attend-serving"} | _attend(96, 8192, 1000, 1, 8, 4, 128, "e4m3", "bf16", False),
        # one sequence of the 1B/3B models' heads just past its budget
        {"name": "evict-single"} | _evict(1, 2049, 0, 1024, 128, 8, 64, "e4m3"),
        # a batch cut to a quarter of its contexts
        {"name": "evict-batch"} | _evict(64, 4097, 1000, 1000, 250, 8, 64, "int8"),
        # few very long contexts
        {"name": "evict-long"} | _evict(2, 131072, 30001, 16384, 1024, 8, 128, "e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict"])
    d, kv, fmt, dtype = rng.choice([64, 128]), rng.choice([1, 2, 4, 8]), rng.choice(["e4m3", "int8"]), rng.choice(["bf16", "f32"])
    batch = _log(rng, 1, 96)
    row = batch * kv * d * 2  # cache bytes of one slot of every sequence
    if op == "append":
        new = rng.choice([1, 1, _log(rng, 2, max(3, min(8192, (1 << 26) // row)))])
        ctx = _log(rng, 1, max(2, min(16384, (1 << 29) // row)))
        return _append(batch, ctx, rng.randint(0, ctx), new, kv, rng.choice([1, 3, 4]), d, fmt, dtype)
    if op == "attend":
        group = rng.choice([1, 2, 3, 4, 8])
        new = rng.choice([1, 1, rng.randint(2, 32)])
        ctx = _log(rng, 33, max(40, min(131072, 1500000000 // row, (1 << 28) // (batch * kv * group * new))))
        return _attend(batch, ctx, rng.randint(0, ctx - new), new, kv, group, d, fmt, dtype, rng.random() < 0.5)
    ctx = _log(rng, 65, max(70, min(131072, 600000000 // row, (1 << 25) // (batch * kv))))
    budget = _log(rng, 17, ctx)
    return _evict(batch, ctx, rng.randint(0, ctx), budget, rng.randint(0, budget), kv, d, fmt)


def _lens(case):
    return [case["ctx"] - (b * 7919) % (case["spread"] + 1) for b in range(case["batch"])]


def _news(case):
    return [max(1, case["new"] // 2) if b % 4 == 3 else case["new"] for b in range(case["batch"])]


def _pages(n):
    return (n + PAGE - 1) // PAGE


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _values(shape, gen, d, spread=0.6):
    """K/V-like values: normal, some channels several times larger than others."""
    chan = torch.exp(spread * torch.randn(d, generator=gen, device="cuda"))
    return torch.randn(shape, generator=gen, device="cuda").mul_(chan)


def _need(amax, fmt):
    """The smallest power of two s >= 2^-126 with amax <= qmax * s: from the mantissa and the exponent, exactly."""
    m, e = torch.frexp(amax)
    top, shift = (0.875, 9) if fmt == "e4m3" else (127 / 128, 7)
    e = torch.where(m > top, e - shift + 1, e - shift).clamp(min=-126)
    e = torch.where(amax == 0, -126, e)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(x, fmt):
    """Values of the format's grid nearest to x (|x| <= qmax)."""
    return x.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(x).to(torch.int8)


def _cache(case, gen, lens):
    """A filled cache whose sequences take randomly placed pages: codes, scales and the page table."""
    kv, d, fmt = case["kv"], case["d"], case["fmt"]
    counts = [_pages(n) for n in lens]
    total, most = max(1, sum(counts)), max(1, max(counts))
    st = {}
    for w in "kv":
        x = _values((total, kv, PAGE // BLOCK, BLOCK, d), gen, d)
        s = _need(x.abs().amax((3, 4)), fmt)
        st[w], st[w + "_scale"] = _codes(x / s[..., None, None], fmt).view(torch.uint8).view(total, kv, PAGE, d), s
    perm = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), most), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    return st | {"page_table": table, "total": total, "most": most}


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _kv8(LB, ctx, case, st, pre=""):
    return LB.Kv8Cache(ctx, case["fmt"], case["batch"], case["kv"], case["d"], st[pre + "total"], st[pre + "most"],
                       st[pre + "k"], st[pre + "v"], st[pre + "k_scale"], st[pre + "v_scale"], st[pre + "page_table"])


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    B, kv, d, op = case["batch"], case["kv"], case["d"], case["op"]
    lens = _lens(case)
    st = {"case": case}
    if op == "evict":
        st |= _cache(case, gen, lens)
        most = max(lens)
        # accumulated weights: skewed, with ties and zeros
        st["mass"] = torch.exp(1.5 * torch.randn((B, kv, most), generator=gen, device="cuda")).mul_(64).floor_().div_(64)
        C = case["budget"]
        st["dst_total"], st["dst_most"] = max(1, B * _pages(C)), max(1, _pages(C))
        st["dst_page_table"] = torch.randperm(st["dst_total"], generator=gen, device="cuda").to(torch.int32).view(B, -1)
        st["lens"] = _ints(lens)
    else:
        news = _news(case)
        T, G, dt = sum(news), case["group"], DTYPES[case["dtype"]]
        off = [0]
        for n in news:
            off.append(off[-1] + n)
        total = [n + (m if op == "append" else 0) for n, m in zip(lens, news)]
        st |= _cache(case, gen, total)
        st["lens"], st["off"] = _ints(lens), _ints(off)
        st["row_seq"] = torch.repeat_interleave(torch.arange(B), torch.tensor(news)).cuda()
        st["row_i"] = torch.cat([torch.arange(n) for n in news]).cuda()
        if op == "append":  # K and V as the fused projection leaves them: slices of one row
            qkv = torch.randn((T, (G + 2) * kv * d), generator=gen, device="cuda").mul_(1.5)
            qkv *= torch.exp2(torch.randint(-1, 3, (T, 1), generator=gen, device="cuda").float())
            qkv = qkv.to(dt)
            st["k_new"] = qkv[:, G * kv * d:(G + 1) * kv * d].view(T, kv, d)
            st["v_new"] = qkv[:, (G + 1) * kv * d:].view(T, kv, d)
            st["pos0"] = _ints([n // BLOCK * BLOCK for n in lens])
        else:
            st["q"] = _values((T, kv * G, d), gen, d, 0.3).mul_(1.5).to(dt)
            if case["mass"]:
                st["mass"] = torch.exp(torch.randn((B, kv, max(lens)), generator=gen, device="cuda"))
    _buffers(case, st)
    if own:
        _handles(case, st)
    return st


def _buffers(case, st):
    """The outputs' buffers, which a serving program keeps from step to step."""
    B, kv, d, op = case["batch"], case["kv"], case["d"], case["op"]
    if op == "attend":
        st["out"] = torch.zeros_like(st["q"])
        st["mass_out"] = torch.zeros_like(st["mass"]) if case["mass"] else None
        return
    n = case["budget"] if op == "evict" else case["new"] + BLOCK
    st["k_out"], st["v_out"] = torch.zeros((2, B, n, kv, d), dtype=torch.bfloat16, device="cuda").unbind()
    st["lens_out"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    if op == "evict":
        st["dst_k"], st["dst_v"] = torch.zeros((2, st["dst_total"], kv, PAGE, d), dtype=torch.uint8, device="cuda").unbind()
        st["dst_k_scale"], st["dst_v_scale"] = torch.zeros((2, st["dst_total"], kv, PAGE // BLOCK), device="cuda").unbind()
        st["kept"] = torch.zeros((B, kv, n), dtype=torch.int32, device="cuda")
        st["mass_out"] = torch.zeros((B, kv, n), device="cuda")
        st["pos0"] = torch.zeros(B, dtype=torch.int32, device="cuda")


def _handles(case, st):
    """The context on the program's stream, the caches' handles and the attention's workspace."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lastro-rust_b200"))
    import lastro_b200 as LB
    ctx = LB.Context(0, torch.cuda.current_stream().cuda_stream or LB.LEGACY_STREAM)
    st["LB"], st["ctx"], st["cache"] = LB, ctx, _kv8(LB, ctx, case, st)
    if case["op"] == "attend":
        n = st["cache"].attend_workspace(case["kv"] * case["group"], case["new"], case["mass"])
        st["work"], st["work_bytes"] = torch.zeros(n, dtype=torch.uint8, device="cuda"), n
    if case["op"] == "evict":
        st["dst"] = _kv8(LB, ctx, case, st, "dst_")


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "evict": _own_evict}[case["op"]](case, st)
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[case["op"]](case, st)


def _own_append(case, st):
    LB, c = st["LB"], st["cache"]
    c.append(st["lens"], st["off"], case["new"], LB.rows_of(st["k_new"]), LB.rows_of(st["v_new"]), st["lens_out"])
    c.read(st["lens_out"], st["pos0"], case["new"] + BLOCK, st["k_out"], st["v_out"], "bf16")
    return {"k": st["k_out"], "v": st["v_out"], "lens": st["lens_out"]}


def _own_attend(case, st):
    LB = st["LB"]
    st["cache"].attend(st["lens"], st["off"], case["new"], case["kv"] * case["group"], LB.rows_of(st["q"]),
                       case["d"] ** -0.5, LB.rows_of(st["out"]), st["work"], st["work_bytes"], mass_in=st.get("mass"),
                       mass_out=st["mass_out"], mass_stride=st["mass"].shape[2] if case["mass"] else 0)
    return {"out": st["out"], "mass": st["mass_out"]} if case["mass"] else {"out": st["out"]}


def _own_evict(case, st):
    C = case["budget"]
    st["cache"].evict(st["dst"], st["lens"], C, case["recent"], st["mass"], st["mass"].shape[2], st["kept"],
                      st["lens_out"], st["mass_out"], C)
    st["dst"].read(st["lens_out"], st["pos0"], C, st["k_out"], st["v_out"], "bf16")
    return {"k": st["k_out"], "v": st["v_out"], "mass": st["mass_out"], "kept": st["kept"], "lens": st["lens_out"]}


def _real(codes, fmt):
    return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).float()


def _quantised(x, s, fmt):
    """x at scale s: rounded onto the grid and back to the values the codes stand for."""
    return _codes(x / s, fmt).float() * s


def _plain_append(case, st):
    B, kv, d, fmt, n = case["batch"], case["kv"], case["d"], case["fmt"], case["new"] + BLOCK
    lens, off, dev = st["lens"].long(), st["off"].long(), "cuda"
    blocks = (n + BLOCK - 1) // BLOCK
    slot = (lens // BLOCK * BLOCK)[:, None] + torch.arange(blocks * BLOCK, device=dev)  # [B, slots]
    count = off[1:] - off[:-1]
    i = slot - lens[:, None]
    fresh = (i >= 0) & (i < count[:, None])
    src = (off[:-1, None] + i).clamp(0, st["k_new"].shape[0] - 1)
    seq = torch.arange(B, device=dev)[:, None]
    old = i < 0
    page = st["page_table"].long()[seq, (slot // PAGE).clamp(max=st["most"] - 1)].clamp(min=0)

    def rows(w):
        new = torch.where(fresh[..., None, None], st[w + "_new"][src].float(), 0.0)  # [B, slots, kv, d]
        had = _real(st[w][page[:, :BLOCK], :, (slot % PAGE)[:, :BLOCK]], fmt)  # the first block may hold earlier rows
        was = st[w + "_scale"][page[:, 0], :, slot[:, 0] % PAGE // BLOCK]  # [B, kv]
        s = _need(new.abs().view(B, blocks, BLOCK, kv, d).amax((2, 4)), fmt)  # [B, blocks, kv]
        s[:, 0] = torch.where(old[:, :1], torch.maximum(s[:, 0], was), s[:, 0])
        new[:, :BLOCK] = torch.where(old[:, :BLOCK, None, None], had * was[:, None, :, None], new[:, :BLOCK])
        return _quantised(new, s.repeat_interleave(BLOCK, 1)[..., None], fmt)[:, :n].to(torch.bfloat16)

    return {"k": rows("k"), "v": rows("v"), "lens": (lens + count).to(torch.int32)}


def _paged(st, w, fmt):
    """K or V of every sequence as f32 [B, kv, slots, d]."""
    table = st["page_table"].long().clamp(min=0)
    x = _real(st[w][table], fmt)  # [B, pages, kv, 64, d]
    x = x.unflatten(3, (PAGE // BLOCK, BLOCK)) * st[w + "_scale"][table][..., None, None]
    return x.flatten(3, 4).transpose(1, 2).flatten(2, 3)


def _plain_attend(case, st):
    B, kv, G, d, n = case["batch"], case["kv"], case["group"], case["d"], case["new"]
    lens, off = st["lens"].long(), st["off"].long()
    k, v = _paged(st, "k", case["fmt"]), _paged(st, "v", case["fmt"])
    slots, dev = k.shape[2], k.device
    count = off[1:] - off[:-1]
    i = torch.arange(n, device=dev)
    src = (off[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][src].float().view(B, n, kv, G, d).permute(0, 2, 1, 3, 4).reshape(B, kv, n * G, d)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(B, kv, n, G, slots)
    see = (lens - count)[:, None] + i  # the last slot query i sees
    seen = (torch.arange(slots, device=dev) <= see[..., None]) & (i < count[:, None])[..., None]  # [B, n, slots]
    s.masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = s.sub_(top).exp_()
    p /= p.sum(-1, keepdim=True).clamp(min=1e-38)
    o = torch.matmul(p.view(B, kv, n * G, slots), v).view(B, kv, n, G, d)
    out = {"out": o[st["row_seq"], :, st["row_i"]].reshape(-1, kv * G, d).to(st["q"].dtype)}
    if case["mass"]:
        m = st["mass"].shape[2]
        got = st["mass"] + p.sum((2, 3))[..., :m]
        out["mass"] = torch.where(torch.arange(m, device=dev) < lens[:, None, None], got, 0.0)
    return out


def _plain_evict(case, st):
    B, kv, d, fmt, C, R = case["batch"], case["kv"], case["d"], case["fmt"], case["budget"], case["recent"]
    lens, mass = st["lens"].long(), st["mass"]
    most, dev = mass.shape[2], mass.device
    t, L = torch.arange(most, device=dev), lens[:, None, None]
    key = torch.where(t >= L - R, torch.inf, mass).masked_fill_(t >= L, -torch.inf)
    take = min(C, most)
    best = key.sort(dim=-1, descending=True, stable=True).indices[..., :take]
    kept = torch.where(best < L, best, most).sort(-1).values
    kept = torch.nn.functional.pad(kept, (0, C - take), value=most)
    there = kept < most
    at = kept.clamp(max=most - 1)
    blocks = (C + BLOCK - 1) // BLOCK
    page = st["page_table"].long().clamp(min=0)[torch.arange(B, device=dev)[:, None, None], at // PAGE]
    head = torch.arange(kv, device=dev)[:, None]

    def rows(w):
        x = _real(st[w][page, head, at % PAGE], fmt) * st[w + "_scale"][page, head, at % PAGE // BLOCK][..., None]
        x = torch.where(there[..., None], x, 0.0)
        x = torch.nn.functional.pad(x, (0, 0, 0, blocks * BLOCK - C)).unflatten(2, (blocks, BLOCK))
        s = _need(x.abs().amax((3, 4), keepdim=True), fmt)
        return _quantised(x, s, fmt).flatten(2, 3)[:, :, :C].transpose(1, 2).to(torch.bfloat16)

    return {"k": rows("k"), "v": rows("v"), "mass": torch.where(there, torch.gather(mass, 2, at), 0.0),
            "kept": torch.where(there, kept, -1).to(torch.int32), "lens": lens.clamp(max=C).to(torch.int32)}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    kv, d, op = case["kv"], case["d"], case["op"]
    lens = _lens(case)
    block = 2 * (BLOCK * d + 4)  # K and V of one block and head: codes and scales
    if op == "evict":
        keep = [min(n, case["budget"]) for n in lens]
        moved = sum(-(-n // BLOCK) for n in keep) * kv * block
        return {"bytes": sum(lens) * kv * 4 + 2 * moved + sum(keep) * kv * (8 + 4 * d), "flops": 0}
    news, item = _news(case), DTYPES[case["dtype"]].itemsize
    if op == "append":  # rows in, their codes out, and the values of the touched blocks handed back
        touched = sum(-(-(n + m) // BLOCK) - n // BLOCK for n, m in zip(lens, news))
        return {"bytes": sum(news) * kv * 2 * d * item + touched * kv * block + touched * BLOCK * kv * 2 * d * 2, "flops": 0}
    rows = sum(news) * kv * case["group"] * d * item * 2
    mass = sum(lens) * kv * 8 if case["mass"] else 0
    seen = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, news))
    return {"bytes": sum(-(-n // BLOCK) for n in lens) * kv * block + rows + mass, "flops": 4 * seen * kv * case["group"] * d}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _scale64(a, fmt):
    """need() by search: every power of two from 2^-126 up, the first that holds the largest magnitude."""
    e = torch.tensor([2.0 ** k for k in range(-126, 128)], device="cuda", dtype=torch.float64)
    return e[torch.searchsorted(e * QMAX[fmt], a.contiguous())]


def _round64(x, fmt):
    """Nearest value of the format's grid, ties to even."""
    if fmt == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _seq64(st, w, b, length, fmt):
    """K or V of sequence b as f64 [kv, length, d]."""
    pages = st["page_table"][b, :_pages(length)].long()
    c = st[w][pages].view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).double()
    s = st[w + "_scale"][pages].double().repeat_interleave(BLOCK, 2)
    return (c * s[..., None]).permute(1, 0, 2, 3).reshape(c.shape[1], c.shape[0] * PAGE, c.shape[3])[:, :length]


def exact(case, seed):
    st = prepare(case, seed)
    lens, fmt, kv, d = _lens(case), case["fmt"], case["kv"], case["d"]
    off = st["off"].tolist() if "off" in st else None
    res = []
    for b, n in enumerate(lens):
        if case["op"] == "append":
            m, first = off[b + 1] - off[b], n // BLOCK * BLOCK
            got = {}
            for w in "kv":
                rows = torch.zeros((case["new"] + BLOCK, kv, d), dtype=torch.float64, device="cuda")
                prior = _seq64(st, w, b, n, fmt)[:, first:].transpose(0, 1)
                rows[:n - first], rows[n - first:n - first + m] = prior, st[w + "_new"][off[b]:off[b + 1]].double()
                pad = -rows.shape[0] % BLOCK
                blk = torch.nn.functional.pad(rows, (0, 0, 0, 0, 0, pad)).unflatten(0, (-1, BLOCK))
                a = blk.abs()
                a[0, :n - first] = 0
                s = _scale64(a.amax((1, 3)), fmt)
                if n > first:
                    s[0] = torch.maximum(s[0], st[w + "_scale"][st["page_table"][b, n // PAGE].long(), :, n % PAGE // BLOCK].double())
                s = s[:, None, :, None]
                got[w] = (_round64(blk / s, fmt) * s).flatten(0, 1)[:rows.shape[0]]
            res.append(got)
        elif case["op"] == "attend":
            m, G = off[b + 1] - off[b], case["group"]
            k, v = (_seq64(st, w, b, n, fmt) for w in "kv")
            q = st["q"][off[b]:off[b + 1]].double().view(m, kv, G, d)
            z = torch.einsum("ihgd,htd->higt", q, k) / d ** 0.5
            z += torch.full((m, n), -torch.inf, device="cuda", dtype=torch.float64).triu(n - m + 1)[:, None]
            p = torch.softmax(z, -1)
            got = {"out": torch.einsum("higt,htd->ihgd", p, v).reshape(m, kv * G, d)}
            if case["mass"]:
                got["mass"] = torch.zeros(st["mass"].shape[1:], dtype=torch.float64, device="cuda")
                got["mass"][:, :n] = st["mass"][b, :, :n].double() + p.sum((1, 2))
            res.append(got)
        else:
            C, R = case["budget"], case["recent"]
            got = {w: torch.zeros((C, kv, d), dtype=torch.float64, device="cuda") for w in "kv"}
            got["mass"] = torch.zeros((kv, C), dtype=torch.float64, device="cuda")
            for h in range(kv):
                mass = st["mass"][b, h, :n].double()
                keep = torch.arange(n, device="cuda")
                if n > C:
                    order = torch.argsort(-mass[:n - R], stable=True)[:C - R].sort().values
                    keep = torch.cat([order, keep[n - R:]])
                got["mass"][h, :keep.numel()] = mass[keep]
                if h == 0:
                    full = {w: _seq64(st, w, b, n, fmt) for w in "kv"}
                for w in "kv" if n else "":
                    x = full[w][h, keep]
                    blk = torch.nn.functional.pad(x, (0, 0, 0, -x.shape[0] % BLOCK)).unflatten(0, (-1, BLOCK))
                    s = _scale64(blk.abs().amax((1, 2)), fmt)[:, None, None]
                    got[w][:keep.numel(), h] = (_round64(blk / s, fmt) * s).flatten(0, 1)[:keep.numel()]
            res.append(got)
    join = torch.cat if case["op"] == "attend" else torch.stack
    out = {w: (join if w == "out" else torch.stack)([r[w] for r in res]) for w in res[0]}
    return out | ({"lens": None} if case["op"] == "append" else {"kept": None, "lens": None} if case["op"] == "evict" else {})
