// 8-bit KV cache: append (quantise), eviction, read-back (attention in kv8_attend.cu).  Layout and rules in
// include/lastro_b200.h.
#include <cuda_runtime.h>

#include "kv8.cuh"

namespace lastro {
namespace {

// ---- append ---------------------------------------------------------------------------------------------------------
// One warp quantises one block (16 slots) of K and V of one head: its new rows are read once into registers (a lane holds
// groups of 8 values), the largest magnitude comes by a warp reduction, then the codes.  The block's earlier rows are read
// and rounded again only where the scale grows.  Bound by memory, 2 or 4 bytes a value in and 1 out, and by loads that each
// warp has on its way only once: 41 us for 28,678 rows of 8 sequences, 8 heads of 128 in bf16 (177 MB, 4.4 TB/s); one row each
// for 64 sequences takes 3.2 us, four dependent loads.
template <int FMT, int D, bool F32>
__global__ void __launch_bounds__(256) kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a) {
    constexpr int LPR = D / 8, RPW = 32 / LPR, N = kKv8Block / RPW;  // lanes a row, rows a pass, passes
    pdl_wait();
    pdl_launch();
    const int lane = threadIdx.x & 31, H = a.kv.kv_heads, b = blockIdx.y;
    const int unit = blockIdx.x * 8 + (threadIdx.x >> 5), j = unit / H, h = unit - j * H;
    if (j >= a.blocks) return;
    int64_t most = (int64_t)a.kv.max_pages * kKv8Page;
    if (a.mass) most = min(most, a.mass_stride);
    const int given = a.lens[b], len = seq_len(a.kv, a.lens, b, most);
    int first, n = seq_rows(a.kv, a.new_off, b, min(a.k.rows, a.v.rows), a.max_new, first);
    if (n > most - len || given != len) {
        if (n > most - len) report(a.kv, LASTRO_KV8_BAD_LENGTH);
        n = 0;
    }
    if (j == 0) {
        if (h == 0 && lane == 0) a.lens_out[b] = given + n;
        if (a.mass)
            for (int i = lane; i < n; i += 32) a.mass[((int64_t)b * H + h) * a.mass_stride + len + i] = 0.0f;
    }
    const int tail = len % kKv8Block;  // earlier rows of the first block
    if (n == 0 || j * kKv8Block >= tail + n) return;
    const int slot0 = len - tail + j * kKv8Block;  // the block's first slot
    const int page = page_of(a.kv, b, slot0);
    if (page < 0) return;
    const int beg = max(0, len - slot0), end = min(kKv8Block, len + n - slot0);  // its new rows
    const int64_t tile = (int64_t)page * H + h;
    const int64_t code0 = (tile * kKv8Page + slot0 % kKv8Page) * D, block = tile * kKv8Blocks + slot0 % kKv8Page / kKv8Block;
    const int r0 = lane / LPR, c = lane % LPR * 8;

    auto fetch = [&](const lastro_rows& src, Raw8<F32> (&x)[N]) {
        const bool vec = vec_rows(src);
        const int64_t base = (int64_t)(first + slot0 - len) * src.row_stride + h * src.head_stride + c;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = r0 + i * RPW;
            if (r >= beg && r < end)
                x[i].load(src, base + r * src.row_stride, vec);
            else
                x[i].zero();
        }
    };
    auto put = [&](uint8_t* codes, float* scale, float was, const Raw8<F32> (&x)[N]) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i].widest(m);
        float s = scale_for<FMT>(warp_umax(Raw8<F32>::f32_bits(m)));
        if (beg && (was != was || was > s)) s = was;  // earlier rows: the larger scale, and NaN stays
        const bool nan = s != s;
        const float inv = nan ? 0.0f : inverse(s);
        const bool again = beg && (nan || was != s);
        if (lane == 0) *scale = s;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = r0 + i * RPW;
            uint2* dst = reinterpret_cast<uint2*>(codes + r * D + c);
            if (r >= beg && r < end) {
                float v[8];
                x[i].values(v);
                uint2 o = make_uint2(0, 0);
                if (!nan) o = make_uint2(encode4<FMT>(v[0], v[1], v[2], v[3], inv), encode4<FMT>(v[4], v[5], v[6], v[7], inv));
                *dst = o;
            } else if (again && r < beg) {
                const uint2 w = *dst;
                float u[4], t[4];
                decode4<FMT>(w.x, u);
                decode4<FMT>(w.y, t);
                const float ratio = nan ? 0.0f : was * inv;
                *dst = make_uint2(encode4<FMT>(u[0], u[1], u[2], u[3], ratio), encode4<FMT>(t[0], t[1], t[2], t[3], ratio));
            }
        }
    };
    uint8_t *kc = static_cast<uint8_t*>(a.kv.k) + code0, *vc = static_cast<uint8_t*>(a.kv.v) + code0;
    const float kwas = a.kv.k_scale[block], vwas = a.kv.v_scale[block];
    Raw8<F32> x[N];
    if (F32) {  // K and V one after the other: both would not fit the registers
        fetch(a.k, x);
        put(kc, a.kv.k_scale + block, kwas, x);
        fetch(a.v, x);
        put(vc, a.kv.v_scale + block, vwas, x);
    } else {
        Raw8<F32> y[N];
        fetch(a.k, x);
        fetch(a.v, y);
        put(kc, a.kv.k_scale + block, kwas, x);
        put(vc, a.kv.v_scale + block, vwas, y);
    }
}

// ---- read-back ------------------------------------------------------------------------------------------------------
// One warp takes kReadSlots slots of a sequence, all heads: a lane turns 8 codes into 16 or 32 bytes, so that a warp's stores
// are whole lines (16 codes a lane, whose stores leave gaps for the next, ran at half the rate).  Bound by memory: 33 us for
// 8 x 4113 slots of 8 heads of 128, 28,747 of them held (194 MB, 5.9 TB/s, some of it still in L2).
constexpr int kReadSlots = 2;

template <int FMT, int D, bool F32>
__global__ void __launch_bounds__(256, 5) kv8_read_kernel(const __grid_constant__ Kv8ReadArgs a) {
    constexpr int LPR = D / 8, HPW = 32 / LPR;  // lanes a row, heads a pass
    pdl_wait();
    pdl_launch();
    const int lane = threadIdx.x & 31, H = a.kv.kv_heads, b = blockIdx.y;
    const int j0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kReadSlots;
    if (j0 >= a.n) return;
    const int len = seq_len(a.kv, a.lens, b, (int64_t)a.kv.max_pages * kKv8Page);
    const int64_t pos0 = (int64_t)a.pos0[b] + j0;
    int page[kReadSlots];
#pragma unroll
    for (int i = 0; i < kReadSlots; ++i)
        page[i] = j0 + i < a.n && pos0 + i >= 0 && pos0 + i < len ? page_of(a.kv, b, (int)(pos0 + i)) : -1;
    for (int h0 = 0; h0 < H; h0 += HPW) {
        const int h = h0 + lane / LPR, c = lane % LPR * 8;
        if (h >= H) continue;
        uint2 w[2][kReadSlots];
        float s[2][kReadSlots];
#pragma unroll
        for (int i = 0; i < kReadSlots; ++i) {
            const int row = (int)((pos0 + i) & (kKv8Page - 1));
            const int64_t tile = (int64_t)page[i] * H + h;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                w[v][i] = make_uint2(0, 0);
                s[v][i] = 0.0f;
                if (page[i] >= 0 && (v ? a.v_out : a.k_out)) {
                    w[v][i] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(v ? a.kv.v : a.kv.k) + (tile * kKv8Page + row) * D + c);
                    s[v][i] = (v ? a.kv.v_scale : a.kv.k_scale)[tile * kKv8Blocks + row / kKv8Block];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kReadSlots; ++i) {
            if (j0 + i >= a.n) break;
            const int64_t at = (((int64_t)b * a.n + j0 + i) * H + h) * D + c;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                void* out = v ? a.v_out : a.k_out;
                if (!out) continue;
                float x[4], y[4];
                decode4<FMT>(w[v][i].x, x);
                decode4<FMT>(w[v][i].y, y);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] *= s[v][i], y[k] *= s[v][i];
                if (F32) {
                    reinterpret_cast<float4*>(static_cast<float*>(out) + at)[0] = make_float4(x[0], x[1], x[2], x[3]);
                    reinterpret_cast<float4*>(static_cast<float*>(out) + at)[1] = make_float4(y[0], y[1], y[2], y[3]);
                } else {
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) =
                        make_uint4(two_bf16(x[0], x[1]), two_bf16(x[2], x[3]), two_bf16(y[0], y[1]), two_bf16(y[2], y[3]));
                }
            }
        }
    }
}

// ---- eviction -------------------------------------------------------------------------------------------------------
// masses as unsigned keys in their order: NaN above everything, -0 as +0
LDEV uint32_t mass_key(float m) {
    if (m != m) return 0xffffffffu;
    const uint32_t u = __float_as_uint(m + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

LDEV float key_mass(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr int kSelSlots = 16384;  // slots whose keys a CTA keeps in shared memory, after its histograms
constexpr int kSelBins = 4096;
// shared memory of a selection by clusters of `cl` CTAs, each with `keys` keys: the most where they are not given
constexpr size_t sel_smem(int cl, size_t keys = kSelSlots) { return (keys + (cl > 1 ? 3 : 1) * kSelBins) * sizeof(uint32_t); }

LDEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
LDEV uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// adds to a word of CTA `rank`'s shared memory, at the address `p` has in this one
LDEV void add_cluster(uint32_t* p, uint32_t rank, uint32_t v) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
// such a word
LDEV uint32_t ld_cluster(const uint32_t* p, uint32_t rank) {
    uint32_t a, v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

// One cluster of CL CTAs per sequence and KV head, each with an equal run of the slots that may be dropped, whose keys it
// holds in shared memory: the key of the (budget - recent)-th largest mass by three radix passes over histograms (12, 10 and
// 10 bits: masses share their leading bits, and 8-bit digits had most of them counted in a few words, one at a time), whose
// counts every CTA adds to all the others' (few are not zero).  Then one pass writes the kept slots in order, all above the
// key and of those at it the lowest: a warp takes consecutive slots and knows from counts what is kept before them.  Bound
// by its barriers and shared memory: 18 us for 64 x 8 heads of 3097 to 4097 slots (512 CTAs at once), 32 us for 2 x 8 of
// 123,153 and 131,072 (16 clusters), 6.4 us for 8 of 2049.
template <int CL>
__global__ void __launch_bounds__(CL > 1 ? 1024 : 512) kv8_select_kernel(const __grid_constant__ Kv8EvictArgs a) {
    constexpr int kSelThreads = CL > 1 ? 1024 : 512, kSelWarps = kSelThreads / 32;
    extern __shared__ uint32_t room[];
    // this CTA's counts; with a cluster, two arrays of everybody's besides, one cleared while the other is added to
    uint32_t *hist = room, *both = room + kSelBins, *keys = room + (CL > 1 ? 3 : 1) * kSelBins;
    __shared__ uint32_t part[kSelWarps], found[2], above[kSelWarps + 1], ties[kSelWarps + 1];
    pdl_wait();
    pdl_launch();
    const int H = a.src.kv_heads, b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, C = a.budget;
    const int lane = tid & 31, warp = tid >> 5, rank = CL > 1 ? (int)cluster_rank() : 0, all = CL * kSelThreads, me = rank * kSelThreads + tid;
    int64_t most = (int64_t)a.src.max_pages * kKv8Page;
    if (a.mass) most = min(most, a.mass_stride);
    const int len = seq_len(a.src, a.lens, b, most);
    const int64_t seq = (int64_t)b * H + h;
    int32_t* kept = a.kept + seq * C;
    const float* mass = a.mass ? a.mass + seq * a.mass_stride : nullptr;
    float* mout = a.mass_out ? a.mass_out + seq * a.mass_out_stride : nullptr;
    const int keep = min(len, C);
    if (h == 0 && me == 0) a.lens_out[b] = keep;
    for (int i = keep + me; i < C; i += all) kept[i] = -1;
    // the slots kept whatever their mass: all, or the last `recent`
    const int want = len <= C ? 0 : C - a.recent, cand = len <= C ? 0 : len - a.recent;
    for (int i = me; i < keep - want; i += all) {
        kept[want + i] = cand + i;
        if (mout) mout[want + i] = mass[cand + i];
    }
    if (want == 0) return;  // the same for the whole cluster

    const int run = ((cand + CL - 1) / CL + 3) & ~3, lo = min(cand, rank * run), n = min(cand, lo + run) - lo;
    // the keys, four at a time; 0, which is no mass's key and below them all, past the last
    const bool held = run <= kSelSlots, vec = (reinterpret_cast<uintptr_t>(mass) & 15) == 0;
    const int n4 = (n + 3) / 4;
    auto fetch = [&](int i) {
        const float* p = mass + lo + 4 * i;
        if (vec && 4 * i + 4 <= n) {
            const float4 m = *reinterpret_cast<const float4*>(p);
            return make_uint4(mass_key(m.x), mass_key(m.y), mass_key(m.z), mass_key(m.w));
        }
        uint32_t k[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) k[q] = 4 * i + q < n ? mass_key(p[q]) : 0u;
        return make_uint4(k[0], k[1], k[2], k[3]);
    };
    if (held) {
#pragma unroll 4
        for (int i = tid; i < n4; i += kSelThreads) reinterpret_cast<uint4*>(keys)[i] = fetch(i);
    }
    auto four = [&](int i, uint32_t (&k)[4]) {
        const uint4 v = held ? reinterpret_cast<const uint4*>(keys)[i] : fetch(i);
        k[0] = v.x, k[1] = v.y, k[2] = v.z, k[3] = v.w;
    };
    if (CL > 1) {
        for (int i = tid; i < kSelBins; i += kSelThreads) both[i] = 0;
        cluster_sync();
    }
    uint32_t prefix = 0, need = want;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 20 : pass == 1 ? 10 : 0, bins = pass == 0 ? kSelBins : 1024;
        const uint32_t* total = CL > 1 ? both + (pass & 1) * kSelBins : hist;
        for (int i = tid; i < bins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xfff00000u : 0xfffffc00u;
#pragma unroll 2
        for (int i = tid; i < n4; i += kSelThreads) {
            uint32_t k[4];
            four(i, k);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if ((k[q] & mask) == prefix) atomicAdd(&hist[(k[q] >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        if (CL > 1) {
            uint32_t* next = both + (~pass & 1) * kSelBins;
            for (int i = tid; i < bins; i += kSelThreads) {
                const uint32_t c = hist[i];
                if (c)
                    for (int r = 0; r < CL; ++r) add_cluster(both + (pass & 1) * kSelBins + i, r, c);
            }
            for (int i = tid; i < 1024; i += kSelThreads) next[i] = 0;  // the later passes' bins
            cluster_sync();
        }
        // thread t's digits, from the largest down: bins - 1 - per t and the per - 1 below it
        const int per = max(1, bins / kSelThreads);
        uint32_t c[kSelBins / kSelThreads], sum = 0;
#pragma unroll
        for (int i = 0; i < kSelBins / kSelThreads; ++i) {
            const int d = bins - 1 - (tid * per + i);
            c[i] = i < per && d >= 0 ? total[d] : 0u;
            sum += c[i];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        if (lane == 31) part[warp] = incl;
        __syncthreads();
        uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? part[lane & (kSelWarps - 1)] : 0u) + incl - sum;
        if (before < need && need <= before + sum) {  // one thread: the digit that the last wanted slot has
            bool done = false;
#pragma unroll
            for (int i = 0; i < kSelBins / kSelThreads; ++i) {
                if (!done && before + c[i] >= need) {
                    found[0] = prefix | (uint32_t)(bins - 1 - (tid * per + i)) << shift;
                    found[1] = need - before;
                    done = true;
                }
                if (!done) before += c[i];
            }
        }
        __syncthreads();
        prefix = found[0];
        need = found[1];
    }
    // kept: every key above prefix, and the first `need` at it
    const int span = (n4 + kSelWarps - 1) / kSelWarps, wlo = min(n4, warp * span), whi = min(n4, wlo + span);
    uint32_t up = 0, at = 0;
    for (int i = wlo + lane; i < whi; i += 32) {
        uint32_t k[4];
        four(i, k);
#pragma unroll
        for (int q = 0; q < 4; ++q) up += k[q] > prefix, at += k[q] == prefix;
    }
    up = __reduce_add_sync(0xffffffffu, up);
    at = __reduce_add_sync(0xffffffffu, at);
    if (lane == 0) above[warp] = up, ties[warp] = at;
    __syncthreads();
    // what is kept before this warp's slots: in the CTA's earlier warps, and in the cluster's earlier CTAs
    const uint32_t wu = lane < kSelWarps ? above[lane] : 0u, wt = lane < kSelWarps ? ties[lane] : 0u;
    up = __reduce_add_sync(0xffffffffu, lane < warp ? wu : 0u);
    at = __reduce_add_sync(0xffffffffu, lane < warp ? wt : 0u);
    if (CL > 1) {
        const uint32_t u = __reduce_add_sync(0xffffffffu, wu), t = __reduce_add_sync(0xffffffffu, wt);
        if (tid == 0) above[kSelWarps] = u, ties[kSelWarps] = t;
        cluster_sync();
        up += __reduce_add_sync(0xffffffffu, lane < rank ? ld_cluster(&above[kSelWarps], lane) : 0u);
        at += __reduce_add_sync(0xffffffffu, lane < rank ? ld_cluster(&ties[kSelWarps], lane) : 0u);
    }
    for (int i0 = wlo; i0 < whi; i0 += 32) {
        const int i = i0 + lane;
        uint32_t k[4] = {}, mine = 0;  // keys above prefix in the low half, at it in the high half
        if (i < whi) four(i, k);
#pragma unroll
        for (int q = 0; q < 4; ++q) mine += (k[q] > prefix) + (k[q] == prefix ? 0x10000u : 0u);
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        uint32_t u = up + ((incl - mine) & 0xffffu), t = at + ((incl - mine) >> 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (k[q] > prefix || (k[q] == prefix && t < need)) {
                const uint32_t pos = u + min(t, need);
                kept[pos] = lo + 4 * i + q;
                if (mout) mout[pos] = key_mass(k[q]);
            }
            u += k[q] > prefix;
            t += k[q] == prefix;
        }
        const uint32_t all32 = __shfl_sync(0xffffffffu, incl, 31);
        up += all32 & 0xffffu;
        at += all32 >> 16;
    }
    if (CL > 1) cluster_sync();  // no CTA leaves while another reads its counts
}

// and back: two f16 pairs to the nearest codes (what they were multiplied by keeps them in the format's range)
template <int FMT>
LDEV uint32_t from_f16(uint32_t lo, uint32_t hi) {
    if (FMT == E4M3) {
        uint16_t a, b;
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(a) : "r"(lo));
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(b) : "r"(hi));
        return a | (uint32_t)b << 16;
    }
    uint32_t a, b;  // 1536 + x rounds x to a whole number, whose low byte is the f16's
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(a) : "r"(lo), "r"(0x66006600u));
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(b) : "r"(hi), "r"(0x66006600u));
    return __byte_perm(a, b, 0x6420);
}
LDEV uint32_t mul_f16(uint32_t x, uint32_t y) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
    return r;
}

// 16 bytes of a row whose neighbours are as likely dropped as kept: no more than its 64 bytes are fetched
LDEV uint4 ld_row(const uint8_t* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.L2::64B.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
    return r;
}

// One warp gathers kGatherBlocks destination blocks of K and V of one head: their kept rows as 16-byte pieces, all on
// their way before the first is used (a row takes three dependent loads: the slot kept, its page, the codes), then for each
// block the largest magnitude, the new scale, and the codes times a ratio of powers of two, in f16 (a code has at most 8
// significant bits).  Bound by memory, each kept row read and written once: 36 us for 64 x 8 heads x 1000 rows of 64 (131 MB,
// 3.7 TB/s: single 64-byte rows, fetched as such, do not come at the rate of whole lines).
constexpr int kGatherBlocks = 2;

template <int FMT, int D>
__global__ void __launch_bounds__(256, D == 64 ? 4 : 2) kv8_gather_kernel(const __grid_constant__ Kv8EvictArgs a) {
    constexpr int LPR = D / 16, RPW = 32 / LPR, N = kKv8Block / RPW;  // lanes a row, rows a pass, passes
    static_assert(kGatherBlocks * kKv8Block == 32, "a lane for each row");
    pdl_wait();
    pdl_launch();
    const int lane = threadIdx.x & 31, H = a.src.kv_heads, h = blockIdx.y, b = blockIdx.z;
    const int slot0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * 32;
    const int keep = a.lens_out[b];
    if (slot0 >= keep) return;
    const int dpage = page_of(a.dst, b, slot0);  // both blocks are in one page
    // lane r: where kept row r is, and its scales
    int64_t from = -1;
    float ks = 0.0f, vs = 0.0f;
    if (slot0 + lane < keep) {
        const int t = a.kept[((int64_t)b * H + h) * a.budget + slot0 + lane], page = page_of(a.src, b, t);
        if (page >= 0) {
            const int64_t tile = (int64_t)page * H + h;
            from = tile * kKv8Page + t % kKv8Page;
            ks = a.src.k_scale[tile * kKv8Blocks + t % kKv8Page / kKv8Block];
            vs = a.src.v_scale[tile * kKv8Blocks + t % kKv8Page / kKv8Block];
        }
    }
    if (dpage < 0) return;
    const int r0 = lane / LPR, c = lane % LPR * 16;
    uint4 w[kGatherBlocks][2][N];
#pragma unroll
    for (int g = 0; g < kGatherBlocks; ++g)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t row = __shfl_sync(0xffffffffu, from, g * kKv8Block + r0 + i * RPW);
            w[g][0][i] = w[g][1][i] = make_uint4(0, 0, 0, 0);
            if (row >= 0) {
                w[g][0][i] = ld_row(static_cast<const uint8_t*>(a.src.k) + row * D + c);
                w[g][1][i] = ld_row(static_cast<const uint8_t*>(a.src.v) + row * D + c);
            }
        }
    const int64_t tile = (int64_t)dpage * H + h;
#pragma unroll
    for (int g = 0; g < kGatherBlocks; ++g) {
        const int first = slot0 + g * kKv8Block;
        if (first >= keep) return;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            uint32_t f[N][8], amax = 0;
            float sc[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                sc[i] = __shfl_sync(0xffffffffu, v ? vs : ks, g * kKv8Block + r0 + i * RPW);
                widen<FMT>(w[g][v][i].x, f[i][0], f[i][1]);
                widen<FMT>(w[g][v][i].y, f[i][2], f[i][3]);
                widen<FMT>(w[g][v][i].z, f[i][4], f[i][5]);
                widen<FMT>(w[g][v][i].w, f[i][6], f[i][7]);
                uint32_t m = 0;  // magnitudes, ordered as their bits
#pragma unroll
                for (int q = 0; q < 8; ++q) m = __vmaxu2(m, f[i][q] & 0x7fff7fffu);
                const float top = __half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))) * sc[i];
                amax = max(amax, __float_as_uint(top) & 0x7fffffffu);
            }
            const float s = scale_for<FMT>(warp_umax(amax));
            const bool nan = s != s;
            const float inv = nan ? 0.0f : inverse(s);
            if (lane == 0) (v ? a.dst.v_scale : a.dst.k_scale)[tile * kKv8Blocks + first % kKv8Page / kKv8Block] = s;
            uint8_t* dst = static_cast<uint8_t*>(v ? a.dst.v : a.dst.k) + (tile * kKv8Page + first % kKv8Page) * D + c;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = r0 + i * RPW;
                // the ratio can pass f16's range where every code is small (2^17 for e4m3): then in two steps
                float ratio = nan ? 0.0f : sc[i] * inv;
                if (__any_sync(0xffffffffu, ratio > 16384.0f)) {
                    const float part = fminf(ratio, 16384.0f);
                    ratio = part > 0.0f ? fminf(ratio / part, 16384.0f) : 0.0f;
                    const uint32_t p = __half_as_ushort(__float2half_rn(part)) * 0x10001u;
#pragma unroll
                    for (int q = 0; q < 8; ++q) f[i][q] = mul_f16(f[i][q], p);
                }
                const uint32_t p = __half_as_ushort(__float2half_rn(ratio)) * 0x10001u;
#pragma unroll
                for (int q = 0; q < 8; ++q) f[i][q] = mul_f16(f[i][q], p);
                if (first + r < keep)
                    *reinterpret_cast<uint4*>(dst + r * D) = make_uint4(from_f16<FMT>(f[i][0], f[i][1]), from_f16<FMT>(f[i][2], f[i][3]),
                                                                        from_f16<FMT>(f[i][4], f[i][5]), from_f16<FMT>(f[i][6], f[i][7]));
            }
        }
    }
}

// ---- variants -------------------------------------------------------------------------------------------------------
unsigned int blocks_of(int64_t units, int per) { return (unsigned int)((units + per - 1) / per); }

struct AppendLaunch {
    const Kv8AppendArgs& a;
    cudaStream_t s;
    template <int FMT, int D>
    cudaError_t run() {
        const dim3 grid(blocks_of((int64_t)a.blocks * a.kv.kv_heads, 8), a.kv.n_seqs);
        if (a.k.dtype == LASTRO_DTYPE_F32) return kv8_launch<kv8_append_kernel<FMT, D, true>, 0>(grid, 256, 0, 1, s, a);
        return kv8_launch<kv8_append_kernel<FMT, D, false>, 0>(grid, 256, 0, 1, s, a);
    }
};

struct ReadLaunch {
    const Kv8ReadArgs& a;
    cudaStream_t s;
    template <int FMT, int D>
    cudaError_t run() {
        const dim3 grid(blocks_of(a.n, 8 * kReadSlots), a.kv.n_seqs);
        if (a.f32) return kv8_launch<kv8_read_kernel<FMT, D, true>, 0>(grid, 256, 0, 1, s, a);
        return kv8_launch<kv8_read_kernel<FMT, D, false>, 0>(grid, 256, 0, 1, s, a);
    }
};

struct EvictLaunch {
    const Kv8EvictArgs& a;
    cudaStream_t s;
    template <int FMT, int D>
    cudaError_t run() {
        // a cluster where one CTA's shared memory might not hold the keys
        const int64_t slots = (int64_t)a.src.max_pages * kKv8Page;
        const int cl = slots > kSelSlots ? 8 : 1;
        const size_t keys = (size_t)min(((slots + cl - 1) / cl + 3) & ~(int64_t)3, (int64_t)kSelSlots);
        const size_t smem = sel_smem(cl, keys);
        const dim3 grid(cl, a.src.kv_heads, a.src.n_seqs);
        const cudaError_t e = cl > 1 ? kv8_launch<kv8_select_kernel<8>, sel_smem(8)>(grid, 1024, smem, 8, s, a)
                                     : kv8_launch<kv8_select_kernel<1>, sel_smem(1)>(grid, 512, smem, 1, s, a);
        if (e != cudaSuccess) return e;
        const dim3 blocks(blocks_of(a.budget, 8 * 32), a.src.kv_heads, a.src.n_seqs);
        return kv8_launch<kv8_gather_kernel<FMT, D>, 0>(blocks, 256, 0, 1, s, a);
    }
};

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t s) { return kv8_by_shape(a.kv, AppendLaunch{a, s}); }
cudaError_t launch_kv8_evict(const Kv8EvictArgs& a, cudaStream_t s) { return kv8_by_shape(a.src, EvictLaunch{a, s}); }
cudaError_t launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t s) { return kv8_by_shape(a.kv, ReadLaunch{a, s}); }

}  // namespace lastro
