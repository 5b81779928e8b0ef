// Attention over the 8-bit KV cache (lastro_kv8_attend): scores, softmax and weighted sum in one pass over the cache, the
// weights every slot received in a second pass over K.
//
// A KV head's query rows (its group's heads times the sequence's queries) are the M side of m16n8k16 matrix products:
// S = Q K^T with a block's 16 slots as two n-tiles, O += P V with the 16 slots as one k-step.  Codes go from shared memory
// to operand registers and are widened to f16 there, which holds every e4m3 and int8 value exactly; the scales, powers of
// two, are applied to the scores (K) and to the weights (V) in f32.
#include <cuda_runtime.h>

#include <type_traits>

#include "kv8.cuh"

namespace lastro {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;  // of the merge and weight kernels
constexpr int kChunkBytes = 4096;                  // K codes a warp of the weight kernel takes at a time
constexpr float kFar = -1e30f;                        // below every score: the running maxima's start

LDEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^e for an integer-valued e, 0 below the normal range, 2^127 above it
LDEV float pow2i(float e) {
    const int i = (int)fminf(fmaxf(e, -127.0f), 127.0f) + 127;
    return __uint_as_float((uint32_t)i << 23);
}

// d (+)= a (16x16, row) * b (16x8, col), f16 operands, f32 accumulators.  NE is the number of row halves that hold rows: 2,
// or 1 when rows 8..15 are empty and their operands zeros.  Operands are ordered [k half][row half], results [row half]
// [column].
template <int NE>
LDEV void mma_f16(float (&d)[4], const uint32_t (&a)[2 * NE], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(NE == 2 ? a[NE - 1] : 0u), "r"(a[NE]), "r"(NE == 2 ? a[2 * NE - 1] : 0u), "r"(b0), "r"(b1));
}
template <int NE>
LDEV void mma_f16_new(float (&d)[4], const uint32_t (&a)[2 * NE], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(NE == 2 ? a[NE - 1] : 0u), "r"(a[NE]), "r"(NE == 2 ? a[2 * NE - 1] : 0u), "r"(b0), "r"(b1), "f"(0.0f));
}

// the smaller, NaN if either is
LDEV float min_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// four codes to two f16 pairs, exactly
template <int FMT>
LDEV void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (FMT == E4M3) {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)w));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
    } else {  // f16 0x6400 + u is 1024 + u for a byte u = code + 128
        const uint32_t u = w ^ 0x80808080u, bias = 0x64806480u;  // 1152 twice
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(bias));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(bias));
    }
}

LDEV uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// what pack_f16 rounded away, as f16
LDEV uint32_t rest_f16(uint32_t packed, float lo, float hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    return pack_f16(lo - f.x, hi - f.y);
}

LDEV void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// The block's slot that n-tile `j`, column 2 * pair + e stands for, and that the PV product takes as k index
// 2 * pair + e + 8 * j.  Any bijection is right; this one spreads the rows that one shared-memory access reads over
// both halves of a 128-byte line.
LDEV int slot_of(int pair, int e, int j) { return j * 8 + e * 4 + (pair & 2) + ((pair & 1) ^ e); }

// ---- the list of work -------------------------------------------------------------------------------------------------
// Every sequence with queries contributes kv_heads * row tiles * chunks items, chunks innermost; equal consecutive shares
// of the whole list go to the groups of warps, so that ragged lengths balance to within one chunk.
struct Seq {
    int len, n, first;  // slots, queries, first query row
    int chunks, tiles;  // of one unit (head and row tile); row tiles of 16 * RW rows
};

template <int TOK>
LDEV Seq seq_of(const Kv8AttendArgs& a, int b, int tile_rows) {
    Seq s;
    int64_t most = (int64_t)a.kv.max_pages * kKv8Page;
    if (a.mass_out) most = min(most, a.mass_stride);
    s.len = seq_len(a.kv, a.lens, b, most);
    s.n = seq_rows(a.kv, a.q_off, b, a.q.rows, a.max_new, s.first);
    s.chunks = max(1, (s.len + TOK - 1) / TOK);  // a query of an empty sequence still gets its zeros
    s.tiles = (int)(((int64_t)s.n * a.group + tile_rows - 1) / tile_rows);
    return s;
}

// items of one share when `total` are dealt to n shares
LDEV int share_of(int total, int n) { return (int)(((unsigned)total + n - 1) / n); }

// The list as a warp sees it: lane l's own sequences l, l + 32, ... and their numbers of items, the first four of them
// kept in registers (128 sequences are read once), the length of the list, and the sequence that holds an item.
template <typename Work>
struct List {
    int n_seqs, total, w[4];
    const Work& work;
    LDEV List(int n, const Work& f) : n_seqs(n), work(f) {
        const int lane = threadIdx.x & 31;
        int sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = lane + 32 * i < n ? work(lane + 32 * i) : 0;
            sum += w[i];
        }
        for (int b = lane + 128; b < n; b += 32) sum += work(b);
        total = (int)__reduce_add_sync(0xffffffffu, (unsigned)sum);
    }
    // the sequence with item `pos` and where its items start (-1 when the list ends before it); `note(b, at)` is told
    // where each sequence up to there starts, all of them with `all`
    template <typename Note>
    LDEV int seek(int pos, bool all, int& base, Note note) const {
        const int lane = threadIdx.x & 31;
        int found = -1, sum = 0;
        auto step = [&](int b0, int n) {
            int x = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const int at = sum + x - n;
            if (b0 + lane < n_seqs) note(b0 + lane, at);
            const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && at <= pos && pos < at + n);
            if (hit) {
                found = b0 + __ffs(hit) - 1;
                base = __shfl_sync(0xffffffffu, at, __ffs(hit) - 1);
            }
            sum += __shfl_sync(0xffffffffu, x, 31);
        };
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (32 * i < n_seqs && (all || found < 0)) step(32 * i, w[i]);
        for (int b0 = 128; b0 < n_seqs && (all || found < 0); b0 += 32) step(b0, b0 + lane < n_seqs ? work(b0 + lane) : 0);
        return found;
    }
};

// ---- query rows ---------------------------------------------------------------------------------------------------------
// The A operand of 16 rows (row r is query r / group, head r % group of the KV head) and each row's factor from the raw
// product to the score in powers of two.  A row is scaled by a power of two to a largest magnitude in [2^14, 2^15), which
// puts a bf16 value exactly into f16 down to 2^-28 of that magnitude; f32 rows take a second term.
template <int D, int NE, bool F32>
struct QFrag {
    static constexpr int KS = D / 16;
    uint32_t hi[KS][2 * NE], lo[F32 ? KS : 1][2 * NE];
    float factor[NE];

    LDEV void load(const Kv8AttendArgs& a, const Seq& s, int h, int row0, bool vec, int lane) {
        const int gq = lane >> 2, c = lane & 3;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int r = row0 + gq + 8 * e;
            float x[D / 64][16];
            uint32_t amax = 0;
#pragma unroll
            for (int hf = 0; hf < D / 64; ++hf) {
                if (r < s.n * a.group) {
                    const int64_t at = (int64_t)(s.first + r / a.group) * a.q.row_stride +
                                       (int64_t)(h * a.group + r % a.group) * a.q.head_stride + hf * 64 + 16 * c;
                    float (&u)[8] = *reinterpret_cast<float (*)[8]>(&x[hf][0]);
                    float (&w)[8] = *reinterpret_cast<float (*)[8]>(&x[hf][8]);
                    load8(a.q, at, vec, u);
                    load8(a.q, at + 8, vec, w);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[hf][i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) amax = max(amax, __float_as_uint(x[hf][i]) & 0x7fffffffu);
            }
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int k = min(126, 141 - (int)(amax >> 23));  // 14 - exponent
            const bool finite = amax < 0x7f800000u;
            // the factor is kept positive, so that the largest product is the largest score
            const float up = finite ? copysignf(__uint_as_float((uint32_t)(k + 127) << 23), a.scale) : 0.0f;
            factor[e] = finite ? fabsf(a.scale) * 1.44269504088896340736f * __uint_as_float((uint32_t)(127 - k) << 23)
                               : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int hf = 0; hf < D / 64; ++hf)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float u = finite ? x[hf][4 * q + 2 * w] * up : 0.0f;
                        const float v = finite ? x[hf][4 * q + 2 * w + 1] * up : 0.0f;
                        hi[hf * 4 + q][w * NE + e] = pack_f16(u, v);
                        if (F32) lo[F32 ? hf * 4 + q : 0][w * NE + e] = rest_f16(hi[hf * 4 + q][w * NE + e], u, v);
                    }
        }
    }
};

// slots that row r of the sequence sees
LDEV int visible(const Kv8AttendArgs& a, const Seq& s, int r) {
    return s.len - s.n + min(r, s.n * a.group - 1) / a.group + 1;
}

// the codes of slot row `row` that this lane feeds to the score product: 16 bytes of every 64
template <int D>
LDEV void k_codes(const uint8_t* row, int lane, uint32_t (&w)[D / 16]) {
    const uint8_t* p = row + 16 * (lane & 3);
    const uint4 a = *reinterpret_cast<const uint4*>(p + (D == 128 && (lane & 4) ? 64 : 0));
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    if (D == 128) {  // odd rows read their halves in the other order: two rows of a line's banks per access
        const uint4 b = *reinterpret_cast<const uint4*>(p + (lane & 4 ? 0 : 64));
        const bool odd = lane & 4;
        w[D / 16 - 4] = odd ? a.x : b.x, w[D / 16 - 3] = odd ? a.y : b.y;
        w[D / 16 - 2] = odd ? a.z : b.z, w[D / 16 - 1] = odd ? a.w : b.w;
        w[0] = odd ? b.x : a.x, w[1] = odd ? b.y : a.y, w[2] = odd ? b.z : a.z, w[3] = odd ? b.w : a.w;
    }
}

// One n-tile of scores.  The matrix unit truncates what it adds to an f32 accumulator, so f32 rows take their second term
// first, while the sum is small, and no more than two steps a chain; the chains are added with rounding.
template <int D, int NE, bool F32>
LDEV void score_tile(const QFrag<D, NE, F32>& q, const uint32_t (&b)[D / 16][2], float (&s)[2 * NE]) {
    constexpr int KS = D / 16, CH = F32 ? 2 : KS;
#pragma unroll
    for (int k0 = 0; k0 < KS; k0 += CH) {
        float x[4];
#pragma unroll
        for (int k = k0; F32 && k < k0 + CH; ++k)
            if (k == k0)
                mma_f16_new<NE>(x, q.lo[F32 ? k : 0], b[k][0], b[k][1]);
            else
                mma_f16<NE>(x, q.lo[F32 ? k : 0], b[k][0], b[k][1]);
#pragma unroll
        for (int k = k0; k < k0 + CH; ++k)
            if (!F32 && k == k0)
                mma_f16_new<NE>(x, q.hi[k], b[k][0], b[k][1]);
            else
                mma_f16<NE>(x, q.hi[k], b[k][0], b[k][1]);
#pragma unroll
        for (int i = 0; i < 2 * NE; ++i) s[i] = k0 == 0 ? x[i] : s[i] + x[i];
    }
}

// ---- partial results ----------------------------------------------------------------------------------------------------
// A share that holds a part of a unit leaves that part's sums: in its slot 0 when the unit began in an earlier share, in
// its slot 1 when it began in this one and goes on in the next.
constexpr int part_floats(int D) { return D + 4; }  // sums, then the running maxima M and R and the sum l

// A row's running state: M the ceiling of the largest score so far (scores and M in powers of two), l the sum of
// 2^(score - M), R the ceiling of the largest score plus its slot's V exponent, o the sum of 2^(score + 14 - R) v.  M
// and R are whole numbers, so bringing sums to new ones is exact, and R keeps the f16 weights in range whatever the
// blocks' scales: the heaviest contribution sits between 2^13 and 2^14.
template <int D, int NE, bool F32>
LDEV void store_row(const Kv8AttendArgs& a, const Seq& s, int h, int r, int lane, const float (&o)[D / 8][4], int e,
                    float M, float R, float l, bool vec) {
    const int c = lane & 3, t = s.first + r / a.group, hq = h * a.group + r % a.group;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l, up = pow2i(R - 14.0f - M);
#pragma unroll
    for (int hf = 0; hf < D / 64; ++hf) {
        const int64_t at = (int64_t)t * a.out.row_stride + (int64_t)hq * a.out.head_stride + hf * 64 + 16 * c;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = l == 0.0f ? 0.0f : o[hf * 8 + (i & 7)][2 * e + (i >> 3)] * inv * up;
        if (F32) {
            float* dst = static_cast<float*>(a.out.ptr) + at;
            if (vec) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    reinterpret_cast<float4*>(dst)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) dst[i] = v[i];
            }
        } else {
            uint16_t* dst = static_cast<uint16_t*>(a.out.ptr) + at;
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = pack_bf16(f32_to_bf16_rne(v[2 * i]), f32_to_bf16_rne(v[2 * i + 1]));
            if (vec) {
                reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) dst[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
            }
        }
    }
    if (a.lse && c == 0) a.lse[(int64_t)t * a.heads + hq] = l == 0.0f ? INFINITY : M + log2f(l);
}

// The parts of one row, `n` (at most 32) of them at at(0), at(1), ..., added to a warp's running sums.
template <int D, typename At>
LDEV void add_parts(int n, At at, float (&o)[D / 32], float& M, float& R, float& l) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    float4 m = make_float4(kFar, kFar, 0.0f, 0.0f);
    if (lane < n) m = *reinterpret_cast<const float4*>(at(lane) + D);
    float Mn = fmaxf(M, m.x), Rn = fmaxf(R, m.y);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
        Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, x));
        Rn = fmaxf(Rn, __shfl_xor_sync(0xffffffffu, Rn, x));
    }
    l = l * pow2i(M - Mn) + warp_sum(m.z * pow2i(m.x - Mn));
    const float old = pow2i(R - Rn), mine = pow2i(m.y - Rn);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] *= old;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
        const float f = __shfl_sync(0xffffffffu, mine, i);
        if (V == 2) {
            const float2 x = reinterpret_cast<const float2*>(at(i))[lane];
            o[0] += x.x * f, o[1] += x.y * f;
        } else {
            const float4 x = reinterpret_cast<const float4*>(at(i))[lane];
            o[0] += x.x * f, o[1] += x.y * f, o[V - 2] += x.z * f, o[V - 1] += x.w * f;
        }
    }
    M = Mn;
    R = Rn;
}

// the merged row to the output: lane l holds D / 32 consecutive values
template <int D, bool F32>
LDEV void store_merged(const Kv8AttendArgs& a, int first, int h, int r, const float (&o)[D / 32], float M, float R, float l) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31, t = first + r / a.group, hq = h * a.group + r % a.group;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l, up = pow2i(R - 14.0f - M);
    const int64_t at = (int64_t)t * a.out.row_stride + (int64_t)hq * a.out.head_stride + lane * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float v = l == 0.0f ? 0.0f : o[e] * inv * up;
        if (F32)
            static_cast<float*>(a.out.ptr)[at + e] = v;
        else
            static_cast<uint16_t*>(a.out.ptr)[at + e] = f32_to_bf16_rne(v);
    }
    if (a.lse && lane == 0) a.lse[(int64_t)t * a.heads + hq] = l == 0.0f ? INFINITY : M + log2f(l);
}

// ---- one pass over the cache ----------------------------------------------------------------------------------------------
// A group of RW warps (RW * 16 query rows) walks its share of the list through its own ring of stages, each 4 KB of K and
// of V codes and their scales brought in by bulk copies; its first warp's lane 0 issues them.  With one warp a group
// (RW 1) the CTA takes one share, its warps equal parts of it in order, and puts together at its end what they cut.
template <int D, int RW, int NE>
struct Ring {
    static constexpr int GROUPS = 8 / RW, TOK = kChunkBytes / D;
    static constexpr int STAGES = RW == 1 ? (NE == 1 ? 3 : 2) : RW == 2 ? 6 : 8;
    // RW 1: each warp's part of a unit that began before it, kept to the end (that of one it leaves open goes to its ring)
    static constexpr size_t head = RW == 1 ? (size_t)8 * NE * part_floats(D) * sizeof(float) : 0;
    static constexpr size_t bytes = (size_t)GROUPS * (STAGES * (2 * kChunkBytes + 8 * sizeof(float) + (RW == 1 ? 8 : 16) + 4) + head);
};
constexpr int ring_tok(int D) { return kChunkBytes / D; }

// what a warp of a CTA with one warp a group leaves behind
struct Ends {
    bool mid, closes, tail;  // its part began inside a unit; ended it; ended inside a unit that it began
    int hh, ht, hn, hfirst;  // KV head, row tile, queries and first query row of the one it began inside
    int th, tt, tn, tfirst;  // and of the one it left open
};

template <int FMT, int D, int RW, int NE, bool F32>
__global__ void __launch_bounds__(kThreads, 1) kv8_attend_kernel(const __grid_constant__ Kv8AttendArgs a) {
    using RG = Ring<D, RW, NE>;
    constexpr int TOK = RG::TOK, NB = TOK / kKv8Block, ST = RG::STAGES, CPP = kKv8Page / TOK, kStageBytes = 2 * kChunkBytes;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Ends ends[RW == 1 ? kWarps : 1];
    pdl_wait();
    pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, c4 = lane & 3;
    const int wg = warp / RW, wrow = warp % RW;
    unsigned char* data = smem + (size_t)wg * ST * kStageBytes;
    unsigned char* tail = smem + (size_t)RG::GROUPS * ST * kStageBytes;
    float* scales = reinterpret_cast<float*>(tail) + wg * ST * 8;
    uint64_t* bars = reinterpret_cast<uint64_t*>(tail + (size_t)RG::GROUPS * ST * 8 * sizeof(float));
    constexpr int BARS = RW == 1 ? 1 : 2;  // a warp on its own needs no barrier to hand stages back
    uint64_t *full = bars + wg * ST, *empty = bars + ((BARS - 1) * RG::GROUPS + wg) * ST;
    int* flags = reinterpret_cast<int*>(bars + BARS * RG::GROUPS * ST);
    int* there = flags + wg * ST;
    float* heads = reinterpret_cast<float*>(flags + RG::GROUPS * ST);
    if (wrow == 0 && lane == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(full + i, 1);
            if (RW > 1) mbar_init(empty + i, RW);
        }
        if (RW == 1) ends[warp].mid = ends[warp].tail = false;
    }
    if (RW == 1)
        __syncwarp();
    else
        __syncthreads();

    // this group's part [beg, end) of the list; the list's offset of each sequence goes to the merge kernel
    const int H = a.kv.kv_heads, tile_rows = 16 * RW;
    const auto work = [&](int b) {
        const Seq s = seq_of<TOK>(a, b, tile_rows);
        return H * s.tiles * s.chunks;
    };
    const List<decltype(work)> list(a.kv.n_seqs, work);
    int beg, end;
    if (RW == 1) {
        const int per = share_of(list.total, gridDim.x), lo = min(list.total, (int)blockIdx.x * per), hi = min(list.total, lo + per);
        const int each = share_of(hi - lo, kWarps);
        beg = min(hi, lo + warp * each), end = min(hi, beg + each);
    } else {  // groups of one CTA are far apart in the list, so that a short one still uses every SM
        const int per = share_of(list.total, gridDim.x * RG::GROUPS);
        beg = min(list.total, (wg * (int)gridDim.x + (int)blockIdx.x) * per), end = min(list.total, beg + per);
    }
    const int group = RW == 1 ? (int)blockIdx.x * kWarps + warp : wg * (int)gridDim.x + (int)blockIdx.x;
    const bool writes = blockIdx.x == 0 && warp == 0;
    int sbase = 0;
    const int sb = list.seek(beg, writes, sbase, [&](int b, int at) {
        if (writes) a.offset[b] = at;
    });
    if (writes && lane == 0) a.offset[a.kv.n_seqs] = list.total;
    const int count = end - beg;
    if (RW > 1 && count == 0) return;
    const bool vo = vec_rows(a.out);
    if (count > 0) {
    struct Cursor {
        int b, h, tile, c;
        Seq s;
    } cur, iss;
    cur.b = sb;
    cur.s = seq_of<TOK>(a, sb, tile_rows);
    {
        const int u = beg - sbase, v = u / cur.s.chunks;
        cur.c = u - v * cur.s.chunks;
        cur.h = v / cur.s.tiles;
        cur.tile = v - cur.h * cur.s.tiles;
    }
    iss = cur;
    auto advance = [&](Cursor& x) {
        if (++x.c < x.s.chunks) return;
        x.c = 0;
        if (++x.tile < x.s.tiles) return;
        x.tile = 0;
        if (++x.h < H) return;
        x.h = 0;
        do {
            if (++x.b >= a.kv.n_seqs) return;
            x.s = seq_of<TOK>(a, x.b, tile_rows);
        } while (x.s.tiles == 0);
    };

    // page numbers ahead of the issuing cursor: lane i holds page pbase + i of sequence pb
    int pb = -1, pbase = 0, pnum = 0;
    int seen = 0;  // chunks of the issuing cursor's unit that any of its rows sees
    auto limit = [&]() {
        const int last = min((iss.tile + 1) * tile_rows, iss.s.n * a.group) - 1;
        seen = (visible(a, iss.s, last) + TOK - 1) / TOK;
    };
    auto issue = [&](int st) {  // the group's first warp: the cursor's chunk into stage st
        const int pg = iss.c / CPP;
        if (iss.b != pb || pg < pbase || pg >= pbase + 32) {
            pb = iss.b, pbase = pg;
            const int pages = (iss.s.len + kKv8Page - 1) / kKv8Page;
            pnum = pg + lane < pages ? __ldg(a.kv.page_table + (int64_t)pb * a.kv.max_pages + pg + lane) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, pnum, pg - pbase);
        if (lane == 0) {
            const bool ok = iss.c < seen && (unsigned)page < (unsigned)a.kv.num_pages;
            if (iss.c < seen && !ok) report(a.kv, LASTRO_KV8_BAD_PAGE);
            there[st] = ok;
            if (ok) {
                const int64_t tile = (int64_t)page * H + iss.h;
                const int64_t at = tile * kKv8Page * D + (int64_t)(iss.c % CPP) * kChunkBytes;
                unsigned char* dst = data + (size_t)st * kStageBytes;
                mbar_expect_tx(full + st, kStageBytes + 32);
                bulk_g2s(dst, static_cast<const uint8_t*>(a.kv.k) + at, kChunkBytes, full + st);
                bulk_g2s(dst + kChunkBytes, static_cast<const uint8_t*>(a.kv.v) + at, kChunkBytes, full + st);
                bulk_g2s(scales + st * 8, a.kv.k_scale + tile * kKv8Blocks, 16, full + st);
                bulk_g2s(scales + st * 8 + 4, a.kv.v_scale + tile * kKv8Blocks, 16, full + st);
            } else {
                mbar_arrive(full + st);
            }
        }
        advance(iss);
        if (iss.c == 0) limit();
    };
    limit();
    if (wrow == 0)
        for (int i = 0; i < min(ST, count); ++i) issue(i);

    const bool vq = vec_rows(a.q);
    QFrag<D, NE, F32> q;
    float o[D / 8][4], M[NE], R[NE], l[NE], g[NE];
    int vis[NE], vmin = 0, rows0 = 0;
    bool mine = false, from0 = false;  // the warp has rows of the unit; the unit began in this share
    auto begin_unit = [&]() {
        rows0 = cur.tile * tile_rows + wrow * 16;
        mine = rows0 < cur.s.n * a.group;
        from0 = cur.c == 0;
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            M[e] = R[e] = kFar;
            l[e] = g[e] = 0.0f;
            vis[e] = visible(a, cur.s, rows0 + gq + 8 * e);
        }
        vmin = visible(a, cur.s, rows0);
        if (mine) q.load(a, cur.s, cur.h, rows0, vq, lane);
    };
    begin_unit();

    // the chunk at t0 in shared memory; WHOLE: every row sees every slot of it
    auto consume = [&](auto whole_tag, const unsigned char* sk, const float* sc, int t0, int item) {
        constexpr bool WHOLE = decltype(whole_tag)::value;
        const unsigned char* sv = sk + kChunkBytes;
        float s[NB][2][2 * NE];  // raw products
        float fk[NB][NE];        // what makes a raw product a score, in powers of two
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float ks = sc[b];
#pragma unroll
            for (int e = 0; e < NE; ++e) fk[b][e] = q.factor[e] * ks;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[D / 16], kf[D / 16][2];
                k_codes<D>(sk + (b * 16 + slot_of(gq >> 1, gq & 1, j)) * D, lane, w);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) widen<FMT>(w[k], kf[k][0], kf[k][1]);
                score_tile<D, NE, F32>(q, kf, s[b][j]);
                if (!WHOLE)
#pragma unroll
                    for (int i = 0; i < 2 * NE; ++i)
                        if (t0 + b * 16 + slot_of(c4, i & 1, j) >= vis[i >> 1]) s[b][j][i] = -INFINITY;
            }
        }
        if (NE == 1 && a.scores && rows0 + gq < cur.s.n * a.group) {  // for the weights: this lane's slots of each block
            float* dst = a.scores + ((int64_t)item * a.score_rows + gq) * TOK + 4 * c4;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = s[b][i >> 1][i & 1] * fk[b][0];
                    if (!WHOLE && s[b][i >> 1][i & 1] == -INFINITY) v[i] = -INFINITY;
                }
                *reinterpret_cast<float4*>(dst + b * 16) = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
        float Mn[NE], Rn[NE];
        bool moved = false;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            float m = -INFINITY, r = -INFINITY;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float top = fmaxf(fmaxf(s[b][0][2 * e], s[b][0][2 * e + 1]), fmaxf(s[b][1][2 * e], s[b][1][2 * e + 1])) * fk[b][e];
                m = fmaxf(m, top);
                r = fmaxf(r, top + (float)((int)(__float_as_uint(sc[4 + b]) >> 23) - 127));
            }
#pragma unroll
            for (int x = 1; x < 4; x <<= 1) {
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, x));
            }
            Mn[e] = fmaxf(M[e], ceilf(m));
            Rn[e] = fmaxf(R[e], ceilf(r));
            moved |= Mn[e] != M[e] || Rn[e] != R[e];
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                l[e] *= pow2i(M[e] - Mn[e]);
                const float f = pow2i(R[e] - Rn[e]);
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    o[j][2 * e] *= f;
                    o[j][2 * e + 1] *= f;
                }
                M[e] = Mn[e];
                R[e] = Rn[e];
                g[e] = pow2i(14.0f + M[e] - R[e]);
            }
        }
        uint32_t pa[NB][2 * NE], pb[F32 ? NB : 1][2 * NE];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                // at most 2^14 / (the block's largest p); kept finite where that p is below the smallest f32
                const float f = min_nan(sc[4 + b] * g[e], 1.7e38f);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float p[2], w[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        p[i] = ex2(fmaf(s[b][j][2 * e + i], fk[b][e], -M[e]));
                        w[i] = p[i] * f;
                        // slots the row does not see; a NaN scale of theirs must not reach it
                        if (!WHOLE && s[b][j][2 * e + i] == -INFINITY) p[i] = w[i] = 0.0f;
                    }
                    l[e] += p[0] + p[1];
                    pa[b][j * NE + e] = pack_f16(w[0], w[1]);
                    if (F32) pb[F32 ? b : 0][j * NE + e] = rest_f16(pa[b][j * NE + e], w[0], w[1]);
                }
            }
        }
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
            // f32 rows: the chunk's sum on its own, added with rounding (the matrix unit truncates)
            float x[F32 ? 8 : 1][4] = {};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                uint2 u[2][2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int t = b * 16 + slot_of(c4, e, j);
                        u[j][e] = *reinterpret_cast<const uint2*>(sv + t * D + hf * 64 + 8 * gq);
                        if (!WHOLE && t0 + t >= cur.s.len) u[j][e] = make_uint2(0, 0);  // not written yet: any bits
                    }
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    uint32_t v[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t y = w ? u[j][0].y : u[j][0].x, z = w ? u[j][1].y : u[j][1].x;
                        widen<FMT>(__byte_perm(y, z, 0x5140), v[j][0], v[j][1]);
                        widen<FMT>(__byte_perm(y, z, 0x7362), v[j][2], v[j][3]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float (&acc)[4] = F32 ? x[F32 ? w * 4 + i : 0] : o[hf * 8 + w * 4 + i];
                        if (F32) mma_f16<NE>(acc, pb[F32 ? b : 0], v[0][i], v[1][i]);
                        mma_f16<NE>(acc, pa[b], v[0][i], v[1][i]);
                    }
                }
            }
            if (F32)
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int i = 0; i < 2 * NE; ++i) o[hf * 8 + j][i] += x[F32 ? j : 0][i];
        }
    };

    bool alive = true;
    for (int it = 0; it < count; ++it) {
        const int st = it % ST, ph = (it / ST) & 1;
        alive = mbar_wait(full + st, ph, a.kv.status, LASTRO_KV8_BAD_WAIT);
        if (!alive) break;
        if (mine && there[st]) {
            const unsigned char* sk = data + (size_t)st * kStageBytes;
            const float* sc = scales + st * 8 + (cur.c % CPP) * NB;
            const int t0 = cur.c * TOK;
            if (t0 + TOK <= vmin)
                consume(std::true_type{}, sk, sc, t0, beg + it);
            else
                consume(std::false_type{}, sk, sc, t0, beg + it);
        }
        __syncwarp();
        if (RW > 1 && lane == 0) mbar_arrive(empty + st);
        if (wrow == 0 && it + ST < count) {
            if (RW > 1) {
                alive = mbar_wait(empty + st, ph, a.kv.status, LASTRO_KV8_BAD_WAIT);
                if (!alive) break;
            }
            issue(st);
        }
        const bool last = cur.c == cur.s.chunks - 1;
        if (last || it == count - 1) {
            if (mine) {
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
                    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
                    const int r = rows0 + gq + 8 * e;
                    if (r >= cur.s.n * a.group) continue;
                    if (last && from0) {
                        store_row<D, NE, F32>(a, cur.s, cur.h, r, lane, o, e, M[e], R[e], l[e], vo);
                    } else {
                        const int at = gq + 8 * e;
                        float* p = RW > 1   ? a.part + (((int64_t)group * 2 + (from0 ? 1 : 0)) * tile_rows + wrow * 16 + at) * part_floats(D)
                                   : from0 ? reinterpret_cast<float*>(data) + at * part_floats(D)
                                           : heads + (warp * 8 * NE + at) * part_floats(D);
#pragma unroll
                        for (int hf = 0; hf < D / 64; ++hf)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                reinterpret_cast<float4*>(p + hf * 64 + 16 * c4)[i] =
                                    make_float4(o[hf * 8 + (4 * i & 7)][2 * e + (i >> 1)], o[hf * 8 + (4 * i & 7) + 1][2 * e + (i >> 1)],
                                                o[hf * 8 + (4 * i & 7) + 2][2 * e + (i >> 1)], o[hf * 8 + (4 * i & 7) + 3][2 * e + (i >> 1)]);
                        if (c4 == 0) *reinterpret_cast<float4*>(p + D) = make_float4(M[e], R[e], l[e], 0.0f);
                    }
                }
            }
            if (RW == 1 && lane == 0 && !(last && from0)) {
                Ends& x = ends[warp];
                if (from0)
                    x.tail = true, x.th = cur.h, x.tt = cur.tile, x.tn = cur.s.n, x.tfirst = cur.s.first;
                else
                    x.mid = true, x.closes = last, x.hh = cur.h, x.ht = cur.tile, x.hn = cur.s.n, x.hfirst = cur.s.first;
            }
            if (it + 1 < count) {
                advance(cur);
                begin_unit();
            }
        } else {
            ++cur.c;
        }
    }
    if (!alive && wrow == 0)  // a copy that did not arrive: leave no other in flight behind
        for (int i = 0; i < ST; ++i) mbar_wait(full + i, 0, nullptr, 0);
    }
    if (RW > 1) return;

    // the units that the warps of this CTA cut, row by row: to the output when all of one is here, else to this share's
    // slots.  A run begins with the unit the share begins inside of (which < 0) or with the one warp `which` left open.
    __syncthreads();
    for (int which = -1; which < kWarps; ++which) {
        if (which < 0 ? !ends[0].mid : !ends[which].tail) continue;
        int n = which < 0 ? 0 : 1;  // parts before warp which + 1's
        bool closed = false;
        for (int j = which + 1; j < kWarps && ends[j].mid && !closed; ++j, ++n) closed = ends[j].closes;
        const Ends& x = ends[max(which, 0)];
        const int h = which < 0 ? x.hh : x.th, tile = which < 0 ? x.ht : x.tt;
        const int row0 = which < 0 ? x.hfirst : x.tfirst;
        const int first = which < 0 ? 0 : which, rows = min(16, (which < 0 ? x.hn : x.tn) * a.group - tile * 16);
        for (int r = warp; r < rows; r += kWarps) {
            float o[D / 32] = {}, M = kFar, R = kFar, l = 0.0f;
            add_parts<D>(n, [&](int i) -> const float* {
                if (which >= 0 && i == 0)
                    return reinterpret_cast<const float*>(smem + (size_t)first * ST * kStageBytes) + r * part_floats(D);
                return heads + ((first + i) * 8 * NE + r) * part_floats(D);
            }, o, M, R, l);
            if (which >= 0 && closed) {
                store_merged<D, F32>(a, row0, h, tile * 16 + r, o, M, R, l);
            } else {
                float* p = a.part + (((int64_t)blockIdx.x * 2 + (which >= 0)) * 16 + r) * part_floats(D);
                if (D == 64)
                    reinterpret_cast<float2*>(p)[lane] = make_float2(o[0], o[1]);
                else
                    reinterpret_cast<float4*>(p)[lane] = make_float4(o[0], o[1], o[D / 32 - 2], o[D / 32 - 1]);
                if (lane == 0) *reinterpret_cast<float4*>(p + D) = make_float4(M, R, l, 0.0f);
            }
        }
    }
}

// ---- merging the shares -----------------------------------------------------------------------------------------------
// One warp per query row and head whose unit was cut between shares, in the order of the shares.
template <int D, int RW, bool F32>
__global__ void __launch_bounds__(kThreads) kv8_merge_kernel(const __grid_constant__ Kv8AttendArgs a) {
    constexpr int TOK = ring_tok(D), tile_rows = 16 * RW;
    pdl_wait();
    pdl_launch();
    const int b = blockIdx.y;
    const Seq s = seq_of<TOK>(a, b, tile_rows);
    const int per = share_of(a.offset[a.kv.n_seqs], a.shares), base = a.offset[b];
    for (int u = blockIdx.x * kWarps + (threadIdx.x >> 5); u < s.n * a.heads; u += gridDim.x * kWarps) {
        const int i = u / a.heads, hq = u - i * a.heads, h = hq / a.group, r = i * a.group + hq - h * a.group, tile = r / tile_rows;
        const int first = base + (h * s.tiles + tile) * s.chunks, g0 = first / per, g1 = (first + s.chunks - 1) / per;
        if (g0 == g1) continue;
        float o[D / 32] = {}, M = kFar, R = kFar, l = 0.0f;
        for (int g = g0; g <= g1; g += 32)
            add_parts<D>(min(32, g1 + 1 - g), [&](int k) {
                return a.part + (((int64_t)(g + k) * 2 + (g + k == g0)) * tile_rows + r - tile * tile_rows) * part_floats(D);
            }, o, M, R, l);
        store_merged<D, F32>(a, s.first, h, r, o, M, R, l);
    }
}

// ---- accumulated weights, from stored scores ------------------------------------------------------------------------------
// With at most 8 query rows the pass over the cache also leaves its scores (4 bytes a row and slot, against d bytes of K),
// and the weights are one elementwise pass over them: a thread takes a block's four slots of one lane of that pass.
template <int D>
__global__ void __launch_bounds__(128) kv8_weights_kernel(const __grid_constant__ Kv8AttendArgs a) {
    constexpr int TOK = ring_tok(D);
    pdl_wait();
    pdl_launch();
    const int b = blockIdx.z, h = blockIdx.y, H = a.kv.kv_heads;
    const Seq s = seq_of<TOK>(a, b, 16);
    const int base = a.offset[b] + h * s.chunks, rows = s.n * a.group, c4 = threadIdx.x & 3;
    float lse[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
        if (r < rows) lse[r] = __ldcg(a.lse + (int64_t)(s.first + r / a.group) * a.heads + h * a.group + r % a.group);
    for (int blk = (blockIdx.x * 128 + threadIdx.x) >> 2; blk * kKv8Block < s.len; blk += gridDim.x * 32) {
        const int t0 = blk * kKv8Block;
        float sum[4] = {};
        if (rows > 0 && page_of(a.kv, b, t0) >= 0) {
            const float* src = a.scores + (int64_t)(base + t0 / TOK) * a.score_rows * TOK + t0 % TOK + 4 * c4;
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < rows) {
                    const float4 v = __ldcg(reinterpret_cast<const float4*>(src + r * TOK));
                    sum[0] += ex2(v.x - lse[r]), sum[1] += ex2(v.y - lse[r]);
                    sum[2] += ex2(v.z - lse[r]), sum[3] += ex2(v.w - lse[r]);
                }
        }
        const int64_t at = ((int64_t)b * H + h) * a.mass_stride + t0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = slot_of(c4, i & 1, i >> 1);
            if (t0 + t < s.len) a.mass_out[at + t] = (a.mass_in ? a.mass_in[at + t] : 0.0f) + sum[i];
        }
    }
}

// ---- accumulated weights, from K ------------------------------------------------------------------------------------------
// More query rows: the scores are computed again, with the finished softmax sums at hand.  CTAs take equal consecutive
// shares of the (sequence, KV head, chunk) list; a warp holds a chunk's K in registers as f16 and runs the query tiles
// past it from shared memory.
constexpr int kMassTiles = kWarps;  // query tiles in shared memory at a time, one loaded by each warp

template <int D, int NE, bool F32>
constexpr size_t mass_smem() {
    return (size_t)kMassTiles * (D / 16) * 32 * 8 * NE * (F32 ? 2 : 1) + kMassTiles * 16 * 3 * 4 + kWarps * 64 * 4;
}

template <int FMT, int D, int NE, bool F32>
__global__ void __launch_bounds__(kThreads) kv8_mass_kernel(const __grid_constant__ Kv8AttendArgs a) {
    constexpr int TOK = kChunkBytes / D, NB = TOK / kKv8Block, CPP = kKv8Page / TOK, KS = D / 16;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    pdl_wait();
    pdl_launch();
    using Frag = std::conditional_t<NE == 2, uint4, uint2>;
    Frag* qs = reinterpret_cast<Frag*>(smem_raw);  // [tile][ks][lane], first terms then second ones
    float* rfac = reinterpret_cast<float*>(qs + (size_t)kMassTiles * KS * 32 * (F32 ? 2 : 1));
    float* rlse = rfac + kMassTiles * 16;
    int* rvis = reinterpret_cast<int*>(rlse + kMassTiles * 16);
    float* sums = reinterpret_cast<float*>(rvis + kMassTiles * 16) + (threadIdx.x >> 5) * 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, c4 = lane & 3, H = a.kv.kv_heads;
    const bool vq = vec_rows(a.q);
    const auto chunks_of = [&](int b) {
        const Seq s = seq_of<TOK>(a, b, 16);
        return (s.len + TOK - 1) / TOK;
    };
    const auto work = [&](int b) { return H * chunks_of(b); };
    const List<decltype(work)> list(a.kv.n_seqs, work);
    const int per = share_of(list.total, gridDim.x), end = min(list.total, (int)(blockIdx.x + 1) * per);
    int pos = blockIdx.x * per, base = 0;  // base: where sequence b's items start
    if (pos >= end) return;
    int b = list.seek(pos, false, base, [](int, int) {});
    while (pos < end) {
        const Seq s = seq_of<TOK>(a, b, 16);
        const int chunks = (s.len + TOK - 1) / TOK;
        if (pos >= base + H * chunks) {
            base += H * chunks;
            ++b;
            continue;
        }
        const int h = (pos - base) / chunks, c0 = (pos - base) % chunks, c1 = min(chunks, c0 + (end - pos));
        const int rows = s.n * a.group, tiles = (rows + 15) / 16;
        for (int tb = 0; tb < max(1, tiles); tb += kMassTiles) {
            const int nt = min(kMassTiles, tiles - tb);
            __syncthreads();  // the tiles before these are done with
            if (warp < nt) {
                const int row0 = (tb + warp) * 16;
                QFrag<D, NE, F32> q;
                q.load(a, s, h, row0, vq, lane);
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    qs[(warp * KS + k) * 32 + lane] = *reinterpret_cast<const Frag*>(q.hi[k]);
                    if (F32) qs[((kMassTiles + warp) * KS + k) * 32 + lane] = *reinterpret_cast<const Frag*>(q.lo[F32 ? k : 0]);
                }
                if (c4 == 0)
#pragma unroll
                    for (int e = 0; e < NE; ++e) {
                        const int r = row0 + gq + 8 * e, at = warp * 16 + gq + 8 * e;
                        rfac[at] = q.factor[e];
                        rvis[at] = visible(a, s, r);
                        rlse[at] = r < rows ? a.lse[(int64_t)(s.first + r / a.group) * a.heads + h * a.group + r % a.group] : INFINITY;
                    }
            }
            __syncthreads();
            for (int c = c0 + warp; c < c1; c += kWarps) {
                const int page = page_of(a.kv, b, c * TOK);
                float sum[NB][2][2] = {};
                if (page >= 0 && nt > 0) {
                    const int64_t tile = (int64_t)page * H + h;
                    const uint8_t* kp = static_cast<const uint8_t*>(a.kv.k) + tile * kKv8Page * D + (int64_t)(c % CPP) * kChunkBytes;
                    uint32_t kf[NB][2][KS][2];
                    float ks[NB];
                    {
                        uint32_t w[NB][2][KS];
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            ks[n] = __ldg(a.kv.k_scale + tile * kKv8Blocks + (c % CPP) * NB + n);
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                k_codes<D>(kp + (n * 16 + slot_of(gq >> 1, gq & 1, j)) * D, lane, w[n][j]);
                        }
#pragma unroll
                        for (int n = 0; n < NB; ++n)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int k = 0; k < KS; ++k) widen<FMT>(w[n][j][k], kf[n][j][k][0], kf[n][j][k][1]);
                    }
                    for (int t = 0; t < nt; ++t) {
                        const bool whole = c * TOK + TOK <= rvis[t * 16];
                        QFrag<D, NE, F32> q;
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            *reinterpret_cast<Frag*>(q.hi[k]) = qs[(t * KS + k) * 32 + lane];
                            if (F32) *reinterpret_cast<Frag*>(q.lo[F32 ? k : 0]) = qs[((kMassTiles + t) * KS + k) * 32 + lane];
                        }
                        float lse[NE];
                        int vis[NE];
#pragma unroll
                        for (int i = 0; i < NE; ++i) {
                            q.factor[i] = rfac[t * 16 + gq + 8 * i];
                            lse[i] = rlse[t * 16 + gq + 8 * i];
                            vis[i] = rvis[t * 16 + gq + 8 * i];
                        }
#pragma unroll
                        for (int n = 0; n < NB; ++n)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                float acc[2 * NE];
                                score_tile<D, NE, F32>(q, kf[n][j], acc);
#pragma unroll
                                for (int i = 0; i < 2 * NE; ++i) {
                                    float p = ex2(acc[i] * (q.factor[i >> 1] * ks[n]) - lse[i >> 1]);
                                    if (!whole && c * TOK + n * 16 + slot_of(c4, i & 1, j) >= vis[i >> 1]) p = 0.0f;
                                    sum[n][j][i & 1] += p;
                                }
                            }
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
#pragma unroll
                                for (int x = 4; x < 32; x <<= 1) sum[n][j][e] += __shfl_xor_sync(0xffffffffu, sum[n][j][e], x);
                }
                if (gq == 0)
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e) sums[n * 16 + slot_of(c4, e, j)] = sum[n][j][e];
                __syncwarp();
                const float* in = tb ? a.mass_out : a.mass_in;
#pragma unroll
                for (int i = lane; i < TOK; i += 32) {
                    const int t = c * TOK + i;
                    const int64_t at = ((int64_t)b * H + h) * a.mass_stride + t;
                    if (t < s.len) a.mass_out[at] = (in ? in[at] : 0.0f) + sums[i];
                }
                __syncwarp();
            }
        }
        pos += c1 - c0;
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------
int sm_count() {
    static const int n = [] {
        int dev = 0, v = 0;
        cudaGetDevice(&dev);
        return cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0 ? v : 148;
    }();
    return n;
}

template <typename K>
cudaError_t launch(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, const Kv8AttendArgs& a) {
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// warps that share a stage: as many 16-row tiles as the largest unit has, up to 8
int row_warps(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }

struct AttendLaunch {
    Kv8AttendArgs a;
    cudaStream_t s;

    template <int FMT, int D, int RW, int NE, bool F32>
    cudaError_t go() {
        using RG = Ring<D, RW, NE>;
        a.shares = sm_count() * (RW == 1 ? 1 : RG::GROUPS);
        cudaError_t e = launch(kv8_attend_kernel<FMT, D, RW, NE, F32>, dim3(sm_count()), kThreads, RG::bytes, s, a);
        if (e != cudaSuccess) return e;
        const int64_t rows = (int64_t)a.max_new * a.heads;
        const dim3 grid((unsigned)min((int64_t)1024, (rows + kWarps - 1) / kWarps), a.kv.n_seqs);
        e = launch(kv8_merge_kernel<D, RW, F32>, grid, kThreads, 0, s, a);
        if (e != cudaSuccess || !a.mass_out) return e;
        if (a.scores) {
            const dim3 blocks(min(64, (a.kv.max_pages * kKv8Blocks + 31) / 32), a.kv.kv_heads, a.kv.n_seqs);
            return launch(kv8_weights_kernel<D>, blocks, 128, 0, s, a);
        }
        return launch(kv8_mass_kernel<FMT, D, NE, F32>, dim3(2 * sm_count()), kThreads, mass_smem<D, NE, F32>(), s, a);
    }
    template <int FMT, int D, int RW, int NE>
    cudaError_t by_type() {
        return a.q.dtype == LASTRO_DTYPE_F32 ? go<FMT, D, RW, NE, true>() : go<FMT, D, RW, NE, false>();
    }
    template <int FMT, int D>
    cudaError_t run() {
        const int64_t rows = (int64_t)a.max_new * a.group;
        switch (row_warps(rows)) {
        case 1: return rows <= 8 ? by_type<FMT, D, 1, 1>() : by_type<FMT, D, 1, 2>();
        case 2: return by_type<FMT, D, 2, 2>();
        case 4: return by_type<FMT, D, 4, 2>();
        default: return by_type<FMT, D, 8, 2>();
        }
    }
};

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

size_t kv8_attend_workspace(const lastro_kv8& kv, int heads, int max_new, bool with_mass, Kv8AttendArgs* a, void* base) {
    const int64_t rows = (int64_t)max_new * (heads / kv.kv_heads);
    const int rw = row_warps(rows);
    const size_t row = part_floats(kv.head_dim) * sizeof(float), sms = sm_count();
    const size_t offset = align16(((size_t)kv.n_seqs + 1) * sizeof(int32_t));
    const size_t part = sms * (rw == 1 ? 1 : 8 / rw) * 2 * rw * 16 * row;
    const size_t lse = with_mass ? align16((size_t)kv.n_seqs * max_new * heads * sizeof(float)) : 0;
    // kept scores save the second pass over K; past 1 GiB of them K is read again instead
    size_t scores = with_mass && rows <= 8 ? (size_t)kv.n_seqs * kv.kv_heads * kv.max_pages * kKv8Page * rows * sizeof(float) : 0;
    if (scores > ((size_t)1 << 30)) scores = 0;
    if (a) {
        unsigned char* p = static_cast<unsigned char*>(base);
        a->offset = reinterpret_cast<int32_t*>(p);
        a->part = reinterpret_cast<float*>(p + offset);
        a->lse = with_mass ? reinterpret_cast<float*>(p + offset + part) : nullptr;
        a->scores = scores ? reinterpret_cast<float*>(p + offset + part + lse) : nullptr;
        a->score_rows = (int32_t)rows;
    }
    return offset + part + lse + scores;
}

int64_t kv8_attend_items(const lastro_kv8& kv, int heads, int max_new) {
    const int64_t rows = (int64_t)max_new * (heads / kv.kv_heads), tile = 16 * row_warps(rows);
    const int64_t chunks = (int64_t)kv.max_pages * (kKv8Page * kv.head_dim / kChunkBytes);
    const double items = (double)kv.n_seqs * kv.kv_heads * chunks * ((rows + tile - 1) / tile + 1);
    return items < 9e18 ? (int64_t)items : INT64_MAX;
}

cudaError_t launch_kv8_attend(const Kv8AttendArgs& a, cudaStream_t s) { return kv8_by_shape(a.kv, AttendLaunch{a, s}); }

}  // namespace lastro
