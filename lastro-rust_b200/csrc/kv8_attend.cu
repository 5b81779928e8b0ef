// Attention over the 8-bit KV cache (lastro_kv8_attend): scores, softmax and weighted sum in one pass over the cache, the
// weights every slot received in a second pass over the scores it kept, or over K.
//
// A KV head's query rows are its group's heads times the sequence's queries.  The products are m16n8k16 matrix products,
// a block's 16 slots at a time, in one of two forms:
//   few rows (at most 8, single-token decode): the rows are the n side, S^T = K Q^T and O^T += V^T P^T with K and V^T as
//     the 16-row operand, so that no part of a tile is empty;
//   many rows: 16 rows are the m side, S = Q K^T and O += P V.
// Codes go from shared memory to operand registers and are widened to f16 there, which holds every e4m3 and int8 value
// exactly; the scales, powers of two, are applied to the scores (K) and to the weights (V) in f32.
#include <cuda_runtime.h>

#include <type_traits>

#include "kv8.cuh"

namespace lastro {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;  // of the merge and mass kernels
constexpr float kFar = -3.402823466e38f;          // no score is below it: the running maxima's start
constexpr float kLow = -112.0f;                   // the least R (WarpRows): 2^(R - 14), which outputs are scaled by, is 2^-126

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

// d (+)= a (16x16, row) * b (16x8, col), f16 operands, f32 accumulators
LDEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the 8x8 matrix of 16-bit values whose row l / 4, columns 2 (l % 4) and + 1 lane l holds, transposed
LDEV uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// A score this far from zero is a product whose rounding counts in 2^(score - M), and adding an exponent to it may round that
// away.  M is the ceiling of rounded products; closer to zero they need not be rounded before M is taken from them.
LDEV bool far_off(float M) { return fabsf(M) > 4096.0f && M != kFar; }

// the smaller, NaN if either is
LDEV float min_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
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

// bulk_g2s for data read once: its lines leave L2 before others
LDEV void bulk_g2s_once(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
                     smem_addr(dst)),
                 "l"(src), "r"(bytes), "r"(smem_addr(bar)), "l"(policy)
                 : "memory");
}
LDEV uint64_t read_once() {
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}

LDEV void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Rows of the same block that one shared-memory access reads: index i = 2 * pair + e + 8 * j of a product stands for slot
// slot_of(pair, e, j).  Any bijection is right; this one spreads those rows over both halves of a 128-byte line.
LDEV int slot_of(int pair, int e, int j) { return j * 8 + e * 4 + (pair & 2) + ((pair & 1) ^ e); }

// ---- shapes -------------------------------------------------------------------------------------------------------------
// How a call's units (one sequence, KV head and tile of query rows) are worked on: RW of a CTA's 8 warps side by side take
// a tile of RW * ROWS rows and share the stages of one ring.
//   Few rows with 16 warps of half the chunk instead: 315 against 267 us at 96 sequences of 8192 slots, 32 heads of 128 (the
//   work around a chunk counts for more than the latency that more warps hide).
//   More than 16 rows in tiles of 16, 32, 64 or 128 rows (RW 1, 2, 4, 8): 39.6, 33.5, 39.4 and 40.6 us at 8 sequences of
//   2048 slots with 32 queries of 24 heads, 28.2, 27.5, 27.4 and 33.8 with 16, 309, 317, 395 and 426 at 32 sequences of
//   8192: two warps that share a stage halve its traffic, more of them wait on one another or have no rows.
template <int D, bool FEW, int RW>
struct Shape {
    static constexpr int WARPS = 8, THREADS = WARPS * 32, GROUPS = WARPS / RW;
    static constexpr int ROWS = FEW ? 8 : 16, TILE = RW * ROWS;       // query rows of a warp and of a unit
    static constexpr int CHUNK = 4096, TOK = CHUNK / D;               // K (or V) codes and slots of a stage
    static constexpr int NB = TOK / kKv8Block, CPP = kKv8Page / TOK;  // blocks of a chunk, chunks of a page
    // as many as shared memory holds beside the rest (two to six with RW 2: 48.2, 47.9, 47.7, 47.7 us at 8 sequences of 2048
    // slots with 32 queries; two or three with few rows: 24.5 and 24.6 us at 64 of 1024, the same at 96 of 8192)
    static constexpr int STAGES = FEW ? 3 : RW == 1 ? 2 : 6;
    static constexpr int PART = D + 4;  // floats of one row's partial result: its sums, then M, R and l
    // items of a share: a chunk for each warp, and of groups enough that merging does not cost more than they do (one
    // sequence of 2048 slots: 32 CTAs and 4 parts a unit, not 128 and 16)
    static constexpr int LEAST = RW == 1 ? WARPS : 4;
    static constexpr int BARS = RW == 1 ? 1 : 2;  // a warp on its own needs no barrier to hand stages back
    static constexpr size_t HEAD = RW == 1 ? (size_t)ROWS * PART * sizeof(float) : 0;
    static constexpr size_t SMEM = (size_t)GROUPS * (STAGES * (2 * CHUNK + 8 * sizeof(float) + BARS * 8 + 4) + HEAD);
};

// the form for units of at most `rows` rows: 0 few rows, else the warps that share a unit
int row_warps(int64_t rows) { return rows <= 8 ? 0 : rows <= 16 ? 1 : 2; }

// ---- the list of work -------------------------------------------------------------------------------------------------
// Every sequence with queries contributes kv_heads * row tiles * chunks items, chunks innermost; equal consecutive shares
// of the whole list go to the CTAs (RW 1) or groups of warps, so that ragged lengths balance to within one chunk.
struct Seq {
    int len, n, first;  // slots, queries, first query row
    int chunks, tiles;  // of one unit; row tiles of one head
};

template <int TOK, int TILE>
LDEV Seq seq_of(const Kv8AttendArgs& a, int b) {
    Seq s;
    int64_t most = (int64_t)a.kv.max_pages * kKv8Page;
    if (a.mass_out) most = min(most, a.mass_stride);
    s.len = seq_len(a.kv, a.lens, b, most);
    s.n = seq_rows(a.kv, a.q_off, b, a.q.rows, a.max_new, s.first);
    s.chunks = max(1, (s.len + TOK - 1) / TOK);  // a query of an empty sequence still gets its zeros
    s.tiles = (s.n * a.group + TILE - 1) / TILE;
    return s;
}

// items of one share when `total` are dealt to n shares, `least` or more to each
LDEV int share_of(int total, int n, int least) { return max(least, (int)(((unsigned)total + n - 1) / n)); }

// exclusive prefix sum of v over the block and the total; `red` holds 32 ints
template <int THREADS>
LDEV int scan_block(int v, int* red, int& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    if (lane == 31) red[w] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
        const int t = red[i];
        if (i < w) before += t;
        total += t;
    }
    return before + s - v;
}

// The whole block finds its list: work(b) items of sequence b.  `part(total)` then says where each warp starts, and the
// warp gets the sequence that holds that item (-1 past the end) and where its items start.  `note(b, at)` is told
// where each sequence starts, by one thread.  `room`: THREADS + THREADS / 32 + 1 ints of shared memory.
template <int THREADS, typename Work, typename Part, typename Note>
LDEV void find_part(int* room, int n_seqs, Work work, Part part, Note note, int& total, int& seq, int& base) {
    int *red = room, *pre = room + THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31;
    int w = tid < n_seqs ? work(tid) : 0, sum = 0, all = 0;
    if (n_seqs > THREADS) {
        int v = w;
        for (int b = tid + THREADS; b < n_seqs; b += THREADS) v += work(b);
        scan_block<THREADS>(v, red, all);
    }
    seq = -1;
    for (int b0 = 0; b0 < n_seqs; b0 += THREADS) {
        if (b0) w = b0 + tid < n_seqs ? work(b0 + tid) : 0;
        __syncthreads();  // the previous use of red and pre is over
        int here;
        const int at = sum + scan_block<THREADS>(w, red, here);
        pre[tid] = at;
        if (b0 + tid < n_seqs) note(b0 + tid, at);
        if (tid == 0) pre[THREADS] = sum + here;
        __syncthreads();
        total = n_seqs > THREADS ? all : here;
        const int pos = part(total);
        if (seq < 0 && pos < sum + here)
            for (int t = lane; __any_sync(0xffffffffu, t < THREADS); t += 32) {
                const unsigned hit = __ballot_sync(0xffffffffu, t < THREADS && pre[t] <= pos && pos < pre[t + 1]);
                if (hit) {
                    const int i = (t & ~31) + __ffs(hit) - 1;
                    seq = b0 + i;
                    base = pre[i];
                    break;
                }
            }
        sum += here;
    }
    // `room` is in the rings: its ordinary accesses before the bulk copies to come, which write through another proxy
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
}

// ---- query rows ---------------------------------------------------------------------------------------------------------
// 8 * E rows as product operands (row r is query r / group, head r % group of the KV head; lane l holds rows l / 4 and
// l / 4 + 8) and each row's factor from the raw product to the score in powers of two.  A row is scaled by a power of two
// to a largest magnitude in [2^14, 2^15), which puts a bf16 value exactly into f16 down to 2^-28 of that magnitude; f32
// rows take a second term.  The factor is positive (a negative scale goes into the operand), so that the largest product
// is the largest score.
template <int D, int E, bool F32>
struct QRaw {  // the rows as they are stored: loads on their way while other work goes on
    Raw8<F32> x[E][D / 32];

    LDEV void fetch(const Kv8AttendArgs& a, const Seq& s, int h, int row0, bool vec) {
        const int lane = threadIdx.x & 31, gq = lane >> 2, c = lane & 3;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int r = row0 + gq + 8 * e, i = query_of(r, a.group);
            const bool there = r < s.n * a.group;
            const int64_t at = (int64_t)(s.first + i) * a.q.row_stride + (int64_t)(h * a.group + r - i * a.group) * a.q.head_stride + 16 * c;
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
                if (there)
                    x[e][k].load(a.q, at + k / 2 * 64 + k % 2 * 8, vec);
                else
                    x[e][k].zero();
        }
    }
};

template <int D, int E, bool F32>
struct QFrag {
    static constexpr int KS = D / 16;
    uint32_t hi[KS][2 * E], lo[F32 ? KS : 1][2 * E];  // [k step][k half, row half]
    float factor[E];

    LDEV void convert(const QRaw<D, E, F32>& raw, float scale) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < D / 32; ++k) raw.x[e][k].widest(m);
            uint32_t amax = Raw8<F32>::f32_bits(m);
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int k = min(126, 141 - (int)(amax >> 23));  // 14 - exponent
            const bool finite = amax < 0x7f800000u;
            const float up = copysignf(__uint_as_float((uint32_t)(k + 127) << 23), scale);
            factor[e] = finite ? fabsf(scale) * 1.44269504088896340736f * __uint_as_float((uint32_t)(127 - k) << 23)
                               : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                float v[8];
                raw.x[e][i].values(v);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float u = finite ? v[2 * j] * up : 0.0f, w = finite ? v[2 * j + 1] * up : 0.0f;
                    uint32_t& t = hi[2 * i + j / 2][(j & 1) * E + e];
                    t = pack_f16(u, w);
                    if (F32) lo[F32 ? 2 * i + j / 2 : 0][(j & 1) * E + e] = rest_f16(t, u, w);
                }
            }
        }
    }
};

// slots that row r of the sequence sees
LDEV int visible(const Kv8AttendArgs& a, const Seq& s, int r) {
    return s.len - s.n + query_of(min(r, s.n * a.group - 1), a.group) + 1;
}

// the codes of slot row `row` that this lane feeds to the score product: 16 bytes of every 64
template <int D>
LDEV void k_codes(const uint8_t* row, uint32_t (&w)[D / 16]) {
    const int lane = threadIdx.x & 31;
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

// A sum of products over the head dimension, `mma(x, k, second)` adding step k's product with the rows' first or second
// term to x.  The matrix unit truncates what it adds to an f32 accumulator, so f32 rows take their second term first,
// while the sum is small, and no more than two steps a chain; the chains are added with rounding.
template <int KS, bool F32, typename Mma>
LDEV void score_sum(float (&s)[4], Mma mma) {
    constexpr int CH = F32 ? 2 : KS;
#pragma unroll
    for (int k0 = 0; k0 < KS; k0 += CH) {
        float x[4] = {};
#pragma unroll
        for (int k = k0; F32 && k < k0 + CH; ++k) mma(x, k, true);
#pragma unroll
        for (int k = k0; k < k0 + CH; ++k) mma(x, k, false);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = k0 == 0 ? x[i] : s[i] + x[i];
    }
}

// ---- a warp's rows --------------------------------------------------------------------------------------------------------
// The running state of a row: M the ceiling of the largest score so far (scores and M in powers of two), l the sum of
// 2^(score - M), R the ceiling of the largest score - M plus its slot's V exponent, o the sum of 2^(score - M + 14 - R) v.
// M and R are whole numbers, so bringing sums to new ones is exact, and R keeps the f16 weights in range whatever the
// blocks' scales: the heaviest contribution sits between 2^13 and 2^14, or lower where V's scales are below 2^-112, so that
// the factors between them and the outputs stay in f32's range.  Scores of any size are as good as scores near zero: a warp
// one of whose rows is far_off takes the branch below for every chunk (this branch, not taken, costs 24.0 -> 24.7 us at 64
// sequences of 1024 slots with 24 heads of 64).  A lane holds two rows, row_of(0) and row_of(1).
template <int FMT, int D, bool FEW, bool F32>
struct WarpRows {
    static constexpr int KS = D / 16, E = FEW ? 1 : 2;
    static constexpr int NT = FEW ? 2 : 4;                // slots of a block a lane holds scores of, for each of its rows
    static constexpr int RUN = FEW ? 8 : 16;              // consecutive output values a lane holds of every 64
    QFrag<D, E, F32> q;
    float o[FEW ? D / 16 : D / 8][4], M[2], R[2], l[2], g[2], fac[2];
    int vis[2];
    bool big;  // a row's M is far_off

    LDEV static int row_of(int e) {
        const int lane = threadIdx.x & 31;
        return FEW ? 2 * (lane & 3) + e : (lane >> 2) + 8 * e;
    }
    LDEV static int col_of(int hf) {
        const int lane = threadIdx.x & 31;
        return hf * 64 + (FEW ? 8 * (lane >> 2) : 16 * (lane & 3));
    }
    LDEV static bool first_of_row() { return FEW ? (threadIdx.x & 31) < 4 : (threadIdx.x & 3) == 0; }
    LDEV static int slot(int k) {  // of the k-th score
        const int lane = threadIdx.x & 31;
        return FEW ? slot_of(lane >> 3, (lane >> 2) & 1, k) : slot_of(lane & 3, k & 1, k >> 1);
    }
    LDEV float value(int hf, int i, int e) const {
        return FEW ? o[hf * 4 + (i >> 1)][2 * (i & 1) + e] : o[(FEW ? 0 : hf * 8) + (FEW ? 0 : i & 7)][2 * e + (FEW ? 0 : i >> 3)];
    }
    template <typename Op>
    LDEV static float over_row(float v, Op op) {  // reduced over the lanes that hold the same row
#pragma unroll
        for (int x = FEW ? 4 : 1; x < (FEW ? 32 : 4); x <<= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, x));
        return v;
    }

    LDEV void begin(const Kv8AttendArgs& a, const Seq& s, int row0, const QRaw<D, E, F32>& raw) {
        q.convert(raw, a.scale);
        big = false;
#pragma unroll
        for (int j = 0; j < (FEW ? D / 16 : D / 8); ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            M[e] = kFar;
            R[e] = kLow;
            l[e] = g[e] = 0.0f;
            vis[e] = visible(a, s, row0 + row_of(e));
            fac[e] = FEW ? __shfl_sync(0xffffffffu, q.factor[0], 4 * row_of(e)) : q.factor[E - 1 < e ? 0 : e];
        }
    }

    // raw products of the block whose K codes are at sk
    LDEV void scores(const uint8_t* sk, float (&s)[2][NT]) const {
        const int lane = threadIdx.x & 31;
        if constexpr (FEW) {
            uint32_t w[2][KS], kf[2][KS][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                k_codes<D>(sk + slot(t) * D, w[t]);
#pragma unroll
                for (int k = 0; k < KS; ++k) widen<FMT>(w[t][k], kf[t][k][0], kf[t][k][1]);
            }
            float x[4];
            score_sum<KS, F32>(x, [&](float (&y)[4], int k, bool second) {
                const uint32_t(&b)[2] = second ? q.lo[F32 ? k : 0] : q.hi[k];
                mma_f16(y, kf[0][k][0], kf[1][k][0], kf[0][k][1], kf[1][k][1], b[0], b[1]);
            });
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i & 1][i >> 1] = x[i];
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[KS], kf[KS][2];
                k_codes<D>(sk + slot_of(lane >> 3, (lane >> 2) & 1, j) * D, w);
#pragma unroll
                for (int k = 0; k < KS; ++k) widen<FMT>(w[k], kf[k][0], kf[k][1]);
                float x[4];
                score_sum<KS, F32>(x, [&](float (&y)[4], int k, bool second) {
                    const uint32_t(&b)[2 * E] = second ? q.lo[F32 ? k : 0] : q.hi[k];
                    mma_f16(y, b[0], b[E - 1], b[E], b[2 * E - 1], kf[k][0], kf[k][1]);
                });
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i >> 1][(2 * j + (i & 1)) % NT] = x[i];
            }
        }
    }

    // One chunk: K codes at sk, V codes at sv, the chunk's K scales at ks[0..] and V scales at vs[0..]; WHOLE: every row
    // sees every slot, from t0 on.  `keep`, where it is not null, takes the scores: row r's at keep + r * TOK.
    template <bool WHOLE, int NB>
    LDEV void consume(const uint8_t* sk, const uint8_t* sv, const float* ks, const float* vs, int t0, int len, float* keep,
                      int rows) {
        const int lane = threadIdx.x & 31, gq = lane >> 2, c4 = lane & 3;
        float s[NB][2][NT], fk[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            scores(sk + b * 16 * D, s[b]);
#pragma unroll
            for (int e = 0; e < 2; ++e) fk[b][e] = fac[e] * ks[b];
        }
        uint32_t hidden = 0;  // of this lane's scores, those whose row does not see the slot
        if (!WHOLE) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int k = 0; k < NT; ++k)
                        if (t0 + b * 16 + slot(k) >= vis[e]) {
                            s[b][e][k] = -INFINITY;
                            hidden |= 1u << ((b * 2 + e) * NT + k);
                        }
        }
        if (FEW && keep) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (row_of(e) < rows)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int k = 0; k < NT; ++k)
                            keep[row_of(e) * NB * 16 + b * 16 + slot(k)] =
                                hidden >> ((b * 2 + e) * NT + k) & 1 ? -INFINITY : __fmul_rn(s[b][e][k], fk[b][e]);
        }
        // the largest score of block b and row e
        const auto block_top = [&](int b, int e) {
            float top = s[b][e][0];
#pragma unroll
            for (int k = 1; k < NT; ++k) top = fmaxf(top, s[b][e][k]);
            // a block that was never written has any scale, a negative one among them
            return !WHOLE && top == -INFINITY ? top : top * fk[b][e];
        };
        const auto larger = [](float x, float y) { return fmaxf(x, y); };
        const auto exponent = [](float x) { return (float)((int)(__float_as_uint(x) >> 23) - 127); };
        float Mn[2], Rn[2];
        bool moved = big;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float m = -INFINITY, r = -INFINITY;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float top = block_top(b, e);
                m = fmaxf(m, top);
                r = fmaxf(r, top + exponent(vs[b]));
            }
            Mn[e] = fmaxf(M[e], ceilf(over_row(m, larger)));
            Rn[e] = fmaxf(fmaxf(R[e] + (M[e] - Mn[e]), ceilf(over_row(r, larger)) - Mn[e]), kLow);
            moved |= Mn[e] != M[e] || Rn[e] != R[e];
        }
        if (__any_sync(0xffffffffu, moved)) {
            float f[2];
            big = __any_sync(0xffffffffu, far_off(Mn[0]) || far_off(Mn[1]));
            if (big) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float r = -INFINITY;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
#pragma unroll
                        for (int k = 0; k < NT; ++k)
                            if (WHOLE || !(hidden >> ((b * 2 + e) * NT + k) & 1)) s[b][e][k] = __fmul_rn(s[b][e][k], fk[b][e]);
                        fk[b][e] = 1.0f;
                        r = fmaxf(r, block_top(b, e) - Mn[e] + exponent(vs[b]));
                    }
                    Rn[e] = fmaxf(fmaxf(R[e] + (M[e] - Mn[e]), ceilf(over_row(r, larger))), kLow);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float up = M[e] - Mn[e];
                l[e] *= pow2i(up);
                f[e] = pow2i(up + (R[e] - Rn[e]));
                M[e] = Mn[e];
                R[e] = Rn[e];
                g[e] = pow2i(14.0f - Rn[e]);
            }
#pragma unroll
            for (int j = 0; j < (FEW ? D / 16 : D / 8); ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[j][i] *= f[FEW ? i & 1 : i >> 1];
        }
        // s becomes the weights: first 2^(score - M), which l sums, then what multiplies the V codes
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int k = 0; k < NT; ++k) s[b][e][k] = ex2(fmaf(s[b][e][k], fk[b][e], -M[e]));
        if (!WHOLE) {
#pragma unroll
            for (int i = 0; i < NB * 2 * NT; ++i)
                if (hidden >> i & 1) s[i / (2 * NT)][i / NT % 2][i % NT] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                // at most 2^14 / (the block's largest weight); kept finite where that weight is below the smallest f32
                const float f = min_nan(vs[b] * g[e], 1.7e38f);
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    l[e] += s[b][e][k];
                    s[b][e][k] *= f;
                }
            }
        if (!WHOLE) {  // a NaN scale must not reach the rows that do not see the slot
#pragma unroll
            for (int i = 0; i < NB * 2 * NT; ++i)
                if (hidden >> i & 1) s[i / (2 * NT)][i / NT % 2][i % NT] = 0.0f;
        }
        // the weights as product operands, first and second terms
        uint32_t pa[NB][FEW ? 2 : 4], pb[F32 ? NB : 1][FEW ? 2 : 4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float(&w)[2][NT] = s[b];
            if constexpr (FEW) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t x = pack_f16(w[0][k], w[1][k]);
                    pa[b][k] = transpose8(x);
                    if (F32) pb[F32 ? b : 0][k] = transpose8(rest_f16(x, w[0][k], w[1][k]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float w0 = w[e][(2 * j) % NT], w1 = w[e][(2 * j + 1) % NT];
                        pa[b][2 * j + e] = pack_f16(w0, w1);
                        if (F32) pb[F32 ? b : 0][2 * j + e] = rest_f16(pa[b][2 * j + e], w0, w1);
                    }
            }
        }
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
            constexpr int NO = FEW ? 4 : 8;  // accumulator tiles of 64 output values
            // f32 rows: the chunk's sum on its own, added with rounding (the matrix unit truncates)
            float x[F32 ? NO : 1][4] = {};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                uint2 u[2][2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int t = b * 16 + slot_of(c4, e, j);
                        u[j][e] = *reinterpret_cast<const uint2*>(sv + t * D + hf * 64 + 8 * gq);
                        if (!WHOLE && t0 + t >= len) u[j][e] = make_uint2(0, 0);  // not written yet: any bits
                    }
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    uint32_t v[2][4];  // values 4w .. 4w + 3 of this lane's 8, pairs of slots
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t y = w ? u[j][0].y : u[j][0].x, z = w ? u[j][1].y : u[j][1].x;
                        widen<FMT>(__byte_perm(y, z, 0x5140), v[j][0], v[j][1]);
                        widen<FMT>(__byte_perm(y, z, 0x7362), v[j][2], v[j][3]);
                    }
                    if constexpr (FEW) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float(&acc)[4] = F32 ? x[F32 ? 2 * w + i : 0] : o[hf * 4 + 2 * w + i];
                            if (F32)
                                mma_f16(acc, v[0][2 * i], v[0][2 * i + 1], v[1][2 * i], v[1][2 * i + 1], pb[F32 ? b : 0][0], pb[F32 ? b : 0][1]);
                            mma_f16(acc, v[0][2 * i], v[0][2 * i + 1], v[1][2 * i], v[1][2 * i + 1], pa[b][0], pa[b][1]);
                        }
                    } else {
                        constexpr int X = FEW ? 0 : 1;  // keeps the indices of the other form in range
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float(&acc)[4] = F32 ? x[F32 ? X * (w * 4 + i) : 0] : o[X * (hf * 8 + w * 4 + i)];
                            const uint32_t(&p)[FEW ? 2 : 4] = pb[F32 ? b : 0];
                            if (F32) mma_f16(acc, p[0], p[1], p[2 * X], p[3 * X], v[0][i], v[1][i]);
                            mma_f16(acc, pa[b][0], pa[b][1], pa[b][2 * X], pa[b][3 * X], v[0][i], v[1][i]);
                        }
                    }
                }
            }
            if (F32)
#pragma unroll
                for (int j = 0; j < NO; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[hf * NO + j][i] += x[F32 ? j : 0][i];
        }
    }

    LDEV void finish() {
#pragma unroll
        for (int e = 0; e < 2; ++e) l[e] = over_row(l[e], [](float x, float y) { return x + y; });
    }

    // row e of this lane to the output: the unit is complete
    LDEV void store(const Kv8AttendArgs& a, const Seq& s, int h, int r, int e, bool vec) const {
        const int i = query_of(r, a.group), t = s.first + i, hq = h * a.group + r - i * a.group;
        const float inv = l[e] == 0.0f ? 0.0f : 1.0f / l[e], up = pow2i(R[e] - 14.0f);
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
            const int64_t at = (int64_t)t * a.out.row_stride + (int64_t)hq * a.out.head_stride + col_of(hf);
            float v[RUN];
#pragma unroll
            for (int k = 0; k < RUN; ++k) v[k] = l[e] == 0.0f ? 0.0f : value(hf, k, e) * inv * up;
            if (F32) {
                float* dst = static_cast<float*>(a.out.ptr) + at;
                if (vec) {
#pragma unroll
                    for (int k = 0; k < RUN; k += 4)
                        *reinterpret_cast<float4*>(dst + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                } else {
#pragma unroll
                    for (int k = 0; k < RUN; ++k) dst[k] = v[k];
                }
            } else {
                uint16_t* dst = static_cast<uint16_t*>(a.out.ptr) + at;
                uint32_t w[RUN / 2];
#pragma unroll
                for (int k = 0; k < RUN / 2; ++k) w[k] = two_bf16(v[2 * k], v[2 * k + 1]);
                if (vec) {
#pragma unroll
                    for (int k = 0; k < RUN / 8; ++k)
                        reinterpret_cast<uint4*>(dst)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                } else {
#pragma unroll
                    for (int k = 0; k < RUN; ++k) dst[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
                }
            }
        }
        if (a.norm && first_of_row()) a.norm[(int64_t)t * a.heads + hq] = make_float2(M[e], inv);
    }

    // row e of this lane as a partial result
    LDEV void leave(float* p, int e) const {
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf)
#pragma unroll
            for (int k = 0; k < RUN; k += 4)
                *reinterpret_cast<float4*>(p + col_of(hf) + k) =
                    make_float4(value(hf, k, e), value(hf, k + 1, e), value(hf, k + 2, e), value(hf, k + 3, e));
        if (first_of_row()) *reinterpret_cast<float4*>(p + D) = make_float4(M[e], R[e], l[e], 0.0f);
    }
};

// ---- partial results ----------------------------------------------------------------------------------------------------
// A share that holds a part of a unit leaves that part's sums: in its slot 0 when the unit began in an earlier share, in
// its slot 1 when it began in this one and goes on in the next.

// The parts of one row, `n` (at most 32) of them at at(0), at(1), ..., added to a warp's running sums.
template <int D, typename At>
LDEV void add_parts(int n, At at, float (&o)[D / 32], float& M, float& R, float& l) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    float4 m = make_float4(kFar, kLow, 0.0f, 0.0f);
    if (lane < n) m = *reinterpret_cast<const float4*>(at(lane) + D);
    float Mn = fmaxf(M, m.x), Rn = fmaxf(M + R, m.x + m.y);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
        Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, x));
        Rn = fmaxf(Rn, __shfl_xor_sync(0xffffffffu, Rn, x));
    }
    Rn = far_off(Mn) ? fmaxf(R + (M - Mn), warp_max(m.y + (m.x - Mn))) : Rn - Mn;
    l = l * pow2i(M - Mn) + warp_sum(m.z * pow2i(m.x - Mn));
    const float old = pow2i((M - Mn) + (R - Rn)), mine = pow2i((m.x - Mn) + (m.y - Rn));
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] *= old;
    for (int i0 = 0; i0 < n; i0 += 4) {  // four parts' loads on their way at a time
        float x[4][V];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int e = 0; e < V; ++e) x[i][e] = 0.0f;
            if (i0 + i < n) {
                const float* p = at(i0 + i) + lane * V;
                if (V == 2)
                    *reinterpret_cast<float2*>(x[i]) = *reinterpret_cast<const float2*>(p);
                else
                    *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(p);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = __shfl_sync(0xffffffffu, mine, i0 + i);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (i0 + i < n) o[e] += x[i][e] * f;
        }
    }
    M = Mn;
    R = Rn;
}

// the merged row to the output: lane l holds D / 32 consecutive values
template <int D, bool F32>
LDEV void store_merged(const Kv8AttendArgs& a, int first, int h, int r, const float (&o)[D / 32], float M, float R, float l) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31, i = query_of(r, a.group), t = first + i, hq = h * a.group + r - i * a.group;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l, up = pow2i(R - 14.0f);
    const int64_t at = (int64_t)t * a.out.row_stride + (int64_t)hq * a.out.head_stride + lane * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float v = l == 0.0f ? 0.0f : o[e] * inv * up;
        if (F32)
            static_cast<float*>(a.out.ptr)[at + e] = v;
        else
            static_cast<uint16_t*>(a.out.ptr)[at + e] = f32_to_bf16_rne(v);
    }
    if (a.norm && lane == 0) a.norm[(int64_t)t * a.heads + hq] = make_float2(M, inv);
}

// ---- one pass over the cache ----------------------------------------------------------------------------------------------
// A group of RW warps walks its part of the list through its own ring of stages, each a chunk of K and of V codes and
// their scales brought in by bulk copies; its first warp's lane 0 issues them.  With one warp a group (RW 1) the CTA takes
// one share, its warps equal parts of it in order, and puts together at its end what they cut.
// Few rows are bound by memory: 262 to 291 us by card at 96 sequences of 7192 to 8192 slots with 32 heads of 128 (1.5 GB, 5.8
// to 5.2 TB/s), 50 us at 4 of 57,618 to 65,537 with 24 heads of 64 (248 MB, 5.0 TB/s).  Many rows are bound by the instructions
// that widen codes for each 16 rows: 28 us at 224 queries over 8 sequences of 2048 slots (98 TFLOP/s).  A list too short for
// the card costs 7.7 us, of which 4.5 pass before the first codes arrive (lengths, then page numbers, then copies).
// bf16 calls: the weighted sums of a part of the list stay in the matrix unit's accumulators, which cut off what is below f32
// (at most 2^-23 of the sum for each block of 16 slots, below 2^-14 over the 311 blocks that a warp takes of 96 sequences
// of 8192 slots with 8 KV heads of 128; the output is rounded to 2^-9).  f32 calls start a sum for each chunk and add the
// chunks with rounding.

// what a warp of a CTA with one warp a group leaves behind
struct Ends {
    bool mid, closes, tail;  // its part began inside a unit; ended it; ended inside a unit that it began
    int hh, ht, hn, hfirst;  // KV head, row tile, queries and first query row of the one it began inside
    int th, tt, tn, tfirst;  // and of the one it left open
};

template <int FMT, int D, bool FEW, int RW, bool F32>
__global__ void __launch_bounds__(Shape<D, FEW, RW>::THREADS, 1) kv8_attend_kernel(const __grid_constant__ Kv8AttendArgs a) {
    using SH = Shape<D, FEW, RW>;
    constexpr int TOK = SH::TOK, NB = SH::NB, ST = SH::STAGES, CPP = SH::CPP, TILE = SH::TILE, STAGE = 2 * SH::CHUNK;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Ends ends[RW == 1 ? SH::WARPS : 1];
    pdl_wait();
    pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp / RW, wrow = warp % RW;
    unsigned char* data = smem + (size_t)wg * ST * STAGE;
    float* scales = reinterpret_cast<float*>(smem + (size_t)SH::GROUPS * ST * STAGE) + wg * ST * 8;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (size_t)SH::GROUPS * ST * (STAGE + 8 * sizeof(float)));
    uint64_t *full = bars + wg * ST, *empty = bars + ((SH::BARS - 1) * SH::GROUPS + wg) * ST;
    int* flags = reinterpret_cast<int*>(bars + SH::BARS * SH::GROUPS * ST);
    int* there = flags + wg * ST;
    float* heads = reinterpret_cast<float*>(flags + SH::GROUPS * ST);
    if (wrow == 0 && lane == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(full + i, 1);
            if (RW > 1) mbar_init(empty + i, RW);
        }
        if (RW == 1) ends[warp].mid = ends[warp].tail = false;
    }

    // this group's part [beg, end) of the list; the list's offset of each sequence goes to the merge kernel
    const int H = a.kv.kv_heads;
    int beg = 0, end = 0, total = 0, sb, sbase = 0;
    find_part<SH::THREADS>(
        reinterpret_cast<int*>(smem), a.kv.n_seqs,
        [&](int b) {
            const Seq s = seq_of<TOK, TILE>(a, b);
            return H * s.tiles * s.chunks;
        },
        [&](int sum) {
            if (RW == 1) {
                const int per = share_of(sum, gridDim.x, SH::LEAST), lo = min(sum, (int)blockIdx.x * per), hi = min(sum, lo + per);
                const int each = share_of(hi - lo, SH::WARPS, 1);
                beg = min(hi, lo + warp * each), end = min(hi, beg + each);
            } else {  // groups of one CTA are far apart in the list, so that a short one still uses every SM
                const int per = share_of(sum, gridDim.x * SH::GROUPS, SH::LEAST);
                beg = min(sum, (wg * (int)gridDim.x + (int)blockIdx.x) * per), end = min(sum, beg + per);
            }
            return beg;
        },
        [&](int b, int at) {
            if (blockIdx.x == 0) a.offset[b] = at;
        },
        total, sb, sbase);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offset[a.kv.n_seqs] = total;
    const int group = wg * (int)gridDim.x + (int)blockIdx.x, count = end - beg;
    if (RW > 1 && count == 0) return;
    const bool vo = vec_rows(a.out);
    if (count > 0) {
        struct Cursor {
            int b, h, tile, c;
            Seq s;
        } cur, iss;
        cur.b = sb;
        cur.s = seq_of<TOK, TILE>(a, sb);
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
                x.s = seq_of<TOK, TILE>(a, x.b);
            } while (x.s.tiles == 0);
        };

        const uint64_t policy = FEW ? read_once() : 0;
        // page numbers ahead of the issuing cursor: lane i holds page pbase + i of sequence pb
        int pb = -1, pbase = 0, pnum = 0;
        int seen = 0;  // chunks of the issuing cursor's unit that any of its rows sees
        auto limit = [&]() {
            const int last = min((iss.tile + 1) * TILE, iss.s.n * a.group) - 1;
            seen = (visible(a, iss.s, last) + TOK - 1) / TOK;
        };
        auto issue = [&](int st) {  // the group's first warp: the cursor's chunk into stage st
            const int pg = iss.c / CPP;
            if (iss.b != pb || pg < pbase || pg >= pbase + 32) {
                pb = iss.b, pbase = pg;
                const int pages = (iss.s.len + kKv8Page - 1) / kKv8Page;
                pnum = pg + lane < pages ? a.kv.page_table[(int64_t)pb * a.kv.max_pages + pg + lane] : -1;
            }
            const int page = __shfl_sync(0xffffffffu, pnum, pg - pbase);
            if (lane == 0) {
                const bool ok = iss.c < seen && (unsigned)page < (unsigned)a.kv.num_pages;
                if (iss.c < seen && !ok) report(a.kv, LASTRO_KV8_BAD_PAGE);
                there[st] = ok;
                if (ok) {
                    const int64_t tile = (int64_t)page * H + iss.h;
                    const int64_t at = tile * kKv8Page * D + (int64_t)(iss.c % CPP) * SH::CHUNK;
                    unsigned char* dst = data + (size_t)st * STAGE;
                    mbar_expect_tx(full + st, STAGE + 32);
                    const uint8_t *k = static_cast<const uint8_t*>(a.kv.k) + at, *v = static_cast<const uint8_t*>(a.kv.v) + at;
                    if (FEW) {  // read once, and the scores kept meanwhile stay in L2 for the weights
                        bulk_g2s_once(dst, k, SH::CHUNK, full + st, policy);
                        bulk_g2s_once(dst + SH::CHUNK, v, SH::CHUNK, full + st, policy);
                    } else {
                        bulk_g2s(dst, k, SH::CHUNK, full + st);
                        bulk_g2s(dst + SH::CHUNK, v, SH::CHUNK, full + st);
                    }
                    bulk_g2s(scales + st * 8, a.kv.k_scale + tile * kKv8Blocks, 16, full + st);
                    bulk_g2s(scales + st * 8 + 4, a.kv.v_scale + tile * kKv8Blocks, 16, full + st);
                } else {
                    mbar_arrive(full + st);
                }
            }
            advance(iss);
            if (iss.c == 0) limit();
        };
        // the rows' loads go out first: they and the page numbers are on their way together
        const bool vq = vec_rows(a.q);
        WarpRows<FMT, D, FEW, F32> rows;
        QRaw<D, FEW ? 1 : 2, F32> raw;
        int row0 = 0, vmin = 0, nrows = 0;  // the warp's first row of the unit, what it sees, and the rows from there on
        bool from0 = false;                 // the unit began in this part
        auto fetch_unit = [&]() { raw.fetch(a, cur.s, cur.h, cur.tile * TILE + wrow * SH::ROWS, vq); };
        auto begin_unit = [&]() {
            row0 = cur.tile * TILE + wrow * SH::ROWS;
            nrows = cur.s.n * a.group - row0;
            from0 = cur.c == 0;
            if (nrows <= 0) return;
            vmin = visible(a, cur.s, row0);
            rows.begin(a, cur.s, row0, raw);
        };
        fetch_unit();
        limit();
        if (wrow == 0)
            for (int i = 0; i < min(ST, count); ++i) issue(i);
        begin_unit();

        bool alive = true;
        for (int it = 0; it < count; ++it) {
            const int st = it % ST, ph = (it / ST) & 1;
            alive = mbar_wait(full + st, ph, a.kv.status, LASTRO_KV8_BAD_WAIT);
            if (!alive) break;
            if (nrows > 0) {
                const unsigned char* sk = data + (size_t)st * STAGE;
                const float* sc = scales + st * 8 + (cur.c % CPP) * NB;
                const int t0 = cur.c * TOK;
                float* keep = FEW && a.scores ? a.scores + (int64_t)(beg + it) * a.score_rows * TOK : nullptr;
                if (!there[st]) {
                    for (int i = lane; keep && i < nrows * TOK; i += 32) keep[i] = -INFINITY;
                } else if (t0 + TOK <= vmin)
                    rows.template consume<true, NB>(sk, sk + SH::CHUNK, sc, sc + 4, t0, cur.s.len, keep, nrows);
                else
                    rows.template consume<false, NB>(sk, sk + SH::CHUNK, sc, sc + 4, t0, cur.s.len, keep, nrows);
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
                const Cursor was = cur;
                if (it + 1 < count) {
                    advance(cur);
                    fetch_unit();
                }
                if (nrows > 0) {
                    rows.finish();
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = rows.row_of(e);
                        if (r >= nrows) continue;
                        if (last && from0)
                            rows.store(a, was.s, was.h, row0 + r, e, vo);
                        else if (RW > 1)
                            rows.leave(a.part + (((int64_t)group * 2 + from0) * TILE + wrow * SH::ROWS + r) * SH::PART, e);
                        else if (from0)  // its ring is empty by now
                            rows.leave(reinterpret_cast<float*>(data) + r * SH::PART, e);
                        else
                            rows.leave(heads + (warp * SH::ROWS + r) * SH::PART, e);
                    }
                }
                if (RW == 1 && lane == 0 && !(last && from0)) {
                    Ends& x = ends[warp];
                    if (from0)
                        x.tail = true, x.th = was.h, x.tt = was.tile, x.tn = was.s.n, x.tfirst = was.s.first;
                    else
                        x.mid = true, x.closes = last, x.hh = was.h, x.ht = was.tile, x.hn = was.s.n, x.hfirst = was.s.first;
                }
                if (it + 1 < count) begin_unit();
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
    const Ends mine = ends[lane & (SH::WARPS - 1)];
    const unsigned low = (1u << SH::WARPS) - 1, mids = __ballot_sync(0xffffffffu, mine.mid) & low;
    const unsigned tails = __ballot_sync(0xffffffffu, mine.tail) & low, closes = __ballot_sync(0xffffffffu, mine.mid && mine.closes) & low;
    int task = 0;  // rows of the runs, dealt to the warps
    for (unsigned starts = tails << 1 | (mids & 1); starts; starts &= starts - 1) {
        const int which = __ffs(starts) - 2;
        // warps which + 1, ... that began inside it, up to the one that closes it
        const unsigned after = mids >> (which + 1), ended = closes >> (which + 1);
        int n = __ffs(~after) - 1;
        const bool closed = (ended & ((1u << n) - 1)) != 0;
        if (closed) n = __ffs(ended);
        n += which >= 0;
        const Ends& x = ends[max(which, 0)];
        const int h = which < 0 ? x.hh : x.th, tile = which < 0 ? x.ht : x.tt, row0 = which < 0 ? x.hfirst : x.tfirst;
        const int first = max(which, 0), nrows = min(SH::ROWS, (which < 0 ? x.hn : x.tn) * a.group - tile * TILE);
        for (int r = 0; r < nrows; ++r, ++task) {
            if (task % SH::WARPS != warp) continue;
            float o[D / 32] = {}, M = kFar, R = kLow, l = 0.0f;
            add_parts<D>(n, [&](int i) -> const float* {
                if (which >= 0 && i == 0)
                    return reinterpret_cast<const float*>(smem + (size_t)first * ST * STAGE) + r * SH::PART;
                return heads + ((first + i) * SH::ROWS + r) * SH::PART;
            }, o, M, R, l);
            if (which >= 0 && closed) {
                store_merged<D, F32>(a, row0, h, tile * TILE + r, o, M, R, l);
            } else {
                float* p = a.part + (((int64_t)blockIdx.x * 2 + (which >= 0)) * TILE + r) * SH::PART;
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
// One warp per query row and head whose unit was cut between shares, in the order of the shares.  3.2 us for a handful of rows
// (three dependent loads), 5.5 us for 5376.
template <int D, bool FEW, int RW, bool F32>
__global__ void __launch_bounds__(kThreads) kv8_merge_kernel(const __grid_constant__ Kv8AttendArgs a) {
    using SH = Shape<D, FEW, RW>;
    pdl_wait();
    pdl_launch();
    const int b = blockIdx.y;
    const Seq s = seq_of<SH::TOK, SH::TILE>(a, b);
    const int per = share_of(a.offset[a.kv.n_seqs], a.shares, SH::LEAST), base = a.offset[b];
    for (int u = blockIdx.x * kWarps + (threadIdx.x >> 5); u < s.n * a.heads; u += gridDim.x * kWarps) {
        const int i = u / a.heads, hq = u - i * a.heads, h = hq / a.group, r = i * a.group + hq - h * a.group, tile = r / SH::TILE;
        const int first = base + (h * s.tiles + tile) * s.chunks, g0 = first / per, g1 = (first + s.chunks - 1) / per;
        if (g0 == g1) continue;
        float o[D / 32] = {}, M = kFar, R = kLow, l = 0.0f;
        for (int g = g0; g <= g1; g += 32)
            add_parts<D>(min(32, g1 + 1 - g), [&](int k) {
                return a.part + (((int64_t)(g + k) * 2 + (g + k == g0)) * SH::TILE + r - tile * SH::TILE) * SH::PART;
            }, o, M, R, l);
        store_merged<D, F32>(a, s.first, h, r, o, M, R, l);
    }
}

// ---- accumulated weights, from stored scores ------------------------------------------------------------------------------
// With few query rows the pass over the cache also leaves its scores (4 bytes a row and slot, against d bytes of K), and
// the weights are one elementwise pass over them: a thread takes four slots.  The kernel merges the shares too: every CTA
// needs the merged sums of its KV head's rows, and the head's first CTA their outputs.  14 us at 4 sequences of 57,618 to 65,537
// slots, 8 KV heads and 3 rows (39 MB of scores and masses), 3.7 us where there is next to nothing to do.
template <int D, bool F32>
__global__ void __launch_bounds__(128) kv8_weights_kernel(const __grid_constant__ Kv8AttendArgs a) {
    using SH = Shape<D, true, 1>;
    __shared__ float2 norms[SH::ROWS];
    pdl_wait();
    pdl_launch();
    const int b = blockIdx.z, h = blockIdx.y, H = a.kv.kv_heads, lane = threadIdx.x & 31;
    const Seq s = seq_of<SH::TOK, SH::TILE>(a, b);
    const int base = a.offset[b] + h * s.chunks, rows = s.n * a.group;
    const int per = share_of(a.offset[a.kv.n_seqs], a.shares, SH::LEAST), g0 = rows ? base / per : 0, g1 = rows ? (base + s.chunks - 1) / per : 0;
    if (blockIdx.x * 512 >= s.len && blockIdx.x > 0) return;
    for (int r = threadIdx.x >> 5; r < rows; r += 4) {
        if (g0 == g1) {
            const int i = query_of(r, a.group);
            if (lane == 0) norms[r] = a.norm[(int64_t)(s.first + i) * a.heads + h * a.group + r - i * a.group];
            continue;
        }
        const auto part = [&](int g) { return a.part + (((int64_t)g * 2 + (g == g0)) * SH::TILE + r) * SH::PART; };
        float o[D / 32] = {}, M = kFar, R = kLow, l = 0.0f;
        for (int g = g0; g <= g1; g += 32) {
            const int n = min(32, g1 + 1 - g);
            if (blockIdx.x == 0) {
                add_parts<D>(n, [&](int k) { return part(g + k); }, o, M, R, l);
            } else {
                const float4 m = lane < n ? *reinterpret_cast<const float4*>(part(g + lane) + D) : make_float4(kFar, kLow, 0.0f, 0.0f);
                const float Mn = fmaxf(M, warp_max(m.x));
                l = l * pow2i(M - Mn) + warp_sum(m.z * pow2i(m.x - Mn));
                M = Mn;
            }
        }
        if (blockIdx.x == 0) store_merged<D, F32>(a, s.first, h, r, o, M, R, l);
        if (lane == 0) norms[r] = make_float2(M, l == 0.0f ? 0.0f : 1.0f / l);
    }
    __syncthreads();
    float2 norm[SH::ROWS];
#pragma unroll
    for (int r = 0; r < SH::ROWS; ++r)
        if (r < rows) norm[r] = norms[r];
    const int64_t at = ((int64_t)b * H + h) * a.mass_stride;
    const bool vec = ((reinterpret_cast<uintptr_t>(a.mass_out + at) | reinterpret_cast<uintptr_t>(a.mass_in ? a.mass_in + at : nullptr)) & 15) == 0;
    for (int t = (blockIdx.x * 128 + threadIdx.x) * 4; t < s.len; t += gridDim.x * 512) {
        float sum[4] = {};
        if (rows > 0) {
            const float* src = a.scores + (int64_t)(base + t / SH::TOK) * a.score_rows * SH::TOK + t % SH::TOK;
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < rows) {
                    const float4 v = *reinterpret_cast<const float4*>(src + r * SH::TOK);
                    // the row's sum may be NaN, which is for the slots it sees
                    const auto add = [&](float& to, float x) {
                        if (x != -INFINITY) to = fmaf(ex2(x - norm[r].x), norm[r].y, to);
                    };
                    add(sum[0], v.x), add(sum[1], v.y), add(sum[2], v.z), add(sum[3], v.w);
                }
        }
        if (vec && t + 4 <= s.len) {
            float4 m = a.mass_in ? *reinterpret_cast<const float4*>(a.mass_in + at + t) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            *reinterpret_cast<float4*>(a.mass_out + at + t) = make_float4(m.x + sum[0], m.y + sum[1], m.z + sum[2], m.w + sum[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t + i < s.len) a.mass_out[at + t + i] = (a.mass_in ? a.mass_in[at + t + i] : 0.0f) + sum[i];
        }
    }
}

// ---- accumulated weights, from K ------------------------------------------------------------------------------------------
// More query rows: the scores are computed again, with the finished softmax sums at hand.  The chunks of each sequence and
// KV head are dealt to the warps of gridDim.x CTAs; a warp holds a chunk's K in registers as f16 and runs the query tiles
// past it from shared memory.  Two CTAs an SM, with half the chunk that one would take: latency is what bounds it (15 us at 224
// queries over 8 sequences of 2048 slots, 96 rows a KV head).
constexpr int kMassTiles = kWarps, kMassChunk = 2048;  // query tiles in shared memory, one loaded by each warp; K codes a warp holds

template <int D, bool F32>
constexpr size_t mass_smem() {
    return (size_t)kMassTiles * (D / 16) * 32 * 16 * (F32 ? 2 : 1) + kMassTiles * 16 * 4 * 4 + kWarps * 64 * 4;
}

template <int FMT, int D, bool F32>
__global__ void __launch_bounds__(kThreads, 2) kv8_mass_kernel(const __grid_constant__ Kv8AttendArgs a) {
    constexpr int TOK = kMassChunk / D, NB = TOK / kKv8Block, CPP = kKv8Page / TOK, KS = D / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    pdl_wait();
    pdl_launch();
    uint4* qs = reinterpret_cast<uint4*>(smem);  // [tile][ks][lane], first terms then second ones
    float2* rnorm = reinterpret_cast<float2*>(qs + (size_t)kMassTiles * KS * 32 * (F32 ? 2 : 1));
    float* rfac = reinterpret_cast<float*>(rnorm + kMassTiles * 16);
    int* rvis = reinterpret_cast<int*>(rfac + kMassTiles * 16);
    float* sums = reinterpret_cast<float*>(rvis + kMassTiles * 16) + (threadIdx.x >> 5) * 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, c4 = lane & 3, H = a.kv.kv_heads;
    const bool vq = vec_rows(a.q);
    const int b = blockIdx.z, h = blockIdx.y;
    const Seq s = seq_of<TOK, 16>(a, b);
    const int chunks = (s.len + TOK - 1) / TOK, c0 = blockIdx.x * kWarps, rows = s.n * a.group, tiles = s.tiles;
    if (c0 >= chunks) return;
    for (int tb = 0; tb < max(1, tiles); tb += kMassTiles) {
        const int nt = min(kMassTiles, tiles - tb);
        // a chunk's K codes as they are stored: the first is on its way while the rows are made ready
        int page = -1;
        uint32_t w[NB][2][KS];
        float ks_next[NB];
        auto load_k = [&](int c) {
            page = c < chunks ? page_of(a.kv, b, c * TOK) : -1;
            if (page < 0) return;
            const int64_t tile = (int64_t)page * H + h;
            const uint8_t* kp = static_cast<const uint8_t*>(a.kv.k) + tile * kKv8Page * D + (int64_t)(c % CPP) * kMassChunk;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                ks_next[n] = a.kv.k_scale[tile * kKv8Blocks + (c % CPP) * NB + n];
#pragma unroll
                for (int j = 0; j < 2; ++j) k_codes<D>(kp + (n * 16 + slot_of(gq >> 1, gq & 1, j)) * D, w[n][j]);
            }
        };
        load_k(c0 + warp);
        __syncthreads();  // the tiles before these are done with
        if (warp < nt) {
            const int row0 = (tb + warp) * 16;
            QFrag<D, 2, F32> q;
            QRaw<D, 2, F32> raw;
            raw.fetch(a, s, h, row0, vq);
            q.convert(raw, a.scale);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                qs[(warp * KS + k) * 32 + lane] = make_uint4(q.hi[k][0], q.hi[k][1], q.hi[k][2], q.hi[k][3]);
                const uint32_t(&lo)[4] = q.lo[F32 ? k : 0];
                if (F32) qs[((kMassTiles + warp) * KS + k) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            if (c4 == 0)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = row0 + gq + 8 * e, at = warp * 16 + gq + 8 * e, i = r / a.group;
                    rfac[at] = q.factor[e];
                    rvis[at] = visible(a, s, r);
                    rnorm[at] = r < rows ? a.norm[(int64_t)(s.first + i) * a.heads + h * a.group + r - i * a.group] : make_float2(0.0f, 0.0f);
                }
        }
        __syncthreads();
        for (int c = c0 + warp; c < chunks; c += gridDim.x * kWarps) {
            float sum[NB][2][2] = {};
            if (page >= 0 && nt > 0) {
                uint32_t kf[NB][2][KS][2];
                float ks[NB];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    ks[n] = ks_next[n];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int k = 0; k < KS; ++k) widen<FMT>(w[n][j][k], kf[n][j][k][0], kf[n][j][k][1]);
                }
                for (int t = 0; t < nt; ++t) {
                    const bool whole = c * TOK + TOK <= rvis[t * 16];
                    uint4 q[KS], p[F32 ? KS : 1];
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        q[k] = qs[(t * KS + k) * 32 + lane];
                        if (F32) p[F32 ? k : 0] = qs[((kMassTiles + t) * KS + k) * 32 + lane];
                    }
                    const float fac[2] = {rfac[t * 16 + gq], rfac[t * 16 + gq + 8]};
                    const float2 norm[2] = {rnorm[t * 16 + gq], rnorm[t * 16 + gq + 8]};
                    const int vis[2] = {rvis[t * 16 + gq], rvis[t * 16 + gq + 8]};
                    const bool far = __any_sync(0xffffffffu, far_off(norm[0].x) || far_off(norm[1].x));  // as the first pass rounded
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float x[4];
                            score_sum<KS, F32>(x, [&](float (&y)[4], int k, bool second) {
                                const uint4& r = second ? p[F32 ? k : 0] : q[k];
                                mma_f16(y, r.x, r.y, r.z, r.w, kf[n][j][k][0], kf[n][j][k][1]);
                            });
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float f = fac[i >> 1] * ks[n], M = norm[i >> 1].x;
                                const float v = ex2(far ? __fmul_rn(x[i], f) - M : fmaf(x[i], f, -M));
                                if (whole || c * TOK + n * 16 + slot_of(c4, i & 1, j) < vis[i >> 1])
                                    sum[n][j][i & 1] = fmaf(v, norm[i >> 1].y, sum[n][j][i & 1]);
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
            for (int i = lane; i < TOK; i += 32) {
                const int t = c * TOK + i;
                const int64_t at = ((int64_t)b * H + h) * a.mass_stride + t;
                if (t < s.len) a.mass_out[at] = (in ? in[at] : 0.0f) + sums[i];
            }
            __syncwarp();
            load_k(c + gridDim.x * kWarps);
        }
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

struct AttendLaunch {
    Kv8AttendArgs a;
    cudaStream_t s;

    template <int FMT, int D, bool FEW, int RW, bool F32>
    cudaError_t go() {
        using SH = Shape<D, FEW, RW>;
        a.shares = sm_count() * (RW == 1 ? 1 : SH::GROUPS);
        cudaError_t e = kv8_launch<kv8_attend_kernel<FMT, D, FEW, RW, F32>, SH::SMEM>(dim3(sm_count()), SH::THREADS, SH::SMEM, 1, s, a);
        if (e != cudaSuccess) return e;
        if (a.scores) {
            // at most 64 CTAs a head: 16, 32, 64 and 128 take 81, 70.6, 67.5 and 67.4 us in all at 4 sequences of 65537, the same elsewhere
            const dim3 blocks(min(64, (a.kv.max_pages * kKv8Page + 511) / 512), a.kv.kv_heads, a.kv.n_seqs);
            return kv8_launch<kv8_weights_kernel<D, F32>, 0>(blocks, 128, 0, 1, s, a);
        }
        const int64_t rows = (int64_t)a.max_new * a.heads;
        const dim3 grid((unsigned)max((int64_t)1, min((int64_t)1024, (rows + kWarps - 1) / kWarps)), a.kv.n_seqs);
        e = kv8_launch<kv8_merge_kernel<D, FEW, RW, F32>, 0>(grid, kThreads, 0, 1, s, a);
        if (e != cudaSuccess || !a.mass_out) return e;
        const int units = a.kv.kv_heads * a.kv.n_seqs, most = (a.kv.max_pages * (kKv8Page * D / kMassChunk) + kWarps - 1) / kWarps;
        const dim3 parts(max(1, min((2 * sm_count() + units - 1) / units, most)), a.kv.kv_heads, a.kv.n_seqs);
        return kv8_launch<kv8_mass_kernel<FMT, D, F32>, mass_smem<D, F32>()>(parts, kThreads, mass_smem<D, F32>(), 1, s, a);
    }
    template <int FMT, int D, bool FEW, int RW>
    cudaError_t by_type() {
        return a.q.dtype == LASTRO_DTYPE_F32 ? go<FMT, D, FEW, RW, true>() : go<FMT, D, FEW, RW, false>();
    }
    template <int FMT, int D>
    cudaError_t run() {
        switch (row_warps((int64_t)a.max_new * a.group)) {
        case 0: return by_type<FMT, D, true, 1>();
        case 1: return by_type<FMT, D, false, 1>();
        default: return by_type<FMT, D, false, 2>();
        }
    }
};

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

size_t kv8_attend_workspace(const lastro_kv8& kv, int heads, int max_new, bool with_mass, Kv8AttendArgs* a, void* base) {
    const int64_t rows = (int64_t)max_new * (heads / kv.kv_heads);
    const int rw = row_warps(rows);
    const size_t row = (kv.head_dim + 4) * sizeof(float), shares = (size_t)sm_count() * (rw <= 1 ? 1 : 8 / rw);
    const size_t offset = align16(((size_t)kv.n_seqs + 1) * sizeof(int32_t));
    const size_t part = shares * 2 * (rw ? rw * 16 : 8) * row;
    const size_t norm = with_mass ? align16((size_t)kv.n_seqs * max_new * heads * sizeof(float2)) : 0;
    // kept scores save the second pass over K; past 1 GiB of them K is read again instead
    size_t scores = with_mass && rw == 0 ? (size_t)kv.n_seqs * kv.kv_heads * kv.max_pages * kKv8Page * rows * sizeof(float) : 0;
    if (scores > ((size_t)1 << 30)) scores = 0;
    if (a) {
        unsigned char* p = static_cast<unsigned char*>(base);
        a->offset = reinterpret_cast<int32_t*>(p);
        a->part = reinterpret_cast<float*>(p + offset);
        a->norm = with_mass ? reinterpret_cast<float2*>(p + offset + part) : nullptr;
        a->scores = scores ? reinterpret_cast<float*>(p + offset + part + norm) : nullptr;
        a->score_rows = (int32_t)rows;
    }
    return offset + part + norm + scores;
}

int64_t kv8_attend_items(const lastro_kv8& kv, int heads, int max_new) {
    const int64_t rows = (int64_t)max_new * (heads / kv.kv_heads);
    const int rw = row_warps(rows), tile = rw ? rw * 16 : 8;
    const double chunks = (double)kv.max_pages * (kKv8Page * kv.head_dim / 4096);
    const double items = kv.n_seqs * (double)kv.kv_heads * chunks * ((rows + tile - 1) / tile + 1);
    return items < 9e18 ? (int64_t)items : INT64_MAX;
}

cudaError_t launch_kv8_attend(const Kv8AttendArgs& a, cudaStream_t s) { return kv8_by_shape(a.kv, AttendLaunch{a, s}); }

}  // namespace lastro
