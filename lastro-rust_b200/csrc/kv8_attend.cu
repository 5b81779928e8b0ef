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

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kChunkBytes = 4096;                     // K (or V) codes of one pipeline stage: 64 slots of d 64, 32 of d 128
constexpr int kStageBytes = 2 * kChunkBytes;
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

// d += a (16x16, row) * b (16x8, col), f16 operands, f32 accumulators
LDEV void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

LDEV int64_t share(int64_t total, int i, int n) { return total * i / n; }

LDEV int64_t warp_sum64(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The sequence whose items hold list item `pos` (-1: none) and where its items start; every lane of a warp calls it.
// `work(b)` is the number of items of sequence b, `note(b, at)` is told where each one passed starts.
template <typename Work, typename Note>
LDEV int seek(int n_seqs, int64_t pos, bool all, int64_t& base, Work work, Note note) {
    const int lane = threadIdx.x & 31;
    int found = -1;
    int64_t sum = 0;
    for (int b0 = 0; b0 < n_seqs; b0 += 32) {
        const int b = b0 + lane;
        const int64_t w = b < n_seqs ? work(b) : 0;
        int64_t x = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const int64_t at = sum + x - w;
        if (b < n_seqs) note(b, at);
        const unsigned hit = __ballot_sync(0xffffffffu, w > 0 && at <= pos && pos < at + w);
        if (hit) {
            found = b0 + __ffs(hit) - 1;
            base = __shfl_sync(0xffffffffu, at, __ffs(hit) - 1);
            if (!all) return found;
        }
        sum += __shfl_sync(0xffffffffu, x, 31);
    }
    return found;
}

// ---- query rows ---------------------------------------------------------------------------------------------------------
// The A operand of 16 rows (row r is query r / group, head r % group of the KV head) and each row's factor from the raw
// product to the score in powers of two.  A row is scaled by a power of two to a largest magnitude in [2^14, 2^15), which
// puts a bf16 value exactly into f16 down to 2^-28 of that magnitude; f32 rows take a second term.
template <int D, bool F32>
struct QFrag {
    static constexpr int KS = D / 16;
    uint32_t hi[KS][4], lo[F32 ? KS : 1][4];
    float factor[2];

    LDEV void load(const Kv8AttendArgs& a, const Seq& s, int h, int row0, bool vec, int lane) {
        const int gq = lane >> 2, c = lane & 3;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
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
            const float up = finite ? __uint_as_float((uint32_t)(k + 127) << 23) : 0.0f;
            factor[e] = finite ? a.scale * 1.44269504088896340736f * __uint_as_float((uint32_t)(127 - k) << 23)
                               : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int hf = 0; hf < D / 64; ++hf)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float u = finite ? x[hf][4 * q + 2 * w] * up : 0.0f;
                        const float v = finite ? x[hf][4 * q + 2 * w + 1] * up : 0.0f;
                        hi[hf * 4 + q][e + 2 * w] = pack_f16(u, v);
                        if (F32) lo[F32 ? hf * 4 + q : 0][e + 2 * w] = rest_f16(hi[hf * 4 + q][e + 2 * w], u, v);
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

// ---- workspace ----------------------------------------------------------------------------------------------------------
// [groups][2] partial results: slot 0 of a unit that began in an earlier share, slot 1 of one that ends in a later share
constexpr int part_floats(int D) { return D + 4; }  // sums, then the running maxima M and R and the sum l

// A row's running state: M the ceiling of the largest score so far (scores and M in powers of two), l the sum of
// 2^(score - M), R the ceiling of the largest score plus its slot's V exponent, o the sum of 2^(score + 14 - R) v.  M
// and R are whole numbers, so bringing sums to new ones is exact, and R keeps the f16 weights in range whatever the
// blocks' scales: the heaviest contribution sits between 2^13 and 2^14.
template <int D, bool F32>
LDEV void store_row(const Kv8AttendArgs& a, const Seq& s, int h, int r, int lane, const float (&o)[D / 8][4], int e, float M,
                    float R, float l, bool vec) {
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

// ---- one pass over the cache ----------------------------------------------------------------------------------------------
// A group of RW warps (RW * 16 query rows) walks its share of the list through its own ring of stages, each 4 KB of K and
// of V codes and their scales brought in by bulk copies; its first warp's lane 0 issues them.
template <int D, int RW>
struct Ring {
    static constexpr int GROUPS = kWarps / RW, STAGES = RW == 1 ? 3 : RW == 2 ? 6 : 8;
    static constexpr size_t bytes = (size_t)GROUPS * STAGES * (kStageBytes + 8 * sizeof(float) + 16 + 16) + 128;
};

template <int FMT, int D, int RW, bool F32>
__global__ void __launch_bounds__(kThreads, 1) kv8_attend_kernel(const __grid_constant__ Kv8AttendArgs a) {
    using RG = Ring<D, RW>;
    constexpr int TOK = kChunkBytes / D, NB = TOK / kKv8Block, ST = RG::STAGES, CPP = kKv8Page / TOK;
    extern __shared__ unsigned char smem_raw[];
    pdl_wait();
    pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, c4 = lane & 3;
    const int wg = warp / RW, wrow = warp % RW;
    unsigned char* smem = smem_raw + ((128 - (smem_addr(smem_raw) & 127)) & 127);
    unsigned char* data = smem + (size_t)wg * ST * kStageBytes;
    unsigned char* tail = smem + (size_t)RG::GROUPS * ST * kStageBytes;
    float* scales = reinterpret_cast<float*>(tail) + wg * ST * 8;
    uint64_t* bars = reinterpret_cast<uint64_t*>(tail + (size_t)RG::GROUPS * ST * 8 * sizeof(float));
    uint64_t *full = bars + wg * ST, *empty = bars + (RG::GROUPS + wg) * ST;
    int* there = reinterpret_cast<int*>(bars + 2 * RG::GROUPS * ST) + wg * ST;
    if (wrow == 0 && lane == 0)
        for (int i = 0; i < ST; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, RW);
        }
    if (RW == 1)
        __syncwarp();
    else
        __syncthreads();

    // this group's share [beg, end) of the list; the list's offset of each sequence goes to the merge kernel
    const int groups = gridDim.x * RG::GROUPS, group = blockIdx.x * RG::GROUPS + wg;
    const int H = a.kv.kv_heads, tile_rows = 16 * RW;
    auto work = [&](int b) {
        const Seq s = seq_of<TOK>(a, b, tile_rows);
        return (int64_t)H * s.tiles * s.chunks;
    };
    int64_t total = 0, sbase = 0;
    for (int b = lane; b < a.kv.n_seqs; b += 32) total += work(b);
    total = warp_sum64(total);
    const int64_t beg = share(total, group, groups), end = share(total, group + 1, groups);
    const bool writes = blockIdx.x == 0 && warp == 0;  // the merge kernel takes the list's offsets from this warp
    const int sb = seek(a.kv.n_seqs, beg, writes, sbase, work, [&](int b, int64_t at) {
        if (writes) a.offset[b] = at;
    });
    if (writes && lane == 0) a.offset[a.kv.n_seqs] = total;
    const int count = (int)(end - beg);  // fits: the host bounds the list
    if (count <= 0) return;

    struct Cursor {
        int b, h, tile, c;
        Seq s;
    } cur, iss;
    cur.b = sb;
    cur.s = seq_of<TOK>(a, sb, tile_rows);
    {
        int64_t u = beg - sbase;
        cur.c = (int)(u % cur.s.chunks);
        u /= cur.s.chunks;
        cur.tile = (int)(u % cur.s.tiles);
        cur.h = (int)(u / cur.s.tiles);
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
    auto issue = [&](int st) {  // the group's first warp: the cursor's chunk into stage st
        const int pg = iss.c / CPP;
        if (iss.b != pb || pg < pbase || pg >= pbase + 32) {
            pb = iss.b, pbase = pg;
            const int pages = (iss.s.len + kKv8Page - 1) / kKv8Page;
            pnum = pg + lane < pages ? __ldg(a.kv.page_table + (int64_t)pb * a.kv.max_pages + pg + lane) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, pnum, pg - pbase);
        if (lane == 0) {
            const int last = min((iss.tile + 1) * tile_rows, iss.s.n * a.group) - 1;
            const bool seen = iss.c * TOK < visible(a, iss.s, last);  // by any row of the tile
            const bool ok = seen && (unsigned)page < (unsigned)a.kv.num_pages;
            if (seen && !ok) report(a.kv, LASTRO_KV8_BAD_PAGE);
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
    };
    if (wrow == 0)
        for (int i = 0; i < min(ST, count); ++i) issue(i);

    const bool vq = vec_rows(a.q), vo = vec_rows(a.out);
    QFrag<D, F32> q;
    float o[D / 8][4], M[2], R[2], l[2];
    int vis[2], vmin = 0, rows0 = 0;
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
        for (int e = 0; e < 2; ++e) {
            M[e] = R[e] = kFar;
            l[e] = 0.0f;
            vis[e] = visible(a, cur.s, rows0 + gq + 8 * e);
        }
        vmin = visible(a, cur.s, rows0);
        if (mine) q.load(a, cur.s, cur.h, rows0, vq, lane);
    };
    begin_unit();

    bool alive = true;
    for (int it = 0; it < count; ++it) {
        const int st = it % ST, ph = (it / ST) & 1;
        alive = mbar_wait(full + st, ph, a.kv.status, LASTRO_KV8_BAD_WAIT);
        if (!alive) break;
        if (mine && there[st]) {
            const unsigned char *sk = data + (size_t)st * kStageBytes, *sv = sk + kChunkBytes;
            const int t0 = cur.c * TOK, blk0 = (cur.c % CPP) * NB;
            const bool whole = t0 + TOK <= vmin;  // every row sees every slot of the chunk
            float s[NB][2][4];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float ks = scales[st * 8 + blk0 + b];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t w[D / 16];
                    k_codes<D>(sk + (b * 16 + slot_of(gq >> 1, gq & 1, j)) * D, lane, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[b][j][i] = 0.0f;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        uint32_t b0, b1;
                        widen<FMT>(w[k], b0, b1);
                        mma_f16(s[b][j], q.hi[k], b0, b1);
                        if (F32) mma_f16(s[b][j], q.lo[F32 ? k : 0], b0, b1);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[b][j][i] *= q.factor[i >> 1] * ks;
                        if (!whole && t0 + b * 16 + slot_of(c4, i & 1, j) >= vis[i >> 1]) s[b][j][i] = -INFINITY;
                    }
                }
            }
            float lsv[NB], Mn[2], Rn[2];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float vs = scales[st * 8 + 4 + blk0 + b];
                lsv[b] = vs != vs ? vs : (float)((int)(__float_as_uint(vs) >> 23) - 127);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                Mn[e] = M[e];
                Rn[e] = R[e];
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float m = ceilf(fmaxf(fmaxf(s[b][0][2 * e], s[b][0][2 * e + 1]), fmaxf(s[b][1][2 * e], s[b][1][2 * e + 1])));
                    Mn[e] = fmaxf(Mn[e], m);
                    Rn[e] = fmaxf(Rn[e], m + lsv[b]);
                }
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) {
                    Mn[e] = fmaxf(Mn[e], __shfl_xor_sync(0xffffffffu, Mn[e], x));
                    Rn[e] = fmaxf(Rn[e], __shfl_xor_sync(0xffffffffu, Rn[e], x));
                }
            }
            if (__any_sync(0xffffffffu, Mn[0] != M[0] || Mn[1] != M[1] || Rn[0] != R[0] || Rn[1] != R[1])) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    l[e] *= pow2i(M[e] - Mn[e]);
                    const float f = pow2i(R[e] - Rn[e]);
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        o[j][2 * e] *= f;
                        o[j][2 * e + 1] *= f;
                    }
                    M[e] = Mn[e];
                    R[e] = Rn[e];
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (!whole && __all_sync(0xffffffffu, t0 + b * 16 >= vis[1])) continue;  // no row sees it
                uint32_t ph_[4], pl_[4];
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = lsv[b] + 14.0f + M[e] - R[e];
                    f[e] = x != x ? x : pow2i(x);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float p0 = ex2(s[b][j][2 * e] - M[e]), p1 = ex2(s[b][j][2 * e + 1] - M[e]);
                        l[e] += p0 + p1;
                        float w0 = p0 * f[e], w1 = p1 * f[e];
                        if (!whole) {  // a NaN scale must not reach the rows that do not see the slot
                            if (s[b][j][2 * e] == -INFINITY) w0 = 0.0f;
                            if (s[b][j][2 * e + 1] == -INFINITY) w1 = 0.0f;
                        }
                        ph_[e + 2 * j] = pack_f16(w0, w1);
                        if (F32) pl_[e + 2 * j] = rest_f16(ph_[e + 2 * j], w0, w1);
                    }
                uint2 u[D / 64][2][2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int t = b * 16 + slot_of(c4, e, j);
                        const unsigned char* p = sv + t * D + 8 * gq;
                        const bool dead = !whole && t0 + t >= cur.s.len;  // not written yet: any bits
                        if (D == 64) {
                            u[0][j][e] = dead ? make_uint2(0, 0) : *reinterpret_cast<const uint2*>(p);
                        } else {
                            const bool odd = lane & 1;  // odd lanes read their halves in the other order
                            const uint2 x = *reinterpret_cast<const uint2*>(p + (odd ? 64 : 0));
                            const uint2 y = *reinterpret_cast<const uint2*>(p + (odd ? 0 : 64));
                            u[0][j][e] = dead ? make_uint2(0, 0) : odd ? y : x;
                            u[D / 64 - 1][j][e] = dead ? make_uint2(0, 0) : odd ? x : y;
                        }
                    }
#pragma unroll
                for (int hf = 0; hf < D / 64; ++hf)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        uint32_t f16[2][4];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t x = w ? u[hf][j][0].y : u[hf][j][0].x, y = w ? u[hf][j][1].y : u[hf][j][1].x;
                            widen<FMT>(__byte_perm(x, y, 0x5140), f16[j][0], f16[j][1]);
                            widen<FMT>(__byte_perm(x, y, 0x7362), f16[j][2], f16[j][3]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_f16(o[hf * 8 + w * 4 + i], ph_, f16[0][i], f16[1][i]);
                            if (F32) mma_f16(o[hf * 8 + w * 4 + i], pl_, f16[0][i], f16[1][i]);
                        }
                    }
            }
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
                for (int e = 0; e < 2; ++e) {
                    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
                    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
                    const int r = rows0 + gq + 8 * e;
                    if (r >= cur.s.n * a.group) continue;
                    if (last && from0) {
                        store_row<D, F32>(a, cur.s, cur.h, r, lane, o, e, M[e], R[e], l[e], vo);
                    } else {
                        float* p = a.part + (((int64_t)group * 2 + (from0 ? 1 : 0)) * tile_rows + wrow * 16 + gq + 8 * e) *
                                                part_floats(D);
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

// ---- merging the shares -----------------------------------------------------------------------------------------------
// One warp per query row and head whose unit was cut between shares, in the order of the shares.
template <int D, int RW, bool F32>
__global__ void __launch_bounds__(kThreads) kv8_merge_kernel(const __grid_constant__ Kv8AttendArgs a) {
    constexpr int TOK = kChunkBytes / D, V = D / 32;
    pdl_wait();
    pdl_launch();
    const int lane = threadIdx.x & 31, b = blockIdx.y, H = a.kv.kv_heads, tile_rows = 16 * RW;
    const Seq s = seq_of<TOK>(a, b, tile_rows);
    const int64_t total = a.offset[a.kv.n_seqs], base = a.offset[b];
    const int groups = a.groups;
    // the share that holds list item x
    auto holder = [&](int64_t x) { return (int)(((x + 1) * groups - 1) / total); };
    for (int64_t u = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); u < (int64_t)s.n * a.heads;
         u += (int64_t)gridDim.x * kWarps) {
        const int i = (int)(u / a.heads), hq = (int)(u % a.heads), h = hq / a.group, r = i * a.group + hq % a.group;
        const int64_t first = base + ((int64_t)h * s.tiles + r / tile_rows) * s.chunks;
        const int g0 = holder(first), g1 = holder(first + s.chunks - 1);
        if (g0 == g1) continue;
        const int64_t row = (int64_t)(r % tile_rows) * part_floats(D);
        const int64_t step = (int64_t)tile_rows * part_floats(D);
        // the unit's first share holds it in its slot 1, the later ones in their slot 0
        auto part = [&](int g) { return a.part + ((int64_t)g * 2 + (g == g0)) * step + row; };
        float M = kFar, R = kFar, l = 0.0f, o[V] = {};
        for (int g = g0; g <= g1; ++g) {
            if (share(total, g, groups) == share(total, g + 1, groups)) continue;  // an empty share
            const float4 m = *reinterpret_cast<const float4*>(part(g) + D);
            M = fmaxf(M, m.x);
            R = fmaxf(R, m.y);
        }
        for (int g = g0; g <= g1; ++g) {
            if (share(total, g, groups) == share(total, g + 1, groups)) continue;
            const float* p = part(g);
            const float4 m = *reinterpret_cast<const float4*>(p + D);
            l += m.z * pow2i(m.x - M);
            const float f = pow2i(m.y - R);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] += p[lane * V + e] * f;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l, up = pow2i(R - 14.0f - M);
        const int64_t at = (int64_t)(s.first + i) * a.out.row_stride + (int64_t)hq * a.out.head_stride + lane * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float v = l == 0.0f ? 0.0f : o[e] * inv * up;
            if (F32)
                static_cast<float*>(a.out.ptr)[at + e] = v;
            else
                static_cast<uint16_t*>(a.out.ptr)[at + e] = f32_to_bf16_rne(v);
        }
        if (a.lse && lane == 0) a.lse[(int64_t)(s.first + i) * a.heads + hq] = l == 0.0f ? INFINITY : M + log2f(l);
    }
}

// ---- accumulated weights ------------------------------------------------------------------------------------------------
// The weights each slot received, rebuilt from the scores and the finished softmax sums: CTAs take equal consecutive
// shares of the (sequence, KV head, chunk) list; a warp holds a chunk's K in registers as f16 and runs the query tiles
// past it from shared memory.
constexpr int kMassTiles = kWarps;  // query tiles in shared memory at a time, one loaded by each warp

template <int D, bool F32>
constexpr size_t mass_smem() {
    return (size_t)kMassTiles * (D / 16) * 32 * 16 * (F32 ? 2 : 1) + kMassTiles * 16 * 3 * 4 + kWarps * 64 * 4;
}

template <int FMT, int D, bool F32>
__global__ void __launch_bounds__(kThreads) kv8_mass_kernel(const __grid_constant__ Kv8AttendArgs a) {
    constexpr int TOK = kChunkBytes / D, NB = TOK / kKv8Block, CPP = kKv8Page / TOK, KS = D / 16;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    pdl_wait();
    pdl_launch();
    uint4* qs = reinterpret_cast<uint4*>(smem_raw);  // [tile][ks][lane], hi then lo
    float* rfac = reinterpret_cast<float*>(qs + (size_t)kMassTiles * KS * 32 * (F32 ? 2 : 1));
    float* rlse = rfac + kMassTiles * 16;
    int* rvis = reinterpret_cast<int*>(rlse + kMassTiles * 16);
    float* sums = reinterpret_cast<float*>(rvis + kMassTiles * 16) + (threadIdx.x >> 5) * 64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, c4 = lane & 3, H = a.kv.kv_heads;
    const bool vq = vec_rows(a.q);
    auto chunks_of = [&](int b) {
        const Seq s = seq_of<TOK>(a, b, 16);
        return (s.len + TOK - 1) / TOK;
    };
    int64_t total = 0;
    for (int b = lane; b < a.kv.n_seqs; b += 32) total += (int64_t)H * chunks_of(b);
    total = warp_sum64(total);
    int64_t pos = share(total, blockIdx.x, gridDim.x);
    const int64_t end = share(total, blockIdx.x + 1, gridDim.x);
    if (pos >= end) return;
    int64_t base = 0;  // of sequence b in the list
    int b = seek(a.kv.n_seqs, pos, false, base, [&](int i) { return (int64_t)H * chunks_of(i); }, [](int, int64_t) {});
    while (pos < end) {
        const Seq s = seq_of<TOK>(a, b, 16);
        const int chunks = (s.len + TOK - 1) / TOK;
        if (pos >= base + (int64_t)H * chunks) {
            base += (int64_t)H * chunks;
            ++b;
            continue;
        }
        const int h = (int)((pos - base) / chunks), c0 = (int)((pos - base) % chunks);
        const int c1 = (int)min((int64_t)chunks, c0 + (end - pos));
        const int rows = s.n * a.group, tiles = (rows + 15) / 16;
        for (int tb = 0; tb < max(1, tiles); tb += kMassTiles) {
            const int nt = min(kMassTiles, tiles - tb);
            __syncthreads();  // the tiles before these are done with
            if (warp < nt) {
                const int row0 = (tb + warp) * 16;
                QFrag<D, F32> q;
                q.load(a, s, h, row0, vq, lane);
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    qs[(warp * KS + k) * 32 + lane] = make_uint4(q.hi[k][0], q.hi[k][1], q.hi[k][2], q.hi[k][3]);
                    if (F32)
                        qs[((kMassTiles + warp) * KS + k) * 32 + lane] =
                            make_uint4(q.lo[F32 ? k : 0][0], q.lo[F32 ? k : 0][1], q.lo[F32 ? k : 0][2], q.lo[F32 ? k : 0][3]);
                }
                if (c4 == 0)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
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
                        const float f0 = rfac[t * 16 + gq], f1 = rfac[t * 16 + gq + 8];
                        const float e0 = rlse[t * 16 + gq], e1 = rlse[t * 16 + gq + 8];
                        const int v0 = rvis[t * 16 + gq], v1 = rvis[t * 16 + gq + 8];
                        const bool whole = c * TOK + TOK <= rvis[t * 16];
                        float acc[NB][2][4] = {};
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            const uint4 x = qs[(t * KS + k) * 32 + lane];
                            const uint32_t hi[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int n = 0; n < NB; ++n)
#pragma unroll
                                for (int j = 0; j < 2; ++j) mma_f16(acc[n][j], hi, kf[n][j][k][0], kf[n][j][k][1]);
                            if (F32) {
                                const uint4 y = qs[((kMassTiles + t) * KS + k) * 32 + lane];
                                const uint32_t lo[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                                for (int n = 0; n < NB; ++n)
#pragma unroll
                                    for (int j = 0; j < 2; ++j) mma_f16(acc[n][j], lo, kf[n][j][k][0], kf[n][j][k][1]);
                            }
                        }
#pragma unroll
                        for (int n = 0; n < NB; ++n)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    float p0 = ex2(acc[n][j][e] * (f0 * ks[n]) - e0), p1 = ex2(acc[n][j][2 + e] * (f1 * ks[n]) - e1);
                                    if (!whole) {
                                        const int at = c * TOK + n * 16 + slot_of(c4, e, j);
                                        if (at >= v0) p0 = 0.0f;
                                        if (at >= v1) p1 = 0.0f;
                                    }
                                    sum[n][j][e] += p0 + p1;
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
cudaError_t launch(K kernel, dim3 grid, size_t smem, cudaStream_t s, const Kv8AttendArgs& a) {
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = kThreads;
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

    template <int FMT, int D, int RW, bool F32>
    cudaError_t go() {
        a.groups = sm_count() * Ring<D, RW>::GROUPS;
        cudaError_t e = launch(kv8_attend_kernel<FMT, D, RW, F32>, dim3(sm_count()), Ring<D, RW>::bytes, s, a);
        if (e != cudaSuccess) return e;
        const int64_t rows = (int64_t)a.max_new * a.heads;
        const dim3 grid((unsigned)min((int64_t)1024, (rows + kWarps - 1) / kWarps), a.kv.n_seqs);
        e = launch(kv8_merge_kernel<D, RW, F32>, grid, 0, s, a);
        if (e != cudaSuccess || !a.mass_out) return e;
        return launch(kv8_mass_kernel<FMT, D, F32>, dim3(2 * sm_count()), mass_smem<D, F32>(), s, a);
    }
    template <int FMT, int D, int RW>
    cudaError_t by_type() {
        return a.q.dtype == LASTRO_DTYPE_F32 ? go<FMT, D, RW, true>() : go<FMT, D, RW, false>();
    }
    template <int FMT, int D>
    cudaError_t run() {
        switch (row_warps((int64_t)a.max_new * a.group)) {
        case 1: return by_type<FMT, D, 1>();
        case 2: return by_type<FMT, D, 2>();
        case 4: return by_type<FMT, D, 4>();
        default: return by_type<FMT, D, 8>();
        }
    }
};

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

size_t kv8_attend_workspace(const lastro_kv8& kv, int heads, int max_new, bool with_mass, Kv8AttendArgs* a, void* base) {
    const int rw = row_warps((int64_t)max_new * (heads / kv.kv_heads));
    const size_t groups = (size_t)sm_count() * kWarps / rw;
    const size_t offset = align16(((size_t)kv.n_seqs + 1) * sizeof(int64_t));
    const size_t part = groups * 2 * rw * 16 * part_floats(kv.head_dim) * sizeof(float);
    const size_t lse = with_mass ? (size_t)kv.n_seqs * max_new * heads * sizeof(float) : 0;
    if (a) {
        unsigned char* p = static_cast<unsigned char*>(base);
        a->offset = reinterpret_cast<int64_t*>(p);
        a->part = reinterpret_cast<float*>(p + offset);
        a->lse = with_mass ? reinterpret_cast<float*>(p + offset + part) : nullptr;
    }
    return offset + part + lse;
}

cudaError_t launch_kv8_attend(const Kv8AttendArgs& a, cudaStream_t s) { return kv8_by_shape(a.kv, AttendLaunch{a, s}); }

}  // namespace lastro
