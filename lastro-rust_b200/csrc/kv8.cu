// 8-bit KV cache: append (quantise), eviction, read-back (attention in kv8_attend.cu).  Layout and rules in
// include/lastro_b200.h.
#include <cuda_runtime.h>

#include "kv8.cuh"

namespace lastro {
namespace {

// ---- append ---------------------------------------------------------------------------------------------------------
// One warp quantises one block (16 slots) of K or V of one head: its new rows pass through registers once (a lane holds
// groups of 8 values), the largest magnitude by a warp reduction, then the codes.  The block's earlier rows are read and
// rounded again only where the scale grows.
template <int FMT, int D>
__global__ void __launch_bounds__(256) kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a) {
    constexpr int LPR = D / 8, RPW = 32 / LPR, N = kKv8Block / RPW;  // lanes a row, rows a pass, passes
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, H = a.kv.kv_heads;
    const int which = (int)(unit & 1), h = (int)((unit >> 1) % H);
    const int64_t bj = (unit >> 1) / H;
    const int b = (int)(bj / a.blocks), j = (int)(bj % a.blocks);
    if (b >= a.kv.n_seqs) return;
    int64_t most = (int64_t)a.kv.max_pages * kKv8Page;
    if (a.mass) most = min(most, a.mass_stride);
    const int len = seq_len(a.kv, a.lens, b, most);
    int first, n = seq_rows(a.kv, a.new_off, b, min(a.k.rows, a.v.rows), a.max_new, first);
    if (n > most - len || __ldg(a.lens + b) != len) {
        if (n > most - len) report(a.kv, LASTRO_KV8_BAD_LENGTH);
        n = 0;
    }
    if (which == 0 && j == 0) {
        if (h == 0 && lane == 0) a.lens_out[b] = len + n;
        if (a.mass)
            for (int i = lane; i < n; i += 32) a.mass[((int64_t)b * H + h) * a.mass_stride + len + i] = 0.0f;
    }
    const int slot0 = (len / kKv8Block + j) * kKv8Block;  // the block's first slot
    if (n == 0 || slot0 >= len + n) return;
    const int page = page_of(a.kv, b, slot0);
    if (page < 0) return;
    const int beg = max(0, len - slot0), end = min(kKv8Block, len + n - slot0);  // its new rows
    const int64_t tile = (int64_t)page * H + h;
    uint8_t* codes = static_cast<uint8_t*>(which ? a.kv.v : a.kv.k) + (tile * kKv8Page + slot0 % kKv8Page) * D;
    float* scale = (which ? a.kv.v_scale : a.kv.k_scale) + tile * kKv8Blocks + slot0 % kKv8Page / kKv8Block;
    const lastro_rows& src = which ? a.v : a.k;
    const bool vec = vec_rows(src);
    const int r0 = lane / LPR, c = lane % LPR * 8;

    float x[N][8];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + i * RPW;
        if (r >= beg && r < end) {
            const int64_t at = (int64_t)(first + slot0 + r - len) * src.row_stride + h * src.head_stride + c;
            if (src.dtype == LASTRO_DTYPE_F32)
                load8<true>(src, at, vec, x[i]);
            else
                load8<false>(src, at, vec, x[i]);
        } else
#pragma unroll
            for (int q = 0; q < 8; ++q) x[i][q] = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) amax = max(amax, __float_as_uint(x[i][q]) & 0x7fffffffu);
    }
    float s = scale_for<FMT>(warp_umax(amax));
    const float was = beg ? *scale : s;
    if (was != was || (s == s && was > s)) s = was;  // earlier rows: the larger scale, NaN stays
    const bool nan = s != s;
    const float inv = nan ? 0.0f : inverse(s);
    __syncwarp();  // every lane has read the old scale
    if (lane == 0) *scale = s;
    const bool again = beg && (nan || was != s);
    const float ratio = nan ? 0.0f : was * inv;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + i * RPW;
        uint2* dst = reinterpret_cast<uint2*>(codes + r * D + c);
        if (r >= beg && r < end) {
            if (nan)
#pragma unroll
                for (int q = 0; q < 8; ++q) x[i][q] = 0.0f;
            uint2 o;
            o.x = encode4<FMT>(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv);
            o.y = encode4<FMT>(x[i][4] * inv, x[i][5] * inv, x[i][6] * inv, x[i][7] * inv);
            *dst = o;
        } else if (again && r < beg) {
            const uint2 w = *dst;
            float u[4], t[4];
            decode4<FMT>(w.x, u);
            decode4<FMT>(w.y, t);
            *dst = make_uint2(encode4<FMT>(u[0] * ratio, u[1] * ratio, u[2] * ratio, u[3] * ratio),
                              encode4<FMT>(t[0] * ratio, t[1] * ratio, t[2] * ratio, t[3] * ratio));
        }
    }
}

// ---- read-back ------------------------------------------------------------------------------------------------------
template <int FMT, bool F32>
__global__ void __launch_bounds__(256) kv8_read_kernel(const __grid_constant__ Kv8ReadArgs a) {
    const int H = a.kv.kv_heads, D = a.kv.head_dim, G = D / 8;
    const int64_t total = (int64_t)a.kv.n_seqs * a.n * H * G;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int c = (int)(i % G) * 8, h = (int)(i / G % H);
        const int64_t bj = i / G / H;
        const int b = (int)(bj / a.n), j = (int)(bj % a.n);
        const int len = seq_len(a.kv, a.lens, b, (int64_t)a.kv.max_pages * kKv8Page);
        const int64_t slot = (int64_t)__ldg(a.pos0 + b) + j;
        const int page = slot >= 0 && slot < len ? page_of(a.kv, b, (int)slot) : -1;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            void* out = which ? a.v_out : a.k_out;
            if (!out) continue;
            float v[8] = {};
            if (page >= 0) {
                const int64_t tile = (int64_t)page * H + h;
                const uint8_t* codes = static_cast<const uint8_t*>(which ? a.kv.v : a.kv.k);
                const uint2 w = __ldg(reinterpret_cast<const uint2*>(codes + (tile * kKv8Page + slot % kKv8Page) * D + c));
                const float s = __ldg((which ? a.kv.v_scale : a.kv.k_scale) + tile * kKv8Blocks + slot % kKv8Page / kKv8Block);
                float lo[4], hi[4];
                decode4<FMT>(w.x, lo);
                decode4<FMT>(w.y, hi);
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = lo[q] * s, v[4 + q] = hi[q] * s;
            }
            if (F32) {
                float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + i * 8);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                uint4 o;
                o.x = pack_bf16(f32_to_bf16_rne(v[0]), f32_to_bf16_rne(v[1]));
                o.y = pack_bf16(f32_to_bf16_rne(v[2]), f32_to_bf16_rne(v[3]));
                o.z = pack_bf16(f32_to_bf16_rne(v[4]), f32_to_bf16_rne(v[5]));
                o.w = pack_bf16(f32_to_bf16_rne(v[6]), f32_to_bf16_rne(v[7]));
                reinterpret_cast<uint4*>(out)[i] = o;
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

constexpr int kSelThreads = 1024;

// exclusive prefix sum of v over the block and the total; `red` holds 33 ints
LDEV int block_scan(int v, int* red, int& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 31) red[w] = s;
    __syncthreads();
    if (w == 0) {
        int x = red[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += t;
        }
        red[lane] = x;
    }
    __syncthreads();
    total = red[31];
    return s - v + (w ? red[w - 1] : 0);
}

// One CTA per sequence and KV head: the key of the (budget - recent)-th largest mass by four 8-bit radix passes, then one
// pass that writes the kept slots in order (all above the key, and of those at it the lowest slots).
__global__ void __launch_bounds__(kSelThreads) kv8_select_kernel(const __grid_constant__ Kv8EvictArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ int red[33];
    __shared__ uint32_t s_key;
    __shared__ int s_need;
    const int H = a.src.kv_heads, h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, C = a.budget;
    int64_t most = (int64_t)a.src.max_pages * kKv8Page;
    if (a.mass) most = min(most, a.mass_stride);
    const int len = seq_len(a.src, a.lens, b, most);
    const int64_t seq = (int64_t)b * H + h;
    int32_t* kept = a.kept + seq * C;
    const float* mass = a.mass ? a.mass + seq * a.mass_stride : nullptr;
    float* mout = a.mass_out ? a.mass_out + seq * a.mass_out_stride : nullptr;
    const int keep = min(len, C);
    if (h == 0 && tid == 0) a.lens_out[b] = keep;
    for (int i = keep + tid; i < C; i += kSelThreads) kept[i] = -1;
    if (len <= C) {
        for (int i = tid; i < len; i += kSelThreads) {
            kept[i] = i;
            if (mout) mout[i] = mass ? mass[i] : 0.0f;
        }
        return;
    }
    const int cand = len - a.recent, want = C - a.recent;  // cand > want
    if (want > 0) {
        uint32_t prefix = 0;
        int need = want;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
            for (int t = tid; t < cand; t += kSelThreads) {
                const uint32_t k = mass_key(mass[t]);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                int left = need, d = 255;
                for (; d > 0 && (int)hist[d] < left; --d) left -= hist[d];
                s_key = prefix | (uint32_t)d << shift;
                s_need = left;
            }
            __syncthreads();
            prefix = s_key;
            need = s_need;
        }
        // `need` of the slots whose key equals prefix are kept
        int ties = 0, out = 0;
        for (int base = 0; base < cand; base += kSelThreads) {
            const int t = base + tid;
            const float m = t < cand ? mass[t] : 0.0f;
            const uint32_t k = mass_key(m);
            const bool tie = t < cand && k == prefix;
            int nt, ns;
            const int rank = ties + block_scan(tie, red, nt);
            const bool sel = t < cand && (k > prefix || (tie && rank < need));
            const int at = out + block_scan(sel, red, ns);
            if (sel) {
                kept[at] = t;
                if (mout) mout[at] = m;
            }
            ties += nt;
            out += ns;
        }
    }
    for (int i = tid; i < a.recent; i += kSelThreads) {
        kept[want + i] = cand + i;
        if (mout) mout[want + i] = mass ? mass[cand + i] : 0.0f;
    }
}

// One warp gathers one destination block of K or V: 16 kept rows, their largest magnitude, the new scale and codes.
template <int FMT, int D>
__global__ void __launch_bounds__(256) kv8_gather_kernel(const __grid_constant__ Kv8EvictArgs a) {
    constexpr int LPR = D / 8, RPW = 32 / LPR, N = kKv8Block / RPW;
    const int lane = threadIdx.x & 31, H = a.src.kv_heads, blocks = (a.budget + kKv8Block - 1) / kKv8Block;
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int which = (int)(unit & 1), j = (int)((unit >> 1) % blocks);
    const int64_t seq = (unit >> 1) / blocks;
    const int b = (int)(seq / H), h = (int)(seq % H);
    if (b >= a.src.n_seqs) return;
    const int keep = a.lens_out[b], slot0 = j * kKv8Block;
    if (slot0 >= keep) return;
    if (keep > (int64_t)a.dst.max_pages * kKv8Page) {
        report(a.dst, LASTRO_KV8_BAD_LENGTH);
        return;
    }
    const int dpage = page_of(a.dst, b, slot0);
    if (dpage < 0) return;
    const int r0 = lane / LPR, c = lane % LPR * 8;
    const uint8_t* src = static_cast<const uint8_t*>(which ? a.src.v : a.src.k);
    const float* sscale = which ? a.src.v_scale : a.src.k_scale;
    uint2 w[N];
    float sc[N];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = slot0 + r0 + i * RPW;
        w[i] = make_uint2(0, 0);
        sc[i] = 0.0f;
        if (r < keep) {
            const int t = a.kept[seq * a.budget + r];
            const int page = page_of(a.src, b, t);
            if (page >= 0) {
                const int64_t tile = (int64_t)page * H + h;
                w[i] = __ldg(reinterpret_cast<const uint2*>(src + (tile * kKv8Page + t % kKv8Page) * D + c));
                sc[i] = __ldg(sscale + tile * kKv8Blocks + t % kKv8Page / kKv8Block);
            }
        }
        float u[4], v[4];
        decode4<FMT>(w[i].x, u);
        decode4<FMT>(w[i].y, v);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            amax = max(amax, __float_as_uint(u[q] * sc[i]) & 0x7fffffffu);
            amax = max(amax, __float_as_uint(v[q] * sc[i]) & 0x7fffffffu);
        }
    }
    const float s = scale_for<FMT>(warp_umax(amax));
    const bool nan = s != s;
    const float inv = nan ? 0.0f : inverse(s);
    const int64_t tile = (int64_t)dpage * H + h;
    uint8_t* dst = static_cast<uint8_t*>(which ? a.dst.v : a.dst.k) + (tile * kKv8Page + slot0 % kKv8Page) * D;
    if (lane == 0) (which ? a.dst.v_scale : a.dst.k_scale)[tile * kKv8Blocks + slot0 % kKv8Page / kKv8Block] = s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = r0 + i * RPW;
        if (slot0 + r >= keep) continue;
        float u[4], v[4];
        decode4<FMT>(w[i].x, u);
        decode4<FMT>(w[i].y, v);
        const float f = nan ? 0.0f : sc[i] * inv;  // a ratio of powers of two
        *reinterpret_cast<uint2*>(dst + r * D + c) = make_uint2(encode4<FMT>(u[0] * f, u[1] * f, u[2] * f, u[3] * f),
                                                                encode4<FMT>(v[0] * f, v[1] * f, v[2] * f, v[3] * f));
    }
}

// ---- variants -------------------------------------------------------------------------------------------------------
unsigned int blocks_of(int64_t units, int per) { return (unsigned int)((units + per - 1) / per); }

struct AppendLaunch {
    const Kv8AppendArgs& a;
    cudaStream_t s;
    template <int FMT, int D>
    cudaError_t run() {
        const int64_t units = (int64_t)a.kv.n_seqs * a.blocks * a.kv.kv_heads * 2;
        kv8_append_kernel<FMT, D><<<blocks_of(units, 8), 256, 0, s>>>(a);
        return cudaGetLastError();
    }
};

struct EvictLaunch {
    const Kv8EvictArgs& a;
    cudaStream_t s;
    template <int FMT, int D>
    cudaError_t run() {
        kv8_select_kernel<<<dim3(a.src.kv_heads, a.src.n_seqs), kSelThreads, 0, s>>>(a);
        const int64_t units = (int64_t)a.src.n_seqs * a.src.kv_heads * ((a.budget + kKv8Block - 1) / kKv8Block) * 2;
        if (units) kv8_gather_kernel<FMT, D><<<blocks_of(units, 8), 256, 0, s>>>(a);
        return cudaGetLastError();
    }
};

}  // namespace

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t s) { return kv8_by_shape(a.kv, AppendLaunch{a, s}); }
cudaError_t launch_kv8_evict(const Kv8EvictArgs& a, cudaStream_t s) { return kv8_by_shape(a.src, EvictLaunch{a, s}); }

cudaError_t launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t s) {
    const int64_t total = (int64_t)a.kv.n_seqs * a.n * a.kv.kv_heads * (a.kv.head_dim / 8);
    const unsigned int grid = (unsigned int)min((int64_t)148 * 16, (total + 255) / 256);
    if (a.kv.format == E4M3)
        (a.f32 ? kv8_read_kernel<E4M3, true> : kv8_read_kernel<E4M3, false>)<<<grid, 256, 0, s>>>(a);
    else
        (a.f32 ? kv8_read_kernel<INT8, true> : kv8_read_kernel<INT8, false>)<<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace lastro
