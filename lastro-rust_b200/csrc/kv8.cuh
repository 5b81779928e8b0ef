// Device helpers of the 8-bit KV cache kernels: checks on device data, codes and scales, activation rows.
#pragma once

#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"
#include "kv8.h"

namespace lastro {

constexpr int E4M3 = LASTRO_KV8_E4M3, INT8 = LASTRO_KV8_INT8;

// ---- checks on device data ------------------------------------------------------------------------------------------
// Lengths, tables, rows, codes, scales and masses are what earlier calls on the stream, or the program between them, left
// behind, and these kernels are resident before that has ended: they are read with ordinary loads, which stay behind
// pdl_wait() and see what it waited for.  (The read-only path promises neither.)
LDEV void report(const lastro_kv8& kv, int code) {
    if (kv.status) atomicExch(kv.status, code);
}

// the page of slot `slot` of sequence b, or -1
LDEV int page_of(const lastro_kv8& kv, int b, int slot) {
    const int p = kv.page_table[(int64_t)b * kv.max_pages + slot / kKv8Page];
    if ((unsigned)p < (unsigned)kv.num_pages) return p;
    report(kv, LASTRO_KV8_BAD_PAGE);
    return -1;
}

// a sequence's length, 0 when it is not one the page table (or `most` slots) can hold
LDEV int seq_len(const lastro_kv8& kv, const int32_t* lens, int b, int64_t most) {
    const int n = lens[b];
    if (n >= 0 && n <= most) return n;
    report(kv, LASTRO_KV8_BAD_LENGTH);
    return 0;
}

// rows of sequence b: first row, and their number (0 when the offsets are not usable)
LDEV int seq_rows(const lastro_kv8& kv, const int32_t* off, int b, int rows, int max_new, int& first) {
    first = off[b];
    const int end = off[b + 1];
    if (first >= 0 && end >= first && end <= rows && end - first <= max_new) return end - first;
    report(kv, LASTRO_KV8_BAD_OFFSET);
    return 0;
}

// ---- values, codes, scales ------------------------------------------------------------------------------------------
// The scale of a block whose largest magnitude has the bits `amax` (sign cleared; NaN and infinities order above every
// finite value): with amax = 1.f * 2^E it is 2^(E-8) or 2^(E-7) for e4m3 (448 = 1.75 * 2^8), 2^(E-6) or 2^(E-5) for int8
// (127 = 1.984375 * 2^6).
template <int FMT>
LDEV float scale_for(uint32_t amax) {
    if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    const uint32_t top = FMT == E4M3 ? 0x600000u : 0x7e0000u;
    const int e = (int)(amax >> 23) - (FMT == E4M3 ? 8 : 6) + ((amax & 0x7fffffu) > top);
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// 1 / s of a power of two s = 2^e, -126 <= e <= 122: exact
LDEV float inverse(float s) { return __uint_as_float((254u << 23) - (__float_as_uint(s) & 0x7f800000u)); }

// the codes of four values times a power of two
template <int FMT>
LDEV uint32_t encode4(float a, float b, float c, float d, float inv) {
    if (FMT == E4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inv, d * inv), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    }
    // 1.5 * 2^23 + x rounds x to a whole number, whose low byte is the sum's (the product is exact)
    const float big = 12582912.0f;
    const uint32_t p = __float_as_uint(fmaf(a, inv, big)), q = __float_as_uint(fmaf(b, inv, big));
    const uint32_t r = __float_as_uint(fmaf(c, inv, big)), t = __float_as_uint(fmaf(d, inv, big));
    return __byte_perm(__byte_perm(p, q, 0x40), __byte_perm(r, t, 0x40), 0x5410);
}

template <int FMT>
LDEV void decode4(uint32_t w, float (&v)[4]) {
    if (FMT == E4M3) {
        const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffff), __NV_E4M3)));
        const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
        v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> (8 * i));
    }
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

// 8 consecutive values of an activation row as they are stored; `vec`: every such group is 16-byte aligned
template <bool F32>
struct Raw8 {
    uint32_t w[F32 ? 8 : 4];

    LDEV void load(const lastro_rows& r, int64_t at, bool vec) {
        const char* p = static_cast<const char*>(r.ptr) + at * (F32 ? 4 : 2);
        if (vec) {
#pragma unroll
            for (int i = 0; i < (F32 ? 2 : 1); ++i) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else if (F32) {
#pragma unroll
            for (int i = 0; i < (F32 ? 8 : 4); ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        } else {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
        }
    }
    LDEV void zero() {
#pragma unroll
        for (int i = 0; i < (F32 ? 8 : 4); ++i) w[i] = 0;
    }
    // magnitudes' bits so far: f32 bits, or two bf16 side by side
    LDEV void widest(uint32_t& m) const {
#pragma unroll
        for (int i = 0; i < (F32 ? 8 : 4); ++i) m = F32 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
    }
    LDEV static uint32_t f32_bits(uint32_t m) { return F32 ? m : max(m << 16, m & 0xffff0000u); }
    LDEV void values(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = F32 ? __uint_as_float(w[F32 ? i : 0]) : i & 1 ? bf_hi(w[F32 ? 0 : i / 2]) : bf_lo(w[F32 ? 0 : i / 2]);
    }
};

LDEV uint32_t two_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

LDEV bool vec_rows(const lastro_rows& r) {
    const int64_t e = r.dtype == LASTRO_DTYPE_F32 ? 4 : 2;
    return ((reinterpret_cast<uintptr_t>(r.ptr) | (uintptr_t)(r.row_stride * e) | (uintptr_t)(r.head_stride * e)) & 15) == 0;
}

// row r of a KV head's query rows: which query, for `group` heads a query (single-token calls need no division)
LDEV int query_of(int r, int group) { return r < group ? 0 : r / group; }

LDEV uint32_t warp_umax(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// programmatic launch: the kernel's CTAs are placed while the stream's previous kernel drains and wait for its end before
// they touch memory.  A kernel's shared memory limit is raised once on each device, to the most any launch of it takes, so
// that threads which launch it at the same time set the same.
template <auto KERNEL, size_t MOST, typename A>
cudaError_t kv8_launch(dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s, const A& a) {
    static_assert(MOST <= 227 * 1024, "beyond what a CTA can have");
    if (MOST > 48 * 1024) {
        static std::atomic<bool> raised[64];
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev >= 64 || !raised[dev].load(std::memory_order_acquire)) {
            e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MOST);
            if (e != cudaSuccess) return e;
            if (dev < 64) raised[dev].store(true, std::memory_order_release);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, KERNEL, a);
}

template <typename F>
cudaError_t kv8_by_shape(const lastro_kv8& kv, F f) {
    if (kv.format == E4M3) return kv.head_dim == 64 ? f.template run<E4M3, 64>() : f.template run<E4M3, 128>();
    return kv.head_dim == 64 ? f.template run<INT8, 64>() : f.template run<INT8, 128>();
}

}  // namespace lastro
