// Device helpers of the 8-bit KV cache kernels: checks on device data, codes and scales, activation rows.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "kv8.h"

namespace lastro {

constexpr int E4M3 = LASTRO_KV8_E4M3, INT8 = LASTRO_KV8_INT8;

// ---- checks on device data ------------------------------------------------------------------------------------------
LDEV void report(const lastro_kv8& kv, int code) {
    if (kv.status) atomicExch(kv.status, code);
}

// the page of slot `slot` of sequence b, or -1
LDEV int page_of(const lastro_kv8& kv, int b, int slot) {
    const int p = __ldg(kv.page_table + (int64_t)b * kv.max_pages + slot / kKv8Page);
    if ((unsigned)p < (unsigned)kv.num_pages) return p;
    report(kv, LASTRO_KV8_BAD_PAGE);
    return -1;
}

// a sequence's length, 0 when it is not one the page table (or `most` slots) can hold
LDEV int seq_len(const lastro_kv8& kv, const int32_t* lens, int b, int64_t most) {
    const int n = __ldg(lens + b);
    if (n >= 0 && n <= most) return n;
    report(kv, LASTRO_KV8_BAD_LENGTH);
    return 0;
}

// rows of sequence b: first row, and their number (0 when the offsets are not usable)
LDEV int seq_rows(const lastro_kv8& kv, const int32_t* off, int b, int rows, int max_new, int& first) {
    first = __ldg(off + b);
    const int end = __ldg(off + b + 1);
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

template <int FMT>
LDEV uint32_t encode4(float a, float b, float c, float d) {
    if (FMT == E4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    }
    return (uint32_t)(__float2int_rn(a) & 0xff) | (uint32_t)(__float2int_rn(b) & 0xff) << 8 |
           (uint32_t)(__float2int_rn(c) & 0xff) << 16 | (uint32_t)(__float2int_rn(d) & 0xff) << 24;
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

// 8 consecutive values of an activation row; `vec`: every such group is 16-byte aligned
template <bool F32>
LDEV void load8(const lastro_rows& r, int64_t at, bool vec, float (&v)[8]) {
    if (F32) {
        const float* p = static_cast<const float*>(r.ptr) + at;
        if (vec) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __ldg(p + i);
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(r.ptr) + at;
        if (vec) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
            v[0] = bf_lo(a.x), v[1] = bf_hi(a.x), v[2] = bf_lo(a.y), v[3] = bf_hi(a.y);
            v[4] = bf_lo(a.z), v[5] = bf_hi(a.z), v[6] = bf_lo(a.w), v[7] = bf_hi(a.w);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float((uint32_t)__ldg(p + i) << 16);
        }
    }
}

LDEV bool vec_rows(const lastro_rows& r) {
    const int64_t e = r.dtype == LASTRO_DTYPE_F32 ? 4 : 2;
    return ((reinterpret_cast<uintptr_t>(r.ptr) | (uintptr_t)(r.row_stride * e) | (uintptr_t)(r.head_stride * e)) & 15) == 0;
}

LDEV uint32_t warp_umax(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

template <typename F>
cudaError_t kv8_by_shape(const lastro_kv8& kv, F f) {
    if (kv.format == E4M3) return kv.head_dim == 64 ? f.template run<E4M3, 64>() : f.template run<E4M3, 128>();
    return kv.head_dim == 64 ? f.template run<INT8, 64>() : f.template run<INT8, 128>();
}

}  // namespace lastro
