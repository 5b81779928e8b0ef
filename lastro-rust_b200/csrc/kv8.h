// 8-bit KV cache: kernel arguments and launchers (kernels in kv8.cu, C ABI in kv8_capi.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/lastro_b200.h"

namespace lastro {

constexpr int kKv8Page = LASTRO_KV8_PAGE, kKv8Block = LASTRO_KV8_BLOCK;
constexpr int kKv8Blocks = kKv8Page / kKv8Block;  // blocks (scales) of one page and head

struct Kv8AppendArgs {
    lastro_kv8 kv;
    const int32_t *lens, *new_off;
    lastro_rows k, v;
    int32_t max_new, blocks;  // blocks: most blocks one sequence's new rows touch
    int32_t* lens_out;
    float* mass;
    int64_t mass_stride;
};

struct Kv8AttendArgs {
    lastro_kv8 kv;
    const int32_t *lens, *q_off;
    lastro_rows q, out;
    int32_t max_new, heads, group;
    float scale;
    const float* mass_in;
    float* mass_out;
    int64_t mass_stride;
    // workspace (kv8_attend_workspace)
    int32_t* offset;       // [n_seqs + 1]: where each sequence's work starts in the list, the list's length
    float* part;           // partial results of units cut between shares of the list
    // [rows, heads]: each softmax's maximum (in powers of two) and 1 / sum, which the weights are rebuilt from; NULL without
    // them.  Not the logarithm of both, which far from zero would round the sum away.
    float2* norm;
    float* scores;         // [list items][score_rows][chunk's slots]: the scores, where they are kept
    int32_t shares, score_rows;
};

// bytes of workspace; with `a`, its pointers into the workspace at `base`
size_t kv8_attend_workspace(const lastro_kv8& kv, int heads, int max_new, bool with_mass, Kv8AttendArgs* a, void* base);
// the longest list of work a call can have
int64_t kv8_attend_items(const lastro_kv8& kv, int heads, int max_new);


struct Kv8EvictArgs {
    lastro_kv8 src, dst;
    const int32_t* lens;
    int32_t budget, recent;
    const float* mass;
    int64_t mass_stride;
    int32_t *kept, *lens_out;
    float* mass_out;
    int64_t mass_out_stride;
};

struct Kv8ReadArgs {
    lastro_kv8 kv;
    const int32_t *lens, *pos0;
    int32_t n;
    void *k_out, *v_out;
    int32_t f32;
};

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t s);
cudaError_t launch_kv8_attend(const Kv8AttendArgs& a, cudaStream_t s);
cudaError_t launch_kv8_evict(const Kv8EvictArgs& a, cudaStream_t s);
cudaError_t launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t s);

}  // namespace lastro
