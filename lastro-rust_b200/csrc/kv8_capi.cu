// C ABI of the 8-bit KV cache: argument checks and launches (lastro_kv8_* in include/lastro_b200.h).
#include <algorithm>
#include <cmath>

#include "capi_internal.h"
#include "kv8.h"

using namespace lastro;
using namespace lastro_capi;

namespace {

bool misaligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

// the cache's description; 0 or the status to return
int check_kv(lastro_ctx* c, const lastro_kv8* kv, const char* what) {
    if (!kv) return set_err(c, LASTRO_E_ARG, "%s: null cache", what);
    if (kv->format != LASTRO_KV8_E4M3 && kv->format != LASTRO_KV8_INT8)
        return set_err(c, LASTRO_E_ARG, "%s: format %d", what, kv->format);
    if (kv->n_seqs < 1 || kv->kv_heads < 1 || kv->num_pages < 1 || kv->max_pages < 1)
        return set_err(c, LASTRO_E_ARG, "%s: n_seqs %d, kv_heads %d, num_pages %d, max_pages %d must be positive", what,
                       kv->n_seqs, kv->kv_heads, kv->num_pages, kv->max_pages);
    if (kv->head_dim != 64 && kv->head_dim != 128)
        return set_err(c, LASTRO_E_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, kv->head_dim);
    if (kv->max_pages > (1 << 24) || kv->n_seqs > 65535 || kv->kv_heads > 1024)
        return set_err(c, LASTRO_E_UNSUPPORTED, "%s: max_pages %d, n_seqs %d or kv_heads %d beyond 2^24, 65535, 1024", what,
                       kv->max_pages, kv->n_seqs, kv->kv_heads);
    if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale || !kv->page_table)
        return set_err(c, LASTRO_E_ARG, "%s: null cache buffer", what);
    if (misaligned(kv->k, 16) || misaligned(kv->v, 16) || misaligned(kv->k_scale, 16) || misaligned(kv->v_scale, 16) ||
        misaligned(kv->page_table, 4) || misaligned(kv->status, 4))
        return set_err(c, LASTRO_E_ARG, "%s: codes and scales start on 16-byte boundaries, tables on 4-byte ones", what);
    return LASTRO_OK;
}

int check_rows(lastro_ctx* c, const lastro_rows* r, const char* what) {
    if (!r || !r->ptr) return set_err(c, LASTRO_E_ARG, "%s: null rows", what);
    if (r->dtype != LASTRO_DTYPE_BF16 && r->dtype != LASTRO_DTYPE_F32)
        return set_err(c, LASTRO_E_ARG, "%s: dtype %d (bf16 or f32)", what, r->dtype);
    if (r->rows < 0) return set_err(c, LASTRO_E_ARG, "%s: %d rows", what, r->rows);
    if (misaligned(r->ptr, r->dtype == LASTRO_DTYPE_F32 ? 4 : 2)) return set_err(c, LASTRO_E_ARG, "%s: misaligned rows", what);
    return LASTRO_OK;
}

// launches that failed: the kernels of the call before the one that failed may be enqueued, so its outputs are not to be used;
// no object of this family holds state that it could leave half-done
int launched(lastro_ctx* c, cudaError_t e, const char* what) {
    if (e == cudaSuccess) return LASTRO_OK;
    cudaGetLastError();
    return set_err(c, LASTRO_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int on_device(lastro_ctx* c, const char* what) { return launched(c, cudaSetDevice(c->device), what); }

#define KV8_TRY(x)             \
    do {                       \
        const int rc_ = (x);   \
        if (rc_) return rc_;   \
    } while (0)

}  // namespace

extern "C" int lastro_kv8_append(lastro_ctx* ctx, const lastro_kv8* kv, const int32_t* lens, const int32_t* new_off,
                                 int32_t max_new, const lastro_rows* k, const lastro_rows* v, int32_t* lens_out,
                                 float* mass, int64_t mass_stride) {
    if (!ctx) return LASTRO_E_ARG;
    KV8_TRY(check_kv(ctx, kv, "kv8_append"));
    KV8_TRY(check_rows(ctx, k, "kv8_append: k"));
    KV8_TRY(check_rows(ctx, v, "kv8_append: v"));
    if (!lens || !new_off || !lens_out) return set_err(ctx, LASTRO_E_ARG, "kv8_append: null lens, new_off or lens_out");
    if (lens == lens_out) return set_err(ctx, LASTRO_E_ARG, "kv8_append: lens_out must not be lens");
    if (misaligned(lens, 4) || misaligned(new_off, 4) || misaligned(lens_out, 4) || misaligned(mass, 4))
        return set_err(ctx, LASTRO_E_ARG, "kv8_append: misaligned lens, new_off, lens_out or mass");
    if (k->dtype != v->dtype) return set_err(ctx, LASTRO_E_ARG, "kv8_append: k and v of different dtypes");
    if (max_new < 0) return set_err(ctx, LASTRO_E_ARG, "kv8_append: max_new %d", max_new);
    if (mass && mass_stride < 1) return set_err(ctx, LASTRO_E_ARG, "kv8_append: mass_stride %lld", (long long)mass_stride);
    Kv8AppendArgs a{};
    a.kv = *kv;
    a.lens = lens;
    a.new_off = new_off;
    a.k = *k;
    a.v = *v;
    // rows beyond the page table are refused on the device, so no sequence takes more, nor more than there are
    a.max_new = (int32_t)std::min({(int64_t)max_new, (int64_t)kv->max_pages * kKv8Page, (int64_t)std::min(k->rows, v->rows)});
    a.blocks = a.max_new ? (a.max_new + 2 * kKv8Block - 2) / kKv8Block : 1;
    a.lens_out = lens_out;
    a.mass = mass;
    a.mass_stride = mass_stride;
    if ((int64_t)a.blocks * kv->kv_heads > INT32_MAX - 7)  // blocks and heads of a sequence, eight to a CTA, counted in 32 bits
        return set_err(ctx, LASTRO_E_UNSUPPORTED, "kv8_append: %d rows of %d KV heads to a sequence in one call", a.max_new,
                       kv->kv_heads);
    KV8_TRY(on_device(ctx, "kv8_append"));
    return launched(ctx, launch_kv8_append(a, ctx->stream), "kv8_append");
}

extern "C" int lastro_kv8_attend_workspace(lastro_ctx* ctx, const lastro_kv8* kv, int32_t heads, int32_t max_new,
                                           int32_t with_mass, size_t* bytes) {
    if (!ctx) return LASTRO_E_ARG;
    KV8_TRY(check_kv(ctx, kv, "kv8_attend_workspace"));
    if (!bytes || heads < 1 || heads % kv->kv_heads || max_new < 0)
        return set_err(ctx, LASTRO_E_ARG, "kv8_attend_workspace: heads %d of %d KV heads, max_new %d", heads, kv->kv_heads,
                       max_new);
    KV8_TRY(on_device(ctx, "kv8_attend_workspace"));
    *bytes = kv8_attend_workspace(*kv, heads, max_new, with_mass != 0, nullptr, nullptr);
    return LASTRO_OK;
}

extern "C" int lastro_kv8_attend(lastro_ctx* ctx, const lastro_kv8* kv, const int32_t* lens, const int32_t* q_off,
                                 int32_t max_new, int32_t heads, const lastro_rows* q, float scale, const lastro_rows* out,
                                 const float* mass_in, float* mass_out, int64_t mass_stride, void* workspace,
                                 size_t workspace_bytes) {
    if (!ctx) return LASTRO_E_ARG;
    KV8_TRY(check_kv(ctx, kv, "kv8_attend"));
    KV8_TRY(check_rows(ctx, q, "kv8_attend: q"));
    KV8_TRY(check_rows(ctx, out, "kv8_attend: out"));
    if (!lens || !q_off || !workspace) return set_err(ctx, LASTRO_E_ARG, "kv8_attend: null lens, q_off or workspace");
    if (misaligned(lens, 4) || misaligned(q_off, 4) || misaligned(mass_in, 4) || misaligned(mass_out, 4))
        return set_err(ctx, LASTRO_E_ARG, "kv8_attend: misaligned lens, q_off or mass");
    if (heads < 1 || heads % kv->kv_heads)
        return set_err(ctx, LASTRO_E_ARG, "kv8_attend: %d heads for %d KV heads", heads, kv->kv_heads);
    if (max_new < 0) return set_err(ctx, LASTRO_E_ARG, "kv8_attend: max_new %d", max_new);
    if (q->dtype != out->dtype || q->rows != out->rows)
        return set_err(ctx, LASTRO_E_ARG, "kv8_attend: out must have q's dtype and rows");
    if ((int64_t)q->rows > (int64_t)kv->n_seqs * max_new)
        return set_err(ctx, LASTRO_E_ARG, "kv8_attend: %d rows for %d sequences of at most %d", q->rows, kv->n_seqs, max_new);
    if (!std::isfinite(scale)) return set_err(ctx, LASTRO_E_ARG, "kv8_attend: scale is not finite");
    if (mass_in && !mass_out) return set_err(ctx, LASTRO_E_ARG, "kv8_attend: mass_in without mass_out");
    if (mass_out && mass_stride < 1) return set_err(ctx, LASTRO_E_ARG, "kv8_attend: mass_stride %lld", (long long)mass_stride);
    size_t need = 0;
    KV8_TRY(lastro_kv8_attend_workspace(ctx, kv, heads, max_new, mass_out != nullptr, &need));
    if (workspace_bytes < need || misaligned(workspace, 16))
        return set_err(ctx, LASTRO_E_ARG, "kv8_attend: workspace of %zu bytes, %zu needed on a 16-byte boundary",
                       workspace_bytes, need);
    Kv8AttendArgs a{};
    a.kv = *kv;
    a.lens = lens;
    a.q_off = q_off;
    a.q = *q;
    a.out = *out;
    a.max_new = max_new;
    a.heads = heads;
    a.group = heads / kv->kv_heads;
    a.scale = scale;
    a.mass_in = mass_in;
    a.mass_out = mass_out;
    a.mass_stride = mass_stride;
    kv8_attend_workspace(*kv, heads, max_new, mass_out != nullptr, &a, workspace);
    if (q->rows > 0 && out->ptr == q->ptr) {  // a unit's rows are read before its outputs are written, but only by the first pass
        if ((q->rows > 1 && q->row_stride != out->row_stride) || (heads > 1 && q->head_stride != out->head_stride))
            return set_err(ctx, LASTRO_E_ARG, "kv8_attend: out at q's address in another layout");
        if (mass_out && !a.scores)
            return set_err(ctx, LASTRO_E_ARG, "kv8_attend: out must not be q, which is read again for the weights");
    }
    if (q->rows == 0 && !mass_out) return LASTRO_OK;
    // counted in 32 bits, the rows that a sequence can have in steps of up to 8192
    if ((int64_t)max_new * a.heads > INT32_MAX || (int64_t)std::min(max_new, q->rows) * a.heads > INT32_MAX - 8192 ||
        kv8_attend_items(*kv, heads, max_new) >= (1 << 30))
        return set_err(ctx, LASTRO_E_UNSUPPORTED, "kv8_attend: n_seqs %d, max_pages %d, max_new %d, heads %d in one call",
                       kv->n_seqs, kv->max_pages, max_new, heads);
    KV8_TRY(on_device(ctx, "kv8_attend"));
    return launched(ctx, launch_kv8_attend(a, ctx->stream), "kv8_attend");
}

extern "C" int lastro_kv8_evict(lastro_ctx* ctx, const lastro_kv8* src, const lastro_kv8* dst, const int32_t* lens,
                                int32_t budget, int32_t recent, const float* mass, int64_t mass_stride, int32_t* kept,
                                int32_t* lens_out, float* mass_out, int64_t mass_out_stride) {
    if (!ctx) return LASTRO_E_ARG;
    KV8_TRY(check_kv(ctx, src, "kv8_evict: src"));
    KV8_TRY(check_kv(ctx, dst, "kv8_evict: dst"));
    if (src->format != dst->format || src->n_seqs != dst->n_seqs || src->kv_heads != dst->kv_heads ||
        src->head_dim != dst->head_dim)
        return set_err(ctx, LASTRO_E_ARG, "kv8_evict: src and dst differ in format, n_seqs, kv_heads or head_dim");
    if (!lens || !kept || !lens_out) return set_err(ctx, LASTRO_E_ARG, "kv8_evict: null lens, kept or lens_out");
    if (lens == lens_out) return set_err(ctx, LASTRO_E_ARG, "kv8_evict: lens_out must not be lens");
    if (misaligned(lens, 4) || misaligned(kept, 4) || misaligned(lens_out, 4) || misaligned(mass, 4) || misaligned(mass_out, 4))
        return set_err(ctx, LASTRO_E_ARG, "kv8_evict: misaligned lens, kept, lens_out or mass");
    if (budget < 1 || budget > (int64_t)dst->max_pages * kKv8Page)
        return set_err(ctx, LASTRO_E_ARG, "kv8_evict: budget %d (1 to the %lld slots of dst's page table)", budget,
                       (long long)dst->max_pages * kKv8Page);
    if (recent < 0 || recent > budget) return set_err(ctx, LASTRO_E_ARG, "kv8_evict: recent %d of budget %d", recent, budget);
    if (!mass && recent != budget) return set_err(ctx, LASTRO_E_ARG, "kv8_evict: null mass with recent %d of budget %d", recent, budget);
    if (mass && mass_stride < 1) return set_err(ctx, LASTRO_E_ARG, "kv8_evict: mass_stride %lld", (long long)mass_stride);
    if (mass_out && (!mass || mass_out_stride < budget))
        return set_err(ctx, LASTRO_E_ARG, "kv8_evict: mass_out needs mass and a stride of at least budget");
    if (mass_out && mass_out == mass) return set_err(ctx, LASTRO_E_ARG, "kv8_evict: mass_out must not be mass");
    Kv8EvictArgs a{};
    a.src = *src;
    a.dst = *dst;
    a.lens = lens;
    a.budget = budget;
    a.recent = recent;
    a.mass = mass;
    a.mass_stride = mass_stride;
    a.kept = kept;
    a.lens_out = lens_out;
    a.mass_out = mass_out;
    a.mass_out_stride = mass_out_stride;
    KV8_TRY(on_device(ctx, "kv8_evict"));
    return launched(ctx, launch_kv8_evict(a, ctx->stream), "kv8_evict");
}

extern "C" int lastro_kv8_read(lastro_ctx* ctx, const lastro_kv8* kv, const int32_t* lens, const int32_t* pos0, int32_t n,
                               void* k_out, void* v_out, int32_t dtype) {
    if (!ctx) return LASTRO_E_ARG;
    KV8_TRY(check_kv(ctx, kv, "kv8_read"));
    if (!lens || !pos0 || n < 0) return set_err(ctx, LASTRO_E_ARG, "kv8_read: null lens or pos0, or n %d", n);
    if (dtype != LASTRO_DTYPE_BF16 && dtype != LASTRO_DTYPE_F32)
        return set_err(ctx, LASTRO_E_ARG, "kv8_read: dtype %d (bf16 or f32)", dtype);
    if (misaligned(lens, 4) || misaligned(pos0, 4)) return set_err(ctx, LASTRO_E_ARG, "kv8_read: misaligned lens or pos0");
    if (misaligned(k_out, 16) || misaligned(v_out, 16))
        return set_err(ctx, LASTRO_E_ARG, "kv8_read: outputs start on 16-byte boundaries");
    if (n == 0 || (!k_out && !v_out)) return LASTRO_OK;
    KV8_TRY(on_device(ctx, "kv8_read"));
    const Kv8ReadArgs a{*kv, lens, pos0, n, k_out, v_out, dtype == LASTRO_DTYPE_F32};
    return launched(ctx, launch_kv8_read(a, ctx->stream), "kv8_read");
}
