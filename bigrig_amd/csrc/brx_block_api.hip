// The C-ABI of the operators around a block's experts: validation and dispatch (kernels in k_pairs.hip,
// k_grouped.hip, k_norm.hip).
#include "block_ops.h"

using namespace brx;

namespace {

constexpr int64_t kMaxRows = (int64_t)1 << 23;      // pairs, sorted rows or tokens of one call: a grid of a block a row stays under 2^32 threads
constexpr int64_t kMaxRowStride = (int64_t)1 << 20; // of a weight: a tile's offsets stay inside 31 bits

int hip_result(hipError_t e, const char* what) {
    return e == hipSuccess ? BRX_OK : api_fail(BRX_EHIP, "%s: %s", what, hipGetErrorString(e));
}

bool known_dtype(int dt) { return dt == BRX_DT_F32 || dt == BRX_DT_BF16 || dt == BRX_DT_F16; }
bool aligned_to(const void* p, int dt) { return ((uintptr_t)p & (dtype_bytes(dt) - 1)) == 0; }

int check_pairs(int64_t T, int k) {
    if (T < 0) return api_fail(BRX_EINVAL, "T %lld is negative", (long long)T);
    if (k < 1 || k > kMaxTopK) return api_fail(BRX_EINVAL, "k %d outside [1, %d]", k, kMaxTopK);
    if (T * k > kMaxRows) return api_fail(BRX_EINVAL, "%lld pairs in one call: at most %lld", (long long)(T * k), (long long)kMaxRows);
    return BRX_OK;
}
int check_experts(int E) {
    return E < 1 || E > kMaxExperts ? api_fail(BRX_EINVAL, "%d experts outside [1, %d]", E, kMaxExperts) : BRX_OK;
}
int check_width(int H) {
    return H < 1 || H > kMaxWidth ? api_fail(BRX_EINVAL, "rows of %d values: 1 to %d", H, kMaxWidth) : BRX_OK;
}
int check_rows(int64_t T, int k, int H, int dtype) {
    int rc = check_pairs(T, k);
    if (rc) return rc;
    if ((rc = check_width(H))) return rc;
    if (!known_dtype(dtype)) return api_fail(BRX_EINVAL, "dtype %d unknown", dtype);
    return api_ready();
}

int check_grouped(int64_t P, int E, int K, int N, int dtype) {
    if (P < 0 || P > kMaxRows) return api_fail(BRX_EINVAL, "%lld rows outside [0, %lld]", (long long)P, (long long)kMaxRows);
    const int rc = check_experts(E);
    if (rc) return rc;
    for (const int w : {K, N})
        if (w < 8 || w % 8 || w > kMaxWidth) return api_fail(BRX_EINVAL, "width %d: a multiple of 8 up to %d", w, kMaxWidth);
    if (dtype != BRX_DT_BF16 && dtype != BRX_DT_F16) return api_fail(BRX_EINVAL, "grouped products take bf16 or fp16 (dtype %d)", dtype);
    return api_ready();
}
int check_weight(int64_t w_expert, int64_t w_row, int K) {
    if (w_row < K || w_row > kMaxRowStride || w_row % 8 || w_expert < 0 || w_expert % 8)
        return api_fail(BRX_EINVAL, "weights %lld and %lld values between experts and rows: multiples of 8, rows from %d to %lld apart",
                        (long long)w_expert, (long long)w_row, K, (long long)kMaxRowStride);
    return BRX_OK;
}
int check_16(std::initializer_list<const void*> ps, const char* names) {
    for (const void* p : ps) {
        if (!p) return api_fail(BRX_EINVAL, "%s are required", names);
        if ((uintptr_t)p & 15) return api_fail(BRX_EINVAL, "%s must be 16-byte aligned", names);
    }
    return BRX_OK;
}

int check_norm(const NormArgs& a, int y_dt, int r_dt) {
    if (a.T < 0 || a.T > kMaxRows) return api_fail(BRX_EINVAL, "%d rows outside [0, %lld]", a.T, (long long)kMaxRows);
    int rc = check_width(a.H);
    if (rc) return rc;
    if (!known_dtype(y_dt) || (r_dt != y_dt && r_dt != BRX_DT_F32))
        return api_fail(BRX_EINVAL, "y of dtype %d with r of dtype %d: the same, or r fp32", y_dt, r_dt);
    if (!a.T) return api_ready();       // (tensors without rows have no addresses)
    if (a.gate_form < kGateNone || a.gate_form > kGateFull || (a.gate_form == kGateNone) != (a.gate == nullptr))
        return api_fail(BRX_EINVAL, "gate form %d %s a gate", a.gate_form, a.gate ? "with" : "without");
    if ((a.post && !known_dtype(a.post_dt)) || (a.next && !known_dtype(a.next_dt)) || (a.gate && !known_dtype(a.gate_dt)))
        return api_fail(BRX_EINVAL, "dtype of the weights or the gate unknown");
    if (!a.y && (a.post || a.gate)) return api_fail(BRX_EINVAL, "post and gate belong to y, which is not given");
    if ((rc = api_ready())) return rc;
    if (!a.r && (a.new_r || a.h || a.d_h)) return api_fail(BRX_EINVAL, "r is required");
    if (!aligned_to(a.r, r_dt) || !aligned_to(a.y, y_dt)) return api_fail(BRX_EINVAL, "y and r must be aligned to their types");
    if ((a.post && !aligned_to(a.post, a.post_dt)) || (a.next && !aligned_to(a.next, a.next_dt)) || (a.gate && !aligned_to(a.gate, a.gate_dt)))
        return api_fail(BRX_EINVAL, "weights and gate must be aligned to their types");
    return BRX_OK;
}

}  // namespace

extern "C" {

int brx_pairs_workspace_bytes(int64_t n_pairs, int n_experts, size_t* out) {
    if (!out) return api_fail(BRX_EINVAL, "out is NULL");
    if (n_pairs < 0 || n_pairs > kMaxRows) return api_fail(BRX_EINVAL, "%lld pairs outside [0, %lld]", (long long)n_pairs, (long long)kMaxRows);
    const int rc = check_experts(n_experts);
    if (rc) return rc;
    *out = pairs_plan_workspace(n_pairs, n_experts);
    return BRX_OK;
}

int brx_pairs_plan(const int32_t* idx, int T, int k, int E, int32_t* order, int32_t* position, int32_t* offsets,
                   void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_pairs(T, k);
    if (rc) return rc;
    if ((rc = check_experts(E))) return rc;
    if ((rc = api_ready())) return rc;
    if (!offsets) return api_fail(BRX_EINVAL, "offsets is required");
    const int64_t n = (int64_t)T * k;
    if (n && (!idx || !order || !position)) return api_fail(BRX_EINVAL, "idx, order and position are required");
    if (((uintptr_t)idx | (uintptr_t)order | (uintptr_t)position | (uintptr_t)offsets | (uintptr_t)workspace) & 3)
        return api_fail(BRX_EINVAL, "idx, order, position, offsets and workspace must be 4-byte aligned");
    const size_t need = pairs_plan_workspace(n, E);
    if (need && (!workspace || workspace_bytes < need))
        return api_fail(BRX_EINVAL, "a plan of %lld pairs needs %zu bytes of workspace, got %zu", (long long)n, need,
                        workspace ? workspace_bytes : 0);
    const PairsPlan p{idx, order, position, offsets, (int32_t*)workspace, (int)n, E};
    return hip_result(launch_pairs_plan(p, (hipStream_t)stream), "plan launch");
}

int brx_pairs_dispatch(const void* x, int64_t x_row, const int32_t* position, int T, int k, int H, int dtype, void* rows,
                       void* stream) {
    int rc = check_rows(T, k, H, dtype);
    if (rc) return rc;
    if (!T) return BRX_OK;
    if (!x || !position || !rows) return api_fail(BRX_EINVAL, "x, position and rows are required");
    if (!aligned_to(x, dtype) || !aligned_to(rows, dtype)) return api_fail(BRX_EINVAL, "x and rows must be aligned to their type");
    const PairRows p{x, nullptr, position, nullptr, rows, nullptr, x_row, T, k, H};
    return hip_result(launch_pairs_dispatch(p, dtype, (hipStream_t)stream), "dispatch launch");
}

int brx_pairs_combine(const void* rows, const float* w, const int32_t* position, int T, int k, int H, int dtype, void* out,
                      void* stream) {
    int rc = check_rows(T, k, H, dtype);
    if (rc) return rc;
    if (!T) return BRX_OK;
    if (!rows || !position || !out) return api_fail(BRX_EINVAL, "rows, position and out are required");
    if (!aligned_to(rows, dtype) || !aligned_to(out, dtype)) return api_fail(BRX_EINVAL, "rows and out must be aligned to their type");
    const PairRows p{nullptr, rows, position, w, out, nullptr, 0, T, k, H};
    return hip_result(launch_pairs_combine(p, dtype, (hipStream_t)stream), "combine launch");
}

int brx_pairs_combine_backward(const void* dout, int64_t dout_row, const void* rows, const float* w, const int32_t* position,
                               int T, int k, int H, int dtype, void* drows, float* dw, void* stream) {
    int rc = check_rows(T, k, H, dtype);
    if (rc) return rc;
    if (!T || (!drows && !dw)) return BRX_OK;
    if (!dout || !position || (dw && !rows)) return api_fail(BRX_EINVAL, "dout, position and (for dw) rows are required");
    if (!aligned_to(dout, dtype) || !aligned_to(rows, dtype) || !aligned_to(drows, dtype))
        return api_fail(BRX_EINVAL, "dout, rows and drows must be aligned to their type");
    const PairRows p{dout, rows, position, w, drows, dw, dout_row, T, k, H};
    if (!dw) return hip_result(launch_pairs_dispatch(p, dtype, (hipStream_t)stream), "combine gradient launch");
    return hip_result(launch_pairs_combine_backward(p, dtype, (hipStream_t)stream), "combine gradient launch");
}

int brx_grouped_product(const void* rows, const void* weight, int64_t w_expert, int64_t w_row, const void* bias,
                        const int32_t* offsets, int P, int E, int K, int N, int dtype, void* out, void* stream) {
    int rc = check_grouped(P, E, K, N, dtype);
    if (rc) return rc;
    if ((rc = check_weight(w_expert, w_row, K))) return rc;
    if (!P) return BRX_OK;
    if ((rc = check_16({rows, weight, out}, "rows, weight and out"))) return rc;
    if (!offsets || ((uintptr_t)bias & 1)) return api_fail(BRX_EINVAL, "offsets are required, bias aligned to its type");
    const GroupedArgs g{(const uint16_t*)rows, (const uint16_t*)weight, (const uint16_t*)bias, (uint16_t*)out, offsets, w_expert, w_row, P, E, K, N, false};
    return hip_result(launch_grouped_rows(g, false, dtype, (hipStream_t)stream), "grouped product launch");
}

int brx_grouped_product_backward(const void* dout, const void* rows, const void* weight, int64_t w_expert, int64_t w_row,
                                 const int32_t* offsets, int P, int E, int K, int N, int dtype, void* drows, void* dweight,
                                 void* dbias, void* stream) {
    int rc = check_grouped(P, E, K, N, dtype);
    if (rc) return rc;
    if (!offsets) return api_fail(BRX_EINVAL, "offsets are required");
    if (P && (!dout || ((uintptr_t)dout & 15))) return api_fail(BRX_EINVAL, "dout is required, 16-byte aligned");
    if (drows && P) {
        if ((rc = check_weight(w_expert, w_row, K))) return rc;
        if ((rc = check_16({weight, drows}, "weight and drows"))) return rc;
    }
    if (dweight && (((uintptr_t)dweight & 15) || (P && (!rows || ((uintptr_t)rows & 15)))))
        return api_fail(BRX_EINVAL, "rows and dweight must be 16-byte aligned, and rows given");
    if ((uintptr_t)dbias & 1) return api_fail(BRX_EINVAL, "dbias must be aligned to its type");
    const hipStream_t s = (hipStream_t)stream;
    if (drows && P) {
        // (the reduction runs over W's N rows, the output over its K columns)
        const GroupedArgs g{(const uint16_t*)dout, (const uint16_t*)weight, nullptr, (uint16_t*)drows, offsets, w_expert, w_row, P, E, N, K, false};
        if ((rc = hip_result(launch_grouped_rows(g, true, dtype, s), "grouped product row gradient launch"))) return rc;
    }
    if (dweight) {
        const GroupedArgs g{(const uint16_t*)dout, (const uint16_t*)rows, nullptr, (uint16_t*)dweight, offsets, 0, 0, P, E, N, K, false};
        if ((rc = hip_result(launch_grouped_weight(g, dtype, s), "grouped product weight gradient launch"))) return rc;
    }
    if (dbias) {
        const GroupedArgs g{(const uint16_t*)dout, nullptr, nullptr, (uint16_t*)dbias, offsets, 0, 0, P, E, N, 0, false};
        return hip_result(launch_grouped_bias(g, dtype, s), "grouped product bias gradient launch");
    }
    return BRX_OK;
}

int brx_norm_workspace_bytes(int T, int H, size_t* out) {
    if (!out) return api_fail(BRX_EINVAL, "out is NULL");
    if (T < 0 || T > kMaxRows) return api_fail(BRX_EINVAL, "%d rows outside [0, %lld]", T, (long long)kMaxRows);
    const int rc = check_width(H);
    if (rc) return rc;
    *out = (size_t)3 * norm_blocks(T, H) * H * sizeof(float);
    return BRX_OK;
}

int brx_norm_forward(const void* y, int64_t y_row, int y_dtype, const void* r, int64_t r_row, int r_dtype, const void* post,
                     int post_dtype, const void* gate, int gate_form, int gate_dtype, const void* next, int next_dtype,
                     float scale, float eps, int T, int H, void* new_r, void* h, float* rstd_y, float* rstd_n, void* stream) {
    NormArgs a{};
    a.y = y; a.r = r; a.post = post; a.next = next; a.gate = gate; a.new_r = new_r; a.h = h;
    a.rstd_y = rstd_y; a.rstd_n = rstd_n; a.y_row = y_row; a.r_row = r_row; a.scale = scale; a.eps = eps; a.T = T; a.H = H;
    a.gate_form = gate_form; a.post_dt = post_dtype; a.next_dt = next_dtype; a.gate_dt = gate_dtype;
    const int rc = check_norm(a, y_dtype, r_dtype);
    if (rc) return rc;
    if (!(eps >= 1.17549435e-38f) || eps > 3.4e38f) return api_fail(BRX_EINVAL, "eps %g must be a positive, normal fp32 value", (double)eps);
    if (!T) return BRX_OK;
    if (y ? !new_r : !h) return api_fail(BRX_EINVAL, "new_r (or, without y, h) is required");
    if (!y && new_r) return api_fail(BRX_EINVAL, "new_r belongs to y, which is not given");
    if ((new_r && !aligned_to(new_r, r_dtype)) || (h && !aligned_to(h, y_dtype)))
        return api_fail(BRX_EINVAL, "new_r and h must be aligned to their types");
    return hip_result(launch_norm_forward(a, y_dtype, r_dtype, (hipStream_t)stream), "norm launch");
}

int brx_norm_backward(const void* y, int64_t y_row, int y_dtype, const void* r, int64_t r_row, int r_dtype, const void* post,
                      int post_dtype, const void* gate, int gate_form, int gate_dtype, const void* next, int next_dtype,
                      float scale, int T, int H, const float* rstd_y, const float* rstd_n, const void* d_new, const void* d_h,
                      void* dy, void* dr, void* dgate, void* dpost, void* dnext, void* workspace, size_t workspace_bytes,
                      void* stream) {
    NormArgs a{};
    a.y = y; a.r = r; a.post = post; a.next = next; a.gate = gate;
    a.rstd_y = const_cast<float*>(rstd_y); a.rstd_n = const_cast<float*>(rstd_n);
    a.d_new = d_new; a.d_h = d_h; a.dy = dy; a.dr = dr; a.dgate = dgate; a.dpost = dpost; a.dnext = dnext;
    a.y_row = y_row; a.r_row = r_row; a.scale = scale; a.T = T; a.H = H;
    a.gate_form = gate_form; a.post_dt = post_dtype; a.next_dt = next_dtype; a.gate_dt = gate_dtype;
    a.partial = (float*)workspace;
    const int rc = check_norm(a, y_dtype, r_dtype);
    if (rc) return rc;
    if (!T) return BRX_OK;      // (the column sums of no rows are the caller's to clear)
    if ((post && !rstd_y) || (d_h && !rstd_n)) return api_fail(BRX_EINVAL, "rstd_y (with post) and rstd_n (with d_h) are required");
    if ((!y && (dy || dgate || dpost)) || (dgate && !gate) || (dpost && !post) || (dnext && !(next && d_h)))
        return api_fail(BRX_EINVAL, "a gradient of what is not given");
    for (const void* p : {d_new, (const void*)dr})
        if (!aligned_to(p, r_dtype)) return api_fail(BRX_EINVAL, "d_new and dr must be aligned to their type");
    for (const void* p : {d_h, (const void*)dy})
        if (!aligned_to(p, y_dtype)) return api_fail(BRX_EINVAL, "d_h and dy must be aligned to their type");
    if (dpost || dnext || (dgate && gate_form == kGateChannel)) {
        const size_t need = (size_t)3 * norm_blocks(T, H) * H * sizeof(float);
        if (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < need)
            return api_fail(BRX_EINVAL, "column sums of %d rows of %d values need %zu bytes of workspace, got %zu", T, H, need,
                            workspace ? workspace_bytes : 0);
    }
    return hip_result(launch_norm_backward(a, y_dtype, r_dtype, (hipStream_t)stream), "norm gradient launch");
}

}  // extern "C"
