// C ABI of the operators beside the search (see include/turbovec_hip.h): checks of the arguments, and the launches on the
// caller's stream.  Nothing here allocates, waits or keeps anything from one call to the next.
#include <cmath>

#include "../../include/turbovec_hip.h"

#include "tv_ops.h"

static_assert(TV_F32 == tv::kF32 && TV_F16 == tv::kF16 && TV_BF16 == tv::kBF16, "types of values");
static_assert(TV_SCALE_E8M0 == tv::kScaleE8M0 && TV_SCALE_F32 == tv::kScaleF32, "types of scales");
static_assert(TV_ROWS_FP8 == tv::kRowsFp8 && TV_ROWS_FP4 == tv::kRowsFp4, "kinds of rows");

namespace {

using tv::op_failed;
using tv::op_refused;

constexpr size_t kMostRows = (size_t(1) << 31) - 1, kMostDim = 16384;

// The device of a call, for its length; the caller's own is current again afterwards.
struct OnDevice {
    int before = -1;
    int rc;
    explicit OnDevice(int device) {
        int count = 0;
        if (hipGetDeviceCount(&count) != hipSuccess || device < 0 || device >= count) {
            op_refused("no HIP device with that ordinal");
            rc = TV_ERR_NO_DEVICE;
            return;
        }
        int now = device;
        hipError_t e = hipGetDevice(&now);
        if (e == hipSuccess && now != device) {
            e = hipSetDevice(device);
            if (e == hipSuccess) before = now;
        }
        rc = e == hipSuccess ? TV_OK : op_failed(e, "hipSetDevice");
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
};

size_t value_bytes(int type) { return type == TV_F32 ? 4 : 2; }
bool value_type(int type) { return type == TV_F32 || type == TV_F16 || type == TV_BF16; }
bool off(const void *p, size_t align) { return reinterpret_cast<uintptr_t>(p) % align != 0; }
size_t blocks_of(size_t dim) { return (dim + tv::kScaleBlock - 1) / tv::kScaleBlock; }

// What is wrong with a set of 8-bit rows, or null.
const char *wrong_rows(const void *codes, const void *scales, size_t rows, size_t dim, int scale_type, int group) {
    if (dim == 0 || dim > kMostDim) return "dim must be 1 to 16384";
    if (rows > kMostRows) return "too many rows";
    if (scale_type != TV_SCALE_E8M0 && scale_type != TV_SCALE_F32) return "unknown type of scales";
    if (group != 1 && group != tv::kScaleBlock) return "a scale is of 1 row or of 128";
    if (rows != 0 && (codes == nullptr || scales == nullptr)) return "null codes or scales";
    if (scale_type == TV_SCALE_F32 && off(scales, 4)) return "scales are not aligned";
    return nullptr;
}
tv::Rows8 rows8(const uint8_t *codes, size_t stride, const void *scales, size_t scale_stride, size_t rows, int group) {
    return tv::Rows8{codes, scales, stride, scale_stride, uint32_t(rows), group == 1 ? 0 : 7};
}

// What is wrong with a set of 4-bit rows, or null.
const char *wrong_rows4(const void *codes, const void *scales, size_t rows, size_t dim) {
    if (dim == 0 || dim > kMostDim) return "dim must be 1 to 16384";
    if (rows > kMostRows) return "too many rows";
    if (rows != 0 && (codes == nullptr || scales == nullptr)) return "null codes or scales";
    return nullptr;
}
size_t code_bytes4(size_t dim) { return (dim + 1) / 2; }
size_t blocks4(size_t dim) { return (dim + tv::kScaleBlock4 - 1) / tv::kScaleBlock4; }
// What is wrong with where 4-bit rows are to be written, or null.
const char *overlap4(size_t rows, size_t dim, size_t code_stride, size_t scale_stride) {
    if (rows > 1 && code_stride < code_bytes4(dim)) return "rows of codes overlap";
    if (rows > 1 && scale_stride < blocks4(dim)) return "rows of scales overlap";
    return nullptr;
}
// What is wrong with rows of scores, their mask and what is asked of them, or null.
const char *wrong_scores(const void *scores, int score_type, size_t rows, size_t n, const void *mask, const void *temperature, const void *slots, size_t given) {
    if (!value_type(score_type)) return "unknown type of values";
    if (rows > kMostRows || n > kMostRows) return "too many rows or scores";
    if (given > tv::kMostGiven) return "at most 128 given slots a row";
    if (rows == 0) return nullptr;
    if (n == 0) return "rows without scores";
    if (scores == nullptr || off(scores, value_bytes(score_type))) return "scores are null or not aligned";
    if (given != 0 && (slots == nullptr || off(slots, 8))) return "slots are null or not aligned";
    if (off(mask, 8) || off(temperature, 4)) return "mask or temperatures are not aligned";
    return nullptr;
}

}  // namespace

extern "C" {

int tv_fp8_quantize_dev(int device, void *stream, const void *d_x, int x_type, size_t x_stride, size_t rows, size_t dim,
                        int scale_type, int group, uint8_t *d_codes, size_t code_stride, void *d_scales, size_t scale_stride) {
    if (const char *why = wrong_rows(d_codes, d_scales, rows, dim, scale_type, group)) return op_refused(why);
    if (!value_type(x_type)) return op_refused("unknown type of values");
    if (rows == 0) return TV_OK;
    if (d_x == nullptr || off(d_x, value_bytes(x_type))) return op_refused("values are null or not aligned");
    if (rows > 1 && code_stride < dim) return op_refused("rows of codes overlap");
    if (rows > size_t(group) && scale_stride < blocks_of(dim)) return op_refused("rows of scales overlap");
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::QuantizeArgs a{d_x, d_codes, d_scales, x_stride, code_stride, scale_stride, uint32_t(rows), uint32_t(dim)};
    const hipError_t e = tv::launch_fp8_quantize(a, x_type, scale_type, group == 1 ? 0 : 7, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_fp8_quantize_dev");
}

int tv_fp8_matmul_dev(int device, void *stream, const uint8_t *d_a, size_t a_stride, const void *d_a_scales, size_t a_scale_stride, size_t m,
                      const uint8_t *d_b, size_t b_stride, const void *d_b_scales, size_t b_scale_stride, size_t n, int group,
                      size_t dim, int scale_type, void *d_out, int out_type, size_t out_stride) {
    if (const char *why = wrong_rows(d_a, d_a_scales, m, dim, scale_type, 1)) return op_refused(why);
    if (const char *why = wrong_rows(d_b, d_b_scales, n, dim, scale_type, group)) return op_refused(why);
    if (!value_type(out_type)) return op_refused("unknown type of values");
    if (m == 0 || n == 0) return TV_OK;
    if (d_out == nullptr || off(d_out, value_bytes(out_type))) return op_refused("the result is null or not aligned");
    if (m > 1 && out_stride < n) return op_refused("rows of the result overlap");
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::MatmulArgs a{rows8(d_a, a_stride, d_a_scales, a_scale_stride, m, 1), rows8(d_b, b_stride, d_b_scales, b_scale_stride, n, group),
                           uint32_t(dim), d_out, out_stride, out_type};
    const hipError_t e = tv::launch_fp8_matmul(a, scale_type, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_fp8_matmul_dev");
}

size_t tv_fp8_rescore_workspace(size_t nq, size_t m, size_t dim) { return tv::rescore_workspace(nq, m, dim); }

int tv_fp8_rescore_dev(int device, void *stream, const void *d_queries, int q_type, size_t q_stride, size_t nq,
                       const uint8_t *d_rows, size_t row_stride, const void *d_scales, size_t scale_stride, size_t n, int group, size_t dim, int scale_type,
                       const int64_t *d_slots, size_t slot_stride, size_t m, size_t k, float *d_out_scores, int64_t *d_out_slots,
                       void *d_workspace, size_t workspace_bytes) {
    if (const char *why = wrong_rows(d_rows, d_scales, n, dim, scale_type, group)) return op_refused(why);
    if (!value_type(q_type)) return op_refused("unknown type of values");
    if (nq > kMostRows) return op_refused("too many queries");
    if (m > tv::kMaxRescore) return op_refused("at most 16384 candidates a query");
    if (k > m) return op_refused("k exceeds the number of candidates");
    if (nq == 0 || k == 0) return TV_OK;
    if (d_queries == nullptr || off(d_queries, value_bytes(q_type))) return op_refused("queries are null or not aligned");
    if (d_slots == nullptr || d_out_scores == nullptr || d_out_slots == nullptr || off(d_slots, 8) || off(d_out_scores, 4) || off(d_out_slots, 8))
        return op_refused("slots or results are null or not aligned");
    if (const size_t need = tv::rescore_workspace(nq, m, dim); need != 0 && (workspace_bytes < need || d_workspace == nullptr || off(d_workspace, 8)))
        return op_refused("workspace is null, not aligned or smaller than tv_fp8_rescore_workspace()");
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::RescoreArgs a{d_queries, d_slots, q_stride, slot_stride, rows8(d_rows, row_stride, d_scales, scale_stride, n, group),
                            uint32_t(dim), uint32_t(nq), uint32_t(m), uint32_t(k), d_out_scores, d_out_slots, static_cast<uint64_t *>(d_workspace)};
    const hipError_t e = tv::launch_fp8_rescore(a, q_type, scale_type, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_fp8_rescore_dev");
}

size_t tv_sample_workspace(size_t rows, size_t n) { return tv::sample_workspace(rows, n); }

int tv_sample_dev(int device, void *stream, const void *d_scores, int score_type, size_t score_stride, size_t rows, size_t n,
                  const uint64_t *d_mask_words, size_t mask_stride, const float *d_u, const float *d_temperature, const int32_t *d_top_k,
                  const float *d_top_p, const float *d_min_p, int64_t *d_out_slots, float *d_out_probs, void *d_workspace, size_t workspace_bytes) {
    if (!value_type(score_type)) return op_refused("unknown type of values");
    if (rows > kMostRows || n > kMostRows) return op_refused("too many rows or scores");
    if (rows == 0) return TV_OK;
    if (n == 0) return op_refused("rows without scores");
    if (d_scores == nullptr || off(d_scores, value_bytes(score_type))) return op_refused("scores are null or not aligned");
    if (d_u == nullptr || d_out_slots == nullptr || d_out_probs == nullptr || off(d_out_slots, 8) || off(d_out_probs, 4) || off(d_u, 4) || off(d_temperature, 4) ||
        off(d_top_k, 4) || off(d_top_p, 4) || off(d_min_p, 4) || off(d_mask_words, 8))
        return op_refused("random numbers, parameters or results are null or not aligned");
    if (const size_t need = tv::sample_workspace(rows, n); need != 0 && (workspace_bytes < need || d_workspace == nullptr || off(d_workspace, 16)))
        return op_refused("workspace is null, not aligned or smaller than tv_sample_workspace()");
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::SampleArgs a{d_scores, d_mask_words, d_u, d_temperature, d_top_p, d_min_p, d_top_k, score_stride, mask_stride,
                           uint32_t(rows), uint32_t(n), d_out_slots, d_out_probs, static_cast<uint8_t *>(d_workspace)};
    const hipError_t e = tv::launch_sample(a, score_type, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_sample_dev");
}

int tv_fp4_quantize_dev(int device, void *stream, const void *d_x, int x_type, size_t x_stride, size_t rows, size_t dim,
                        uint8_t *d_codes, size_t code_stride, uint8_t *d_scales, size_t scale_stride) {
    if (const char *why = wrong_rows4(d_codes, d_scales, rows, dim)) return op_refused(why);
    if (!value_type(x_type)) return op_refused("unknown type of values");
    if (rows == 0) return TV_OK;
    if (d_x == nullptr || off(d_x, value_bytes(x_type))) return op_refused("values are null or not aligned");
    if (const char *why = overlap4(rows, dim, code_stride, scale_stride)) return op_refused(why);
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::Quantize4Args a{d_x, d_codes, d_scales, x_stride, code_stride, scale_stride, uint32_t(rows), uint32_t(dim)};
    const hipError_t e = tv::launch_fp4_quantize(a, x_type, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_fp4_quantize_dev");
}

int tv_fp4_values_dev(int device, void *stream, const uint8_t *d_codes, size_t code_stride, const uint8_t *d_scales, size_t scale_stride,
                      size_t rows, size_t dim, void *d_out, int out_type, size_t out_stride) {
    if (const char *why = wrong_rows4(d_codes, d_scales, rows, dim)) return op_refused(why);
    if (!value_type(out_type)) return op_refused("unknown type of values");
    if (rows == 0) return TV_OK;
    if (d_out == nullptr || off(d_out, value_bytes(out_type))) return op_refused("the result is null or not aligned");
    if (rows > 1 && out_stride < dim) return op_refused("rows of the result overlap");
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::Values4Args a{{d_codes, d_scales, code_stride, scale_stride, uint32_t(rows)}, uint32_t(dim), d_out, out_stride};
    const hipError_t e = tv::launch_fp4_values(a, out_type, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_fp4_values_dev");
}

int tv_fp4_matmul_dev(int device, void *stream, const uint8_t *d_a, size_t a_stride, const uint8_t *d_a_scales, size_t a_scale_stride, size_t m,
                      const uint8_t *d_b, size_t b_stride, const uint8_t *d_b_scales, size_t b_scale_stride, size_t n,
                      size_t dim, void *d_out, int out_type, size_t out_stride) {
    if (const char *why = wrong_rows4(d_a, d_a_scales, m, dim)) return op_refused(why);
    if (const char *why = wrong_rows4(d_b, d_b_scales, n, dim)) return op_refused(why);
    if (!value_type(out_type)) return op_refused("unknown type of values");
    if (m == 0 || n == 0) return TV_OK;
    if (d_out == nullptr || off(d_out, value_bytes(out_type))) return op_refused("the result is null or not aligned");
    if (m > 1 && out_stride < n) return op_refused("rows of the result overlap");
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::Matmul4Args a{{d_a, d_a_scales, a_stride, a_scale_stride, uint32_t(m)}, {d_b, d_b_scales, b_stride, b_scale_stride, uint32_t(n)},
                            uint32_t(dim), d_out, out_stride, out_type};
    const hipError_t e = tv::launch_fp4_matmul(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_fp4_matmul_dev");
}

int tv_rms_norm_dev(int device, void *stream, const void *d_x, int x_type, size_t x_stride, const void *d_residual, size_t residual_stride,
                    void *d_sum, size_t sum_stride, const void *d_weight, int weight_type, float eps, size_t rows, size_t dim,
                    int row_kind, int scale_type, uint8_t *d_codes, size_t code_stride, void *d_scales, size_t scale_stride) {
    if (row_kind != TV_ROWS_FP8 && row_kind != TV_ROWS_FP4) return op_refused("unknown kind of rows");
    if (row_kind == TV_ROWS_FP4 && scale_type != TV_SCALE_E8M0) return op_refused("4-bit rows have e8m0 scales");
    if (const char *why = row_kind == TV_ROWS_FP4 ? wrong_rows4(d_codes, d_scales, rows, dim) : wrong_rows(d_codes, d_scales, rows, dim, scale_type, 1)) return op_refused(why);
    if (!value_type(x_type) || (d_weight != nullptr && !value_type(weight_type))) return op_refused("unknown type of values");
    if (!(eps >= 0.0f) || std::isinf(eps)) return op_refused("eps must be finite and not below 0");
    if (rows == 0) return TV_OK;
    const size_t size = value_bytes(x_type);
    if (d_x == nullptr || off(d_x, size) || off(d_residual, size) || off(d_sum, size)) return op_refused("values are null or not aligned");
    if (d_weight != nullptr && off(d_weight, value_bytes(weight_type))) return op_refused("the weight is not aligned");
    if (d_sum != nullptr && rows > 1 && sum_stride < dim) return op_refused("rows of the sum overlap");
    if (rows > 1 && d_sum != nullptr && ((d_sum == d_x && sum_stride != x_stride) || (d_sum == d_residual && sum_stride != residual_stride)))
        return op_refused("the sum takes the place of an input with another stride");
    if (row_kind == TV_ROWS_FP4) {
        if (const char *why = overlap4(rows, dim, code_stride, scale_stride)) return op_refused(why);
    } else {
        if (rows > 1 && code_stride < dim) return op_refused("rows of codes overlap");
        if (rows > 1 && scale_stride < blocks_of(dim)) return op_refused("rows of scales overlap");
    }
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::NormArgs a{d_x, d_residual, d_sum, d_weight, d_codes, d_scales, x_stride, residual_stride, sum_stride, code_stride, scale_stride,
                         uint32_t(rows), uint32_t(dim), 1.0 / double(dim), weight_type, eps};
    const hipError_t e = tv::launch_rms_norm(a, x_type, row_kind, scale_type, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_rms_norm_dev");
}

size_t tv_log_probs_workspace(size_t rows, size_t n, size_t top) { return tv::log_probs_workspace(rows, n, top); }

int tv_log_probs_dev(int device, void *stream, const void *d_scores, int score_type, size_t score_stride, size_t rows, size_t n,
                     const uint64_t *d_mask_words, size_t mask_stride, const float *d_temperature, const int64_t *d_slots, size_t slot_stride, size_t given,
                     size_t top, float *d_out_log_probs, float *d_out_entropy, int64_t *d_out_top_slots, float *d_out_top_log_probs, float *d_out_stats,
                     void *d_workspace, size_t workspace_bytes) {
    if (const char *why = wrong_scores(d_scores, score_type, rows, n, d_mask_words, d_temperature, d_slots, given)) return op_refused(why);
    if (top > tv::kMostTop) return op_refused("at most 128 alternatives a row");
    if (rows == 0) return TV_OK;
    if ((given != 0 && d_out_log_probs == nullptr) || d_out_entropy == nullptr || (top != 0 && (d_out_top_slots == nullptr || d_out_top_log_probs == nullptr)) ||
        off(d_out_log_probs, 4) || off(d_out_entropy, 4) || off(d_out_top_slots, 8) || off(d_out_top_log_probs, 4) || off(d_out_stats, 16))
        return op_refused("results are null or not aligned");
    if (const size_t need = tv::log_probs_workspace(rows, n, top); need != 0 && (workspace_bytes < need || d_workspace == nullptr || off(d_workspace, 16)))
        return op_refused("workspace is null, not aligned or smaller than tv_log_probs_workspace()");
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::LogProbArgs a{d_scores, d_mask_words, d_temperature, d_slots, score_stride, mask_stride, slot_stride, uint32_t(rows), uint32_t(n), uint32_t(given), uint32_t(top),
                            d_out_log_probs, d_out_entropy, d_out_top_slots, d_out_top_log_probs, d_out_stats, static_cast<uint8_t *>(d_workspace)};
    const hipError_t e = tv::launch_log_probs(a, score_type, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_log_probs_dev");
}

int tv_log_probs_grad_dev(int device, void *stream, const void *d_scores, int score_type, size_t score_stride, size_t rows, size_t n,
                          const uint64_t *d_mask_words, size_t mask_stride, const float *d_temperature, const int64_t *d_slots, size_t slot_stride, size_t given,
                          const float *d_stats, const float *d_grad_log_probs, const float *d_grad_entropy, void *d_grad_scores, size_t grad_stride) {
    if (const char *why = wrong_scores(d_scores, score_type, rows, n, d_mask_words, d_temperature, d_slots, given)) return op_refused(why);
    if (rows == 0) return TV_OK;
    if (d_stats == nullptr || off(d_stats, 16) || off(d_grad_log_probs, 4) || off(d_grad_entropy, 4)) return op_refused("stats are null, or stats or gradients are not aligned");
    if (d_grad_scores == nullptr || off(d_grad_scores, value_bytes(score_type))) return op_refused("the result is null or not aligned");
    if (rows > 1 && grad_stride < n) return op_refused("rows of the result overlap");
    OnDevice on(device);
    if (on.rc != TV_OK) return on.rc;
    const tv::LogProbGradArgs a{d_scores, d_mask_words, d_temperature, d_slots, score_stride, mask_stride, slot_stride, uint32_t(rows), uint32_t(n),
                                d_grad_log_probs == nullptr ? 0u : uint32_t(given), d_stats, d_grad_log_probs, d_grad_entropy, d_grad_scores, grad_stride};
    const hipError_t e = tv::launch_log_probs_grad(a, score_type, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? TV_OK : op_failed(e, "tv_log_probs_grad_dev");
}

}  // extern "C"
