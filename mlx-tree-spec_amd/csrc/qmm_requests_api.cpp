// C ABI of the per-request operators (declared in include/qmm_requests.h): argument checks and launches.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <mutex>

#include "qmm4.h"
#include "qmm4_dispatch.h"
#include "qmm4_kernels.h"
#include "qmm_requests.h"
#include "qmm_requests_kernels.h"

namespace {

using qmm4::hip_error;
using qmm4::set_error;

constexpr int64_t kMaxDim = 1LL << 30;
constexpr int64_t kMaxLoraRows = 1LL << 26;  // (row numbers of a tile past the last stay far below 2^31)

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// No exception leaves a C entry point (the host state's maps and messages may allocate).
template <class F>
int guarded(F&& f) {
  try {
    qmm4::clear_error();
    return f();
  } catch (const std::exception&) {
    return QMM4_ERR_NOMEM;
  }
}

int index_bits_ok(int bits, const char* what) {
  if (bits != 32 && bits != 64) return set_error(QMM4_ERR_UNSUPPORTED, "%s of %d bits: 32 or 64 are supported", what, bits);
  return QMM4_OK;
}

int check_lora(const void* x, const void* a, const void* b, const float* scale, const void* adapters, int adapter_bits,
               const void* y, const void* workspace, int64_t M, int64_t N, int64_t K, int64_t L, int64_t R) {
  if (int rc = index_bits_ok(adapter_bits, "adapters")) return rc;
  if (M < 0 || N < 0 || K <= 0 || L < 0 || M > kMaxLoraRows || N > kMaxDim || K > kMaxDim || L > kMaxDim || K % 8 != 0)
    return set_error(QMM4_ERR_INVALID, "invalid shape M=%lld N=%lld K=%lld L=%lld (K must be a positive multiple of 8, "
                     "at most 2^26 rows, each other at most 2^30)", (long long)M, (long long)N, (long long)K, (long long)L);
  if (R < 8 || R > QMM4_LORA_MAX_RANK || R % 8 != 0)
    return set_error(QMM4_ERR_INVALID, "R=%lld must be a multiple of 8 from 8 to %d", (long long)R, QMM4_LORA_MAX_RANK);
  if (M == 0 || N == 0 || L == 0) return QMM4_OK;
  if (!x || !a || !b || !scale || !adapters || !y || !workspace) return set_error(QMM4_ERR_INVALID, "null pointer argument");
  if (!aligned(x, 16) || !aligned(a, 16) || !aligned(b, 16) || !aligned(workspace, 16))
    return set_error(QMM4_ERR_INVALID, "x, lora_a, lora_b and workspace must be 16-byte aligned");
  if (!aligned(scale, 4) || !aligned(adapters, adapter_bits / 8) || !aligned(y, 2))
    return set_error(QMM4_ERR_INVALID, "lora_scale, adapters and y must be aligned to their elements");
  return QMM4_OK;
}

struct Lora {
  qmm4::LoraTables tables;
  qmm4::LoraAdd add;
  Lora(const void* a, const void* b, const float* scale, const void* adapters, int adapter_bits, void* workspace,
       int64_t L, int64_t R) {
    const qmm4::Index ids{adapters, adapter_bits == 64};
    tables = {static_cast<const uint16_t*>(a), scale, ids, L, (int)R};
    add = {static_cast<const uint32_t*>(workspace), static_cast<const uint16_t*>(b), ids, L, (int)R};
  }
};

// x A^T into the caller's workspace (api_mutex held).
int run_shrink(qmm4::DeviceInfo* di, qmm4::WorkspaceSource& ws, const Lora& lora, const void* x, void* workspace,
               int64_t M, int64_t K, hipStream_t stream) {
  const qmm4::LoraShrinkPlan plan = qmm4::lora_shrink_plan(lora.tables, (int)M, (int)K, qmm4::device_cus(di));
  uint32_t* cnt = nullptr;
  float* part = nullptr;
  if (plan.part_bytes > 0)
    if (int rc = ws.get(plan.counter_bytes, plan.part_bytes, &cnt, &part)) return rc;
  const hipError_t e = qmm4::launch_lora_shrink(plan, lora.tables, static_cast<const uint16_t*>(x),
                                                static_cast<uint32_t*>(workspace), part, cnt, (int)M, (int)K, stream);
  if (e != hipSuccess) return hip_error(e, "adapter shrink kernel launch");
  return QMM4_OK;
}

int check_sample_shape(int64_t M, int64_t V) {
  if (M < 0 || M > (1LL << 20) || V < 1 || V > QMM4_SAMPLE_MAX_VOCAB)
    return set_error(QMM4_ERR_INVALID, "invalid shape M=%lld V=%lld (at most 2^20 rows, 1 to %d tokens)", (long long)M,
                     (long long)V, QMM4_SAMPLE_MAX_VOCAB);
  return QMM4_OK;
}

int current_cus(int* cus) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_error(e, "hipGetDevice");
  std::lock_guard<std::mutex> lock(qmm4::api_mutex());
  qmm4::DeviceInfo* di = nullptr;
  if (int rc = qmm4::device_info(dev, &di)) return rc;
  *cus = qmm4::device_cus(di);
  return QMM4_OK;
}

}  // namespace

extern "C" {

int64_t qmm4_lora_workspace(int64_t M, int64_t R) { return M > 0 && R > 0 ? M * R * (int64_t)sizeof(uint32_t) : 0; }

int qmm4_lora_add_bf16(const void* x, const void* lora_a, const void* lora_b, const float* lora_scale,
                       const void* adapters, int adapter_bits, void* y, void* workspace, int64_t M, int64_t N,
                       int64_t K, int64_t L, int64_t R, void* hip_stream) {
  return guarded([&] {
    int rc = check_lora(x, lora_a, lora_b, lora_scale, adapters, adapter_bits, y, workspace, M, N, K, L, R);
    if (rc || M == 0 || N == 0 || L == 0) return rc;
    const Lora lora(lora_a, lora_b, lora_scale, adapters, adapter_bits, workspace, L, R);
    const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    return qmm4::with_stream_workspace(stream, [&](qmm4::DeviceInfo* di, qmm4::WorkspaceSource& ws) {
      if (int rc2 = run_shrink(di, ws, lora, x, workspace, M, K, stream)) return rc2;
      const hipError_t e = qmm4::launch_lora_expand(lora.add, static_cast<uint16_t*>(y), (int)M, (int)N, stream);
      if (e != hipSuccess) return hip_error(e, "adapter expand kernel launch");
      return (int)QMM4_OK;
    });
  });
}

int qmm4_affine_lora_bf16(const void* x, const uint32_t* w, const void* scales, const void* biases,
                          const void* lora_a, const void* lora_b, const float* lora_scale, const void* adapters,
                          int adapter_bits, void* y, void* workspace, int64_t M, int64_t N, int64_t K, int64_t L,
                          int64_t R, int group_size, int bits, int transpose, void* hip_stream) {
  return guarded([&] {
    if (transpose != 1) return set_error(QMM4_ERR_UNSUPPORTED, "transpose=%d: only transpose=True is supported", transpose);
    const bool packed = bits == 4 && group_size == 64 && K % 128 == 0 && N % 16 == 0;
    int rc = packed ? qmm4::check_qmm_args(x, w, scales, biases, y, M, N, K, group_size, bits, transpose)
                    : qmm4::check_general_args(x, w, scales, biases, y, M, N, K, group_size, bits);
    if (rc) return rc;
    rc = check_lora(x, lora_a, lora_b, lora_scale, adapters, adapter_bits, y, workspace, M, N, K, L, R);
    if (rc || M == 0 || N == 0) return rc;
    const Lora lora(lora_a, lora_b, lora_scale, adapters, adapter_bits, workspace, L, R);
    const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    return qmm4::with_stream_workspace(stream, [&](qmm4::DeviceInfo* di, qmm4::WorkspaceSource& ws) {
      const qmm4::LoraAdd* add = L > 0 ? &lora.add : nullptr;
      if (add)
        if (int rc2 = run_shrink(di, ws, lora, x, workspace, M, K, stream)) return rc2;
      if (packed) return qmm4::dispatch_qmm(di, x, w, scales, biases, y, M, N, K, stream, ws, add);
      const hipError_t e = qmm4::launch_general(static_cast<const uint16_t*>(x), w, static_cast<const uint16_t*>(scales),
                                                static_cast<const uint16_t*>(biases), static_cast<uint16_t*>(y), (int)M,
                                                (int)N, (int)K, group_size, bits, qmm4::device_cus(di), stream, add);
      if (e != hipSuccess) return hip_error(e, "general quantized matmul kernel launch");
      return (int)QMM4_OK;
    });
  });
}

int qmm4_qk_norm_rope_bf16(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                           const void* q_weight, const void* k_weight, float eps, const void* positions,
                           int position_bits, const void* inv_freq, int freq_bits, void* q_out, void* k_out,
                           int64_t M, int64_t Hq, int64_t Hk, int64_t D, int64_t P, int interleaved,
                           void* hip_stream) {
  return guarded([&] {
    if (int rc = index_bits_ok(position_bits, "positions")) return rc;
    if (int rc = index_bits_ok(freq_bits, "inv_freq")) return rc;
    if (M < 0 || M > kMaxDim || Hq < 0 || Hk < 0 || Hq + Hk > 65536)
      return set_error(QMM4_ERR_INVALID, "invalid shape M=%lld, %lld and %lld heads", (long long)M, (long long)Hq, (long long)Hk);
    if (D <= 0 || D % 8 != 0 || D > QMM4_HEAD_MAX_DIM)
      return set_error(QMM4_ERR_INVALID, "D=%lld must be a positive multiple of 8, at most %d", (long long)D, QMM4_HEAD_MAX_DIM);
    if (P < 0 || 2 * P > D)
      return set_error(QMM4_ERR_INVALID, "P=%lld frequencies do not fit heads of %lld", (long long)P, (long long)D);
    if (!(eps >= 0.0f) || std::isinf(eps)) return set_error(QMM4_ERR_INVALID, "eps must be finite and >= 0");
    if (M == 0 || Hq + Hk == 0) return (int)QMM4_OK;
    const struct {
      const void *x, *w, *out;
      int64_t row, head, heads;
    } sides[] = {{q, q_weight, q_out, q_row, q_head, Hq}, {k, k_weight, k_out, k_row, k_head, Hk}};
    for (const auto& s : sides) {
      if (s.heads == 0) continue;
      if (!s.x || !s.w || !s.out) return set_error(QMM4_ERR_INVALID, "null pointer argument");
      if (!aligned(s.x, 16) || !aligned(s.w, 16) || !aligned(s.out, 16) || s.row % 8 != 0 || s.head % 8 != 0)
        return set_error(QMM4_ERR_INVALID, "heads, weights and outputs must be 16-byte aligned, strides multiples of 8");
    }
    if (!positions || (P > 0 && !inv_freq)) return set_error(QMM4_ERR_INVALID, "null pointer argument");
    if (!aligned(positions, position_bits / 8) || !aligned(inv_freq, freq_bits / 8))
      return set_error(QMM4_ERR_INVALID, "positions and inv_freq must be aligned to their elements");
    auto side = [](const void* x, int64_t row, int64_t head, const void* w, void* out, int64_t heads) {
      return qmm4::RopeHeads{static_cast<const uint16_t*>(x), row, head, static_cast<const uint16_t*>(w),
                             static_cast<uint16_t*>(out), (int)heads};
    };
    const qmm4::RopeParams p{side(q, q_row, q_head, q_weight, q_out, Hq), side(k, k_row, k_head, k_weight, k_out, Hk),
                             {positions, position_bits == 64}, inv_freq, freq_bits == 64, eps, (int)D, (int)P};
    hipError_t e = qmm4::launch_qk_norm_rope(p, M, interleaved != 0, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return hip_error(e, "head norm and rotation kernel launch");
    return (int)QMM4_OK;
  });
}

int64_t qmm4_sample_workspace(int64_t M, int64_t V) {
  int64_t bytes = 0;
  const int rc = guarded([&] {
    if (int bad = check_sample_shape(M, V)) return bad;
    int cus = 0;
    if (int bad = current_cus(&cus)) return bad;
    bytes = qmm4::sample_workspace(M, V, cus);
    return (int)QMM4_OK;
  });
  return rc ? rc : bytes;
}

int qmm4_sample_bf16(const void* logits, int64_t M, int64_t V, int64_t row_stride, const float* uniform,
                     const float* temperature, float temperature_value, const int32_t* top_k, int32_t top_k_value,
                     const float* top_p, float top_p_value, const float* min_p, float min_p_value, int64_t* tokens,
                     float* logprobs, void* workspace, void* hip_stream) {
  return guarded([&] {
    if (int rc = check_sample_shape(M, V)) return rc;
    if (M > 1 && row_stride < V)
      return set_error(QMM4_ERR_INVALID, "row_stride=%lld is less than V=%lld", (long long)row_stride, (long long)V);
    if (M == 0) return (int)QMM4_OK;
    if (!logits || !uniform || !tokens || !logprobs || !workspace) return set_error(QMM4_ERR_INVALID, "null pointer argument");
    if (!aligned(logits, 2) || !aligned(uniform, 4) || !aligned(temperature, 4) || !aligned(top_k, 4) ||
        !aligned(top_p, 4) || !aligned(min_p, 4) || !aligned(tokens, 8) || !aligned(logprobs, 4) || !aligned(workspace, 16))
      return set_error(QMM4_ERR_INVALID, "arrays must be aligned to their elements and workspace to 16 bytes");
    const qmm4::SampleParams p{static_cast<const uint16_t*>(logits), row_stride, uniform,
                               {temperature, temperature_value}, {top_p, top_p_value}, {min_p, min_p_value},
                               {top_k, top_k_value}, tokens, logprobs, (int)V};
    int cus = 0;
    if (int rc = current_cus(&cus)) return rc;
    hipError_t e = qmm4::launch_sample(p, M, workspace, cus, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return hip_error(e, "sampling kernel launch");
    return (int)QMM4_OK;
  });
}

}  // extern "C"
