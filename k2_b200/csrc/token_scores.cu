// Log-probs of given classes, entropies and top classes of rows of scores, and their gradient.
#include "class_rows.cuh"

namespace k2b {

constexpr int kTokenThreads = 128;

template <typename V>
__device__ __forceinline__ V BlockMax(V v, V *smem) {
  v = TeamMax(v);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = smem[0];
  for (int w = 1; w < kTokenThreads / 32; ++w) v = smem[w] > v ? smem[w] : v;
  __syncthreads();
  return v;
}
__device__ __forceinline__ float BlockSum(float v, float *smem) {
  v = TeamSum(v);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int w = 0; w < kTokenThreads / 32; ++w) v += smem[w];
  __syncthreads();
  return v;
}

struct TokenOut {
  const void *tokens;
  int32_t tokens_64, top_k;
  float *log_probs, *entropy, *top_log_probs;
  int32_t *top_tokens;
  float4 *norm;
};

// log p of a score.
__device__ __forceinline__ float LogProb(float x, RowNorm n) {
  return n.sum == 0.0f ? -INFINITY : (x - n.high) - logf(n.sum);
}

// A block per row, which it reads once for the largest score, once for the sums and once for each
// of its top classes.
template <typename T>
__global__ void __launch_bounds__(kTokenThreads)
TokenScores(Rows<T> rows, TokenOut out) {
  __shared__ float smem[kTokenThreads / 32];
  __shared__ uint64_t smem_key[kTokenThreads / 32];
  const int32_t r = blockIdx.x, tid = threadIdx.x, C = rows.classes;
  const RowPlace at = PlaceOf(rows, r);
  if (!at.counts) {
    if (tid == 0) {
      if (out.log_probs) out.log_probs[r] = 0.0f;
      if (out.entropy) out.entropy[r] = 0.0f;
      if (out.norm) out.norm[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (int32_t k = tid; k < out.top_k; k += kTokenThreads) {
      out.top_log_probs[(int64_t)r * out.top_k + k] = 0.0f;
      out.top_tokens[(int64_t)r * out.top_k + k] = -1;
    }
    return;
  }
  const T *x = rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride;
  RowNorm n;
  float high = -INFINITY;
  for (int32_t c = tid; c < C; c += kTokenThreads) high = fmaxf(high, ToFloat(x[c]));
  high = BlockMax(high, smem);
  n.high = high == -INFINITY ? 0.0f : high;
  float sum = 0.0f, slope = 0.0f;
  for (int32_t c = tid; c < C; c += kTokenThreads) {
    const float d = (ToFloat(x[c]) - n.high) * kLog2e, e = Exp2(d);
    sum += e;
    slope += e * fmaxf(d, -1e30f);  // 0 and not 0 * -inf where p = 0
  }
  n.sum = BlockSum(sum, smem);
  slope = BlockSum(slope, smem);
  const float h = n.sum == 0.0f ? 0.0f : logf(n.sum) - slope * kLn2 / n.sum;
  if (tid == 0) {
    if (out.entropy) out.entropy[r] = h;
    if (out.norm) out.norm[r] = make_float4(n.high, n.sum, h, 0.0f);
    if (out.log_probs) {
      const int64_t token = IntAt(out.tokens, out.tokens_64, r);
      out.log_probs[r] = token == -1              ? 0.0f
                         : token < 0 || token >= C ? NAN
                                                   : LogProb(ToFloat(x[token]), n);
    }
  }
  uint64_t last = ~0ull;
  for (int32_t k = 0; k < out.top_k; ++k) {
    uint64_t best = 0;
    for (int32_t c = tid; c < C; c += kTokenThreads) {
      const uint64_t key = KeyOf(ToFloat(x[c]), c);
      if (key < last && key > best) best = key;
    }
    last = BlockMax(best, smem_key);
    if (tid == 0) {
      const int32_t c = (int32_t)~(uint32_t)last;
      out.top_tokens[(int64_t)r * out.top_k + k] = c;
      out.top_log_probs[(int64_t)r * out.top_k + k] = LogProb(ToFloat(x[c]), n);
    }
  }
}

struct TokenGrad {
  const void *tokens;
  int32_t tokens_64, top_k;
  const int32_t *top_tokens;
  const float4 *norm;
  k2b200_row_grad log_probs, entropy, top;
  int64_t outer_stride, inner_stride;
};

__device__ __forceinline__ float GradAt(const k2b200_row_grad &g, RowPlace at, int32_t k = 0) {
  return g.grad ? g.grad[at.o * g.outer + at.i * g.inner + k * g.top] : 0.0f;
}

// dL/dx_c = -p_c (all + slope * (log p_c + h)), with `all` the upstream of every log-prob of the
// row; what a class gets as a given or a top one is added where it is.
__device__ __forceinline__ float SpreadGrad(float x, float4 n, float inverse, float log_sum,
                                            float all, float slope) {
  const float d = x - n.x, p = Exp2(d * kLog2e) * inverse;
  return p == 0.0f ? 0.0f : -p * (all + slope * (d - log_sum + n.z));
}

template <typename T>
__global__ void __launch_bounds__(kTokenThreads)
TokenScoresBackward(Rows<T> rows, TokenGrad g, T *grad) {
  __shared__ float top_grad[K2B200_MAX_TOP];
  const int32_t r = blockIdx.x, tid = threadIdx.x, C = rows.classes;
  const RowPlace at = PlaceOf(rows, r);
  T *out = grad + at.o * g.outer_stride + at.i * g.inner_stride;
  if (!at.counts) {
    for (int32_t c = tid; c < C; c += kTokenThreads) out[c] = FromFloat<T>(0.0f);
    return;
  }
  const T *x = rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride;
  const int32_t *top = g.top_tokens + (int64_t)r * g.top_k;
  for (int32_t k = tid; k < g.top_k; k += kTokenThreads) top_grad[k] = GradAt(g.top, at, k);
  __syncthreads();
  const float4 n = g.norm[r];
  const int64_t token = g.log_probs.grad ? IntAt(g.tokens, g.tokens_64, r) : -1;
  const float token_grad = token == -1              ? 0.0f
                           : token < 0 || token >= C ? NAN
                                                     : GradAt(g.log_probs, at);
  float all = token_grad;
  for (int32_t k = 0; k < g.top_k; ++k) all += top_grad[k];
  const float slope = GradAt(g.entropy, at);
  const float inverse = n.y == 0.0f ? 0.0f : 1.0f / n.y, log_sum = logf(n.y);
  for (int32_t c = tid; c < C; c += kTokenThreads) {
    float v = SpreadGrad(ToFloat(x[c]), n, inverse, log_sum, all, slope);
    if (c == token) v += token_grad;
    for (int32_t k = 0; k < g.top_k; ++k)
      if (c == top[k]) v += top_grad[k];
    out[c] = FromFloat<T>(v);
  }
}

}  // namespace k2b

using namespace k2b;

namespace {

template <typename T>
int32_t LaunchTokenScores(const k2b200_class_rows *rows, const TokenOut &out, cudaStream_t s) {
  TokenScores<T><<<(uint32_t)(rows->outer * rows->inner), kTokenThreads, 0, s>>>(RowsOf<T>(rows),
                                                                                 out);
  NoteLaunch();
  K2B_CUDA_OK(cudaGetLastError());
  return kOk;
}

template <typename T>
int32_t LaunchTokenBackward(const k2b200_class_rows *rows, const TokenGrad &g, void *grad,
                            cudaStream_t s) {
  TokenScoresBackward<T><<<(uint32_t)(rows->outer * rows->inner), kTokenThreads, 0, s>>>(
      RowsOf<T>(rows), g, static_cast<T *>(grad));
  NoteLaunch();
  K2B_CUDA_OK(cudaGetLastError());
  return kOk;
}

}  // namespace

extern "C" {

int32_t k2b200_token_scores(const k2b200_class_rows *rows, const void *tokens, int32_t tokens_64,
                            int32_t top_k, float *log_probs, float *entropy,
                            float *top_log_probs, int32_t *top_tokens, float *norm,
                            void *stream) {
  K2B_FORWARD(CheckRows(rows));
  K2B_REQUIRE(top_k >= 0 && top_k <= K2B200_MAX_TOP && top_k <= rows->num_classes,
              "top_k is %d: 0 to %d, and at most the %d classes", top_k, K2B200_MAX_TOP,
              rows->num_classes);
  if (rows->outer * rows->inner == 0) return kOk;
  K2B_REQUIRE((log_probs == nullptr) == (tokens == nullptr),
              "tokens and log_probs are given together");
  K2B_REQUIRE(top_k == 0 || (top_log_probs && top_tokens), "NULL pointer");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const TokenOut out = {tokens,        tokens_64,  top_k, log_probs, entropy,
                        top_log_probs, top_tokens, reinterpret_cast<float4 *>(norm)};
  return rows->type == K2B200_F32   ? LaunchTokenScores<float>(rows, out, s)
         : rows->type == K2B200_F16 ? LaunchTokenScores<__half>(rows, out, s)
                                    : LaunchTokenScores<__nv_bfloat16>(rows, out, s);
}

int32_t k2b200_token_scores_backward(const k2b200_class_rows *rows, const void *tokens,
                                     int32_t tokens_64, int32_t top_k, const int32_t *top_tokens,
                                     const float *norm, const k2b200_row_grad *log_probs_grad,
                                     const k2b200_row_grad *entropy_grad,
                                     const k2b200_row_grad *top_log_probs_grad,
                                     void *grad_scores, int64_t grad_outer_stride,
                                     int64_t grad_inner_stride, void *stream) {
  K2B_FORWARD(CheckRows(rows));
  K2B_REQUIRE(log_probs_grad && entropy_grad && top_log_probs_grad, "NULL pointer");
  K2B_REQUIRE(top_k >= 0 && top_k <= K2B200_MAX_TOP && top_k <= rows->num_classes,
              "top_k is %d: 0 to %d, and at most the %d classes", top_k, K2B200_MAX_TOP,
              rows->num_classes);
  if (rows->outer * rows->inner == 0) return kOk;
  K2B_REQUIRE(norm && grad_scores, "NULL pointer");
  K2B_REQUIRE(!log_probs_grad->grad || tokens, "a gradient of log-probs without tokens");
  K2B_REQUIRE(!top_log_probs_grad->grad || (top_k > 0 && top_tokens),
              "a gradient of top log-probs without top classes");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const TokenGrad g = {tokens,
                       tokens_64,
                       top_log_probs_grad->grad ? top_k : 0,
                       top_tokens,
                       reinterpret_cast<const float4 *>(norm),
                       *log_probs_grad,
                       *entropy_grad,
                       *top_log_probs_grad,
                       grad_outer_stride,
                       grad_inner_stride};
  return rows->type == K2B200_F32   ? LaunchTokenBackward<float>(rows, g, grad_scores, s)
         : rows->type == K2B200_F16 ? LaunchTokenBackward<__half>(rows, g, grad_scores, s)
                                    : LaunchTokenBackward<__nv_bfloat16>(rows, g, grad_scores, s);
}

}  // extern "C"
