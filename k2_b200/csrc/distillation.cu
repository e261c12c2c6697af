// Divergence of rows of scores from a teacher's distribution over its top classes, and its
// gradient.
#include "class_rows.cuh"

namespace k2b {

constexpr int kDistilThreads = 128;

// The workspace: what the row's gradient is multiplied with (weight, or weight / rows that count),
// and the rows' losses.
struct DistilScale {
  double exact;
  float rounded;
};
constexpr size_t kDistilHead = 256;

struct Teacher {
  const void *tokens, *scores;
  int32_t tokens_64, type, entries;
  float temperature;
};

__device__ __forceinline__ float TeacherScore(const Teacher &t, int64_t k) {
  return t.type == K2B200_F32   ? static_cast<const float *>(t.scores)[k]
         : t.type == K2B200_F16 ? __half2float(static_cast<const __half *>(t.scores)[k])
                                : __bfloat162float(static_cast<const __nv_bfloat16 *>(t.scores)[k]);
}

__global__ void __launch_bounds__(1024)
DistilScaleOf(const void *lengths, int32_t lengths_64, int64_t outer, int64_t inner, double weight,
              int32_t mean, DistilScale *scale) {
  __shared__ long long counted;
  if (threadIdx.x == 0) counted = 0;
  __syncthreads();
  long long mine = 0;
  if (mean && lengths)
    for (int64_t o = threadIdx.x; o < outer; o += 1024) {
      const int64_t n = IntAt(lengths, lengths_64, o);
      mine += n < 0 ? 0 : n > inner ? inner : n;
    }
  atomicAdd(reinterpret_cast<unsigned long long *>(&counted), (unsigned long long)mine);
  __syncthreads();
  if (threadIdx.x == 0) {
    const long long n = !mean ? 1 : lengths ? counted : outer * inner;
    scale->exact = weight / (double)(n > 1 ? n : 1);
    scale->rounded = (float)scale->exact;
  }
}

__device__ __forceinline__ float DistilMax(float v, float *smem) {
  v = TeamMax(v);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = smem[0];
  for (int w = 1; w < kDistilThreads / 32; ++w) v = fmaxf(v, smem[w]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float DistilSum(float v, float *smem) {
  v = TeamSum(v);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int w = 0; w < kDistilThreads / 32; ++w) v += smem[w];
  __syncthreads();
  return v;
}

// A block per row: the student's largest score and sum, the teacher's distribution, the loss, and
// the gradient T * (p - q) * scale.  kBackward: the norm is known, the upstream multiplies, and no
// loss is written.
template <typename T, bool kBackward>
__global__ void __launch_bounds__(kDistilThreads)
Distil(Rows<T> rows, Teacher t, float4 *norm, float *row_loss, int32_t scaled_loss, T *grad,
       int64_t outer_stride, int64_t inner_stride, const DistilScale *scale, k2b200_row_grad up,
       int32_t unless_one) {
  __shared__ float smem[kDistilThreads / 32];
  __shared__ int32_t token[K2B200_MAX_TOP];
  __shared__ float share[K2B200_MAX_TOP];
  const int32_t r = blockIdx.x, tid = threadIdx.x, C = rows.classes;
  if (kBackward && unless_one && up.grad[0] == 1.0f) return;
  const RowPlace at = PlaceOf(rows, r);
  T *out = grad ? grad + at.o * outer_stride + at.i * inner_stride : nullptr;
  if (!at.counts) {
    if (out)
      for (int32_t c = tid; c < C; c += kDistilThreads) out[c] = FromFloat<T>(0.0f);
    if (tid == 0 && row_loss) row_loss[r] = 0.0f;
    return;
  }
  const T *x = rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride;
  const float inverse_t = 1.0f / t.temperature, k = kLog2e / t.temperature;
  // the teacher
  bool bad = false, some = false;
  float mine = -INFINITY;
  int32_t my_token = -1;
  if (tid < t.entries) {
    const int64_t j = (int64_t)r * t.entries + tid, c = IntAt(t.tokens, t.tokens_64, j);
    bad = c < -1 || c >= C;
    if (c >= 0 && c < C) {
      my_token = (int32_t)c;
      mine = TeacherScore(t, j);
    }
  }
  const bool nan = __syncthreads_or(bad || mine != mine || mine == INFINITY);
  const float best = DistilMax(mine, smem);
  some = best > -INFINITY;
  const float part = some && mine > -INFINITY ? Exp2((mine - best) * k) : 0.0f;
  const float mass = DistilSum(part, smem);
  const float q = nan ? NAN : some ? part / mass : 0.0f;
  if (tid < t.entries) {
    token[tid] = my_token;
    share[tid] = my_token >= 0 ? q : 0.0f;
  }
  __syncthreads();
  // the student
  RowNorm n;
  if (kBackward) {
    const float4 v = norm[r];
    n.high = v.x;
    n.sum = v.y;
  } else {
    float high = -INFINITY;
    for (int32_t c = tid; c < C; c += kDistilThreads) high = fmaxf(high, ToFloat(x[c]));
    high = DistilMax(high, smem);
    n.high = high == -INFINITY ? 0.0f : high;
    float sum = 0.0f;
    for (int32_t c = tid; c < C; c += kDistilThreads) sum += Exp2((ToFloat(x[c]) - n.high) * k);
    n.sum = DistilSum(sum, smem);
    float term = 0.0f;
    if (my_token >= 0 && (q > 0.0f || q != q)) {
      const float log_q = (mine - best) * inverse_t - logf(mass);
      const float log_p = n.sum == 0.0f ? -INFINITY
                                        : (ToFloat(x[my_token]) - n.high) * inverse_t - logf(n.sum);
      term = q * (log_q - log_p);
    }
    term = DistilSum(term, smem);
    // a student row of NaN is NaN even where the teacher says nothing of it
    if (nan || (some && n.sum != n.sum)) term = NAN;
    if (tid == 0) {
      const float loss = t.temperature * t.temperature * term;
      row_loss[r] = scaled_loss ? loss * scale->rounded : loss;
      if (norm) norm[r] = make_float4(n.high, n.sum, 0.0f, 0.0f);
    }
  }
  if (!out) return;
  const float by = t.temperature * scale->rounded *
                   (kBackward ? up.grad[at.o * up.outer + at.i * up.inner] : 1.0f);
  const float inverse = n.sum == 0.0f ? 0.0f : 1.0f / n.sum;
  for (int32_t c = tid; c < C; c += kDistilThreads) {
    float v = !some ? 0.0f : Exp2((ToFloat(x[c]) - n.high) * k) * inverse;
    if (nan) v = NAN;
    for (int32_t j = 0; j < t.entries; ++j)
      if (token[j] == c) v -= share[j];
    out[c] = FromFloat<T>(v * by);
  }
}

__global__ void __launch_bounds__(1024)
DistilLoss(const float *row_loss, int32_t rows, const DistilScale *scale, float *loss) {
  __shared__ double smem[32];
  double sum = 0.0;
  for (int32_t r = threadIdx.x; r < rows; r += 1024) sum += row_loss[r];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < 32; ++w) sum += smem[w];
    *loss = (float)(sum * scale->exact);
  }
}

}  // namespace k2b

using namespace k2b;

namespace {

int32_t CheckTeacher(const k2b200_teacher *t, const k2b200_class_rows *rows) {
  K2B_REQUIRE(t != nullptr, "NULL pointer");
  K2B_REQUIRE(t->type >= K2B200_F32 && t->type <= K2B200_BF16, "unknown type %d", t->type);
  K2B_REQUIRE(t->entries >= 1 && t->entries <= K2B200_MAX_TOP,
              "a teacher of %d classes per row: 1 to %d", t->entries, K2B200_MAX_TOP);
  K2B_REQUIRE(t->temperature > 0.0f && t->temperature <= 1e18f, "the temperature is %g",
              t->temperature);
  K2B_REQUIRE(t->reduction >= 0 && t->reduction <= 2, "unknown reduction %d", t->reduction);
  K2B_REQUIRE((t->tokens && t->scores) || rows->outer * rows->inner == 0, "NULL pointer");
  return kOk;
}

template <typename T>
int32_t LaunchDistil(const k2b200_class_rows *rows, const k2b200_teacher *t, float *loss,
                     float *norm, void *grad, int64_t outer_stride, int64_t inner_stride,
                     void *workspace, cudaStream_t s) {
  const int32_t num = (int32_t)(rows->outer * rows->inner);
  DistilScale *scale = static_cast<DistilScale *>(workspace);
  float *row_loss = reinterpret_cast<float *>(static_cast<char *>(workspace) + kDistilHead);
  const Teacher teacher = {t->tokens, t->scores, t->tokens_64, t->type, t->entries,
                           t->temperature};
  DistilScaleOf<<<1, 1024, 0, s>>>(rows->lengths, rows->lengths_64, rows->outer, rows->inner,
                                   t->weight, t->reduction == 2, scale);
  NoteLaunch();
  if (num > 0) {
    Distil<T, false><<<num, kDistilThreads, 0, s>>>(
        RowsOf<T>(rows), teacher, reinterpret_cast<float4 *>(norm),
        t->reduction == 0 ? loss : row_loss, t->reduction == 0, static_cast<T *>(grad),
        outer_stride, inner_stride, scale, k2b200_row_grad{}, 0);
    NoteLaunch();
  }
  if (t->reduction != 0) {
    DistilLoss<<<1, 1024, 0, s>>>(row_loss, num, scale, loss);
    NoteLaunch();
  }
  K2B_CUDA_OK(cudaGetLastError());
  return kOk;
}

template <typename T>
int32_t LaunchDistilBackward(const k2b200_class_rows *rows, const k2b200_teacher *t,
                             const float *norm, const k2b200_row_grad *up, int32_t unless_one,
                             void *grad, int64_t outer_stride, int64_t inner_stride,
                             const void *workspace, cudaStream_t s) {
  const Teacher teacher = {t->tokens, t->scores, t->tokens_64, t->type, t->entries,
                           t->temperature};
  Distil<T, true><<<(uint32_t)(rows->outer * rows->inner), kDistilThreads, 0, s>>>(
      RowsOf<T>(rows), teacher, reinterpret_cast<float4 *>(const_cast<float *>(norm)), nullptr, 0,
      static_cast<T *>(grad), outer_stride, inner_stride,
      static_cast<const DistilScale *>(workspace), *up, unless_one);
  NoteLaunch();
  K2B_CUDA_OK(cudaGetLastError());
  return kOk;
}

}  // namespace

extern "C" {

size_t k2b200_distillation_workspace_bytes(const k2b200_class_rows *rows) {
  return rows ? kDistilHead + sizeof(float) * (size_t)(rows->outer * rows->inner) : 0;
}

int32_t k2b200_distillation(const k2b200_class_rows *rows, const k2b200_teacher *teacher,
                            float *loss, float *norm, void *grad_scores,
                            int64_t grad_outer_stride, int64_t grad_inner_stride,
                            void *workspace, size_t workspace_bytes, void *stream) {
  K2B_FORWARD(CheckRows(rows));
  K2B_FORWARD(CheckTeacher(teacher, rows));
  K2B_REQUIRE(!grad_scores || teacher->reduction != 0,
              "the gradient of row losses needs their upstream");
  K2B_REQUIRE(workspace, "NULL pointer");
  K2B_REQUIRE(loss || (teacher->reduction == 0 && rows->outer * rows->inner == 0),
              "NULL pointer");
  if (workspace_bytes < k2b200_distillation_workspace_bytes(rows)) {
    SetError("workspace of %zu bytes, %zu are needed", workspace_bytes,
             k2b200_distillation_workspace_bytes(rows));
    return kWorkspaceTooSmall;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto launch = rows->type == K2B200_F32   ? LaunchDistil<float>
                : rows->type == K2B200_F16 ? LaunchDistil<__half>
                                           : LaunchDistil<__nv_bfloat16>;
  return launch(rows, teacher, loss, norm, grad_scores, grad_outer_stride, grad_inner_stride,
                workspace, s);
}

int32_t k2b200_distillation_backward(const k2b200_class_rows *rows, const k2b200_teacher *teacher,
                                     const float *norm, const k2b200_row_grad *upstream,
                                     int32_t unless_one, void *grad_scores,
                                     int64_t grad_outer_stride, int64_t grad_inner_stride,
                                     const void *workspace, size_t workspace_bytes,
                                     void *stream) {
  K2B_FORWARD(CheckRows(rows));
  K2B_FORWARD(CheckTeacher(teacher, rows));
  if (rows->outer * rows->inner == 0) return kOk;
  K2B_REQUIRE(norm && upstream && upstream->grad && grad_scores && workspace, "NULL pointer");
  if (workspace_bytes < kDistilHead) {
    SetError("workspace of %zu bytes, %zu are needed", workspace_bytes, kDistilHead);
    return kWorkspaceTooSmall;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto launch = rows->type == K2B200_F32   ? LaunchDistilBackward<float>
                : rows->type == K2B200_F16 ? LaunchDistilBackward<__half>
                                           : LaunchDistilBackward<__nv_bfloat16>;
  return launch(rows, teacher, norm, upstream, unless_one, grad_scores, grad_outer_stride,
                grad_inner_stride, workspace, s);
}

}  // extern "C"
