// Divergence of rows of scores from a teacher's distribution over its top classes, and its
// gradient.
//
// With q = softmax(t / T) over a row's entries and p = softmax(x / T) over its classes, the loss is
// T^2 sum_j q_j (log q_j - log p_j) and its gradient T (p_c - sum_j q_j [c = j]).  Distil holds the
// row in registers (class_rows.cuh), so that loss and gradient take one read and one write of it;
// the gradient is for an upstream of 1, and DistilBackward makes it again for another one.  All
// classes are written as if the teacher had named none, whole vectors at a time, and its classes
// again behind them.
#include "class_rows.cuh"

namespace k2b {

// What a row's loss and gradient are multiplied with: weight, or weight / rows that count.
struct DistilScale {
  double exact;
  float rounded;
};
// Known to the host, or to the device (a kernel before this one counts the rows).
struct DistilBy {
  const DistilScale *device;
  DistilScale host;
};
constexpr size_t kDistilHead = 256;  // of the workspace; the blocks' losses follow

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

// Rows that count, of given lengths.  The kernel behind it starts meanwhile.
__global__ void __launch_bounds__(1024)
DistilCount(const void *lengths, int32_t lengths_64, int64_t outer, int64_t inner, double weight,
            DistilScale *scale) {
  LetNextStart();
  __shared__ long long counted;
  if (threadIdx.x == 0) counted = 0;
  __syncthreads();
  long long mine = 0;
  for (int64_t o = threadIdx.x; o < outer; o += 1024) {
    const int64_t n = IntAt(lengths, lengths_64, o);
    mine += n < 0 ? 0 : n > inner ? inner : n;
  }
  if (mine) atomicAdd(reinterpret_cast<unsigned long long *>(&counted), (unsigned long long)mine);
  __syncthreads();
  if (threadIdx.x == 0) {
    scale->exact = weight / (double)(counted > 1 ? counted : 1);
    scale->rounded = (float)scale->exact;
  }
}

// A teacher's row, by one warp: tokens (-1 where there is none) and shares q to shared memory.
struct TeacherRow {
  float best, mass;
  bool some, wrong;  // wrong: a class that is none, or a score that is no number
};
__device__ __forceinline__ TeacherRow ReadTeacher(const Teacher &t, int64_t r, int32_t classes,
                                                  int32_t lane, int32_t *token, float *share) {
  TeacherRow row;
  bool wrong = false;
  float best = -INFINITY;
  for (int32_t j = lane; j < t.entries; j += 32) {
    const int64_t at = r * t.entries + j, c = IntAt(t.tokens, t.tokens_64, at);
    float score = -INFINITY;
    wrong |= c < -1 || c >= classes;
    if (c >= 0 && c < classes) {
      score = TeacherScore(t, at);
      wrong |= !(score < INFINITY);
    }
    best = fmaxf(best, score);
    token[j] = c >= 0 && c < classes ? (int32_t)c : -1;
    share[j] = score;
  }
  row.wrong = __any_sync(0xffffffffu, wrong);
  row.best = WarpMaxF(best);
  row.some = row.best > -INFINITY || row.wrong;
  row.mass = 0.0f;
  return row;
}
// ... the scores there become shares.
__device__ __forceinline__ void ShareOut(const Teacher &t, TeacherRow &row, float k, int32_t lane,
                                         float *share) {
  float mass = 0.0f;
  for (int32_t j = lane; j < t.entries; j += 32) {
    const float part = row.best > -INFINITY ? Exp2((share[j] - row.best) * k) : 0.0f;
    mass += part;
    share[j] = part;
  }
  row.mass = WarpSumF(mass);
  const float by = row.best > -INFINITY ? 1.0f / row.mass : 0.0f;
  for (int32_t j = lane; j < t.entries; j += 32) share[j] *= by;
}

// The teacher's classes among [begin, end) of a row, behind the stores of all others: a class that
// comes several times has the sum of its shares, whoever writes it.
template <typename T>
__device__ __forceinline__ void WriteNamed(const Rows<T> &rows, const T *x, T *out, int32_t begin,
                                           int32_t end, int32_t entries, const int32_t *token,
                                           const float *share, int32_t tid, int32_t team,
                                           float high, float k, float inverse, float by) {
  for (int32_t j = tid; j < entries; j += team) {
    const int32_t c = token[j];
    if (c < begin || c >= end) continue;
    float hit = 0.0f;
    for (int32_t o = 0; o < entries; ++o) hit += token[o] == c ? share[o] : 0.0f;
    out[c] = FromFloat<T>((Exp2((ToFloat(x[c]) - high) * k) * inverse - hit) * by);
  }
}

// Zeros for a row.
template <typename T>
__device__ __forceinline__ void WriteZeros(T *out, int32_t classes, int32_t first, int32_t last,
                                           int32_t tid, int32_t team) {
  const RowSpan<T> zeros(out, classes);
  const float f[kPer<T>] = {};
  for (int32_t j = first + tid; j < min(last, zeros.vectors); j += team)
    Store(out, zeros, true, j, f);
}

template <int kTeam>
struct DistilShared {
  float high[kTeam / 32], sum[kTeam / 32];
  float all_high, all_sum;  // of a block, for its cluster
  int32_t some, wrong;
};

// kTeam threads per row and block with kVectors vectors each; kAgain: the row does not fit and is
// read again for each pass.  Rows of a cluster of blocks (kTeam 256) are dealt out in slices.
// loss: of the rows, or NULL and `partial` has the sum of each block's rows.
template <typename T, int kTeam, int kVectors, bool kAgain>
__global__ void __launch_bounds__(kTeam == 128 ? 128 : 256, MinBlocks(kTeam, kVectors))
Distil(Rows<T> rows, Teacher t, float4 *norm, float *loss, double *partial, T *grad,
       int64_t outer_stride, int64_t inner_stride, DistilBy by) {
  extern __shared__ int32_t all_entries[];
  __shared__ DistilShared<kTeam> all_shared[kTeam == 32 ? 8 : 1];
  __shared__ float losses[kTeam == 32 ? 8 : 1];
  LetNextStart();
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t tid = kTeam == 32 ? lane : (int32_t)threadIdx.x;
  DistilShared<kTeam> &sh = all_shared[kTeam == 32 ? warp : 0];
  int32_t *token = all_entries + (kTeam == 32 ? warp * 2 * t.entries : 0);
  float *share = reinterpret_cast<float *>(token + t.entries);
  const uint32_t cluster = kTeam == 256 ? ClusterSize() : 1,
                 rank = kTeam == 256 ? ClusterRank() : 0;
  const int32_t r = kTeam == 32 ? (int32_t)(blockIdx.x * (blockDim.x >> 5)) + warp
                                : (int32_t)(blockIdx.x / cluster);
  float row_loss = 0.0f;
  if (r < rows.count) {
    const RowPlace at = PlaceOf(rows, r);
    T *out = grad ? grad + at.o * outer_stride + at.i * inner_stride : nullptr;
    const RowSpan<T> span(rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride,
                          rows.classes);
    const int32_t slice = (span.vectors + (int32_t)cluster - 1) / (int32_t)cluster;
    const int32_t first = min(span.vectors, (int32_t)rank * slice),
                  last = min(span.vectors, first + slice);
    if (!at.counts) {
      if (out)
        WriteZeros(out, rows.classes, (int32_t)rank * slice,
                   rank + 1 == cluster ? INT32_MAX : ((int32_t)rank + 1) * slice, tid, kTeam);
    } else {
      uint4 v[kVectors];
      const auto each = [&](auto &&f) {
        if constexpr (kAgain) {
          for (int32_t tile = first; tile < last; tile += kTeam * kVectors) {
            LoadTile<kTeam, kVectors>(v, span, tile, last, tid);
#pragma unroll
            for (int i = 0; i < kVectors; ++i) f(Packed(v[i]), tile + i * kTeam + tid, i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kVectors; ++i) f(Packed(v[i]), first + i * kTeam + tid, i);
        }
      };
      if (!kAgain) LoadTile<kTeam, kVectors>(v, span, first, last, tid);
      const float k = kLog2e / t.temperature;
      TeacherRow teacher = {};
      if (kTeam == 32 || warp == 0) {
        teacher = ReadTeacher(t, r, rows.classes, lane, token, share);
        if (kTeam > 32 && lane == 0) {
          sh.some = teacher.some;
          sh.wrong = teacher.wrong;
        }
      }
      // the largest score
      float high = -INFINITY;
      each([&](uint4 &x, int32_t, int) { high = fmaxf(high, VectorMax(x, span.row)); });
      high = WarpMaxF(high);
      if (kTeam > 32) {
        if (lane == 0) sh.high[warp] = high;
        TeamSync<kTeam>();
#pragma unroll
        for (int w = 0; w < kTeam / 32; ++w) high = fmaxf(high, sh.high[w]);
      }
      float from = high == -INFINITY ? 0.0f : high;
      // the sum, of two vectors at a time
      float sums[2] = {0.0f, 0.0f};
      each([&](uint4 &x, int32_t, int i) {
        After(x, sums[i & 1]);
        float f[kPer<T>];
        Unpack(x, f, span.row);
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e) sums[i & 1] += Exp2((f[e] - from) * k);
      });
      float sum = WarpSumF(sums[0] + sums[1]);
      if (kTeam == 32 || warp == 0) ShareOut(t, teacher, k, lane, share);
      if (kTeam > 32) {
        if (lane == 0) sh.sum[warp] = sum;
        TeamSync<kTeam>();
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kTeam / 32; ++w) sum += sh.sum[w];
        teacher.some = sh.some;
        teacher.wrong = sh.wrong;
      } else {
        TeamSync<kTeam>();
      }
      if (kTeam == 256 && cluster > 1) {
        if (tid == 0) {
          sh.all_high = high;
          sh.all_sum = sum;
        }
        ClusterSync();
        for (uint32_t b = 0; b < cluster; ++b) high = fmaxf(high, ReadFrom(&sh.all_high, b));
        from = high == -INFINITY ? 0.0f : high;
        sum = 0.0f;
        for (uint32_t b = 0; b < cluster; ++b) {
          const float part = ReadFrom(&sh.all_sum, b);
          if (part == 0.0f) continue;  // (nothing but -inf)
          sum = fmaf(part, Exp2((ReadFrom(&sh.all_high, b) - from) * k), sum);
        }
        ClusterSync();  // nobody goes on while others read its memory
      }
      // the loss
      if ((kTeam == 32 || warp == 0) && rank == 0) {
        const float inverse_t = 1.0f / t.temperature, log_mass = logf(teacher.mass),
                    log_sum = logf(sum);
        float term = 0.0f;
        for (int32_t j = lane; j < t.entries; j += 32) {
          const float q = share[j];
          if (token[j] < 0 || q == 0.0f) continue;
          const float log_q =
              (TeacherScore(t, (int64_t)r * t.entries + j) - teacher.best) * inverse_t - log_mass;
          const float log_p = sum == 0.0f
                                  ? -INFINITY
                                  : (ToFloat(span.row[token[j]]) - from) * inverse_t - log_sum;
          term += q * (log_q - log_p);
        }
        term = WarpSumF(term);
        if (teacher.wrong || (teacher.some && sum != sum)) term = NAN;
        row_loss = t.temperature * t.temperature * term;
        if (norm && lane == 0) norm[r] = make_float4(from, sum, 0.0f, 0.0f);
      }
      if (out && !teacher.some) {
        WriteZeros(out, rows.classes, (int32_t)rank * slice,
                   rank + 1 == cluster ? INT32_MAX : ((int32_t)rank + 1) * slice, tid, kTeam);
      } else if (out) {
        if (by.device) WaitForPrevious();
        const float times = t.temperature * (by.device ? by.device->rounded : by.host.rounded);
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        const bool aligned = (((uintptr_t)out ^ (uintptr_t)span.row) & 15) == 0;
        const float spread = teacher.wrong ? NAN : inverse * times;
        each([&](uint4 &x, int32_t j, int) {
          if (j >= last) return;
          float f[kPer<T>];
          Unpack(x, f, span.row);
#pragma unroll
          for (int e = 0; e < kPer<T>; ++e) f[e] = Exp2((f[e] - from) * k) * spread;
          Store(out, span, aligned, j, f);
        });
        TeamSync<kTeam>();
        if (!teacher.wrong)
          WriteNamed(rows, span.row, out, max(0, span.Column(first)),
                     min(span.classes, span.Column(last)), t.entries, token, share, tid, kTeam,
                     from, k, inverse, times);
      }
    }
    if (loss && rank == 0 && tid == 0)
      loss[r] = row_loss * by.host.rounded;
  }
  if (loss) return;
  // (the next kernel reads the scale too, and waits for nothing but this one's end)
  if (by.device) WaitForPrevious();
  if (kTeam == 32) {
    if (lane == 0) losses[warp] = row_loss;
    __syncthreads();
    if (threadIdx.x == 0) {
      double sum = 0.0;
      for (uint32_t w = 0; w < blockDim.x / 32; ++w) sum += losses[w];
      partial[blockIdx.x] = sum;
    }
  } else if (rank == 0 && tid == 0) {
    partial[blockIdx.x / cluster] = row_loss;
  }
}

__global__ void __launch_bounds__(1024)
DistilLoss(const double *partial, int32_t parts, DistilBy by, float *loss) {
  __shared__ double smem[32];
  WaitForPrevious();
  double sum = 0.0;
  for (int32_t r = threadIdx.x; r < parts; r += 1024) sum += partial[r];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = smem[threadIdx.x];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (threadIdx.x == 0) *loss = (float)(sum * (by.device ? by.device->exact : by.host.exact));
  }
}

// The gradient for an upstream, of rows whose norm is known: `items` parts of rows (kTeam 256) or
// eight rows (kTeam 32), dealt out to the blocks there are.  unless_one: what is there stays where
// the upstream is 1.
template <typename T, int kTeam>
__global__ void __launch_bounds__(256, 4)
DistilBackward(Rows<T> rows, Teacher t, const float4 *norm, T *grad, int64_t outer_stride,
               int64_t inner_stride, DistilBy by, k2b200_row_grad up, int32_t unless_one,
               int64_t items, int32_t parts, int32_t part) {
  constexpr int kTile = 4;
  extern __shared__ int32_t all_entries[];
  __shared__ int32_t flags[2];
  if (unless_one && up.grad[0] == 1.0f) return;
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t tid = kTeam == 32 ? lane : (int32_t)threadIdx.x;
  int32_t *token = all_entries + (kTeam == 32 ? warp * 2 * t.entries : 0);
  float *share = reinterpret_cast<float *>(token + t.entries);
  const float k = kLog2e / t.temperature;
  const float scale = t.temperature * (by.device ? by.device->rounded : by.host.rounded);
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r64 = kTeam == 32 ? item * (blockDim.x >> 5) + warp : item / parts;
    if (r64 >= rows.count) continue;  // (a whole team)
    const int32_t r = (int32_t)r64;
    const int32_t first = kTeam == 32 ? 0 : (int32_t)(item % parts) * part;
    const RowPlace at = PlaceOf(rows, r);
    T *out = grad + at.o * outer_stride + at.i * inner_stride;
    const int32_t zeros_end = kTeam == 32 ? INT32_MAX : first + part;
    if (!at.counts) {
      WriteZeros(out, rows.classes, first, zeros_end, tid, kTeam);
      continue;
    }
    const RowSpan<T> span(rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride,
                          rows.classes);
    const int32_t last = kTeam == 32 ? span.vectors : min(span.vectors, first + part);
    uint4 v[kTile];
    LoadTile<kTeam, kTile>(v, span, first, last, tid);
    TeacherRow teacher = {};
    if (kTeam == 32 || warp == 0) {
      teacher = ReadTeacher(t, r, rows.classes, lane, token, share);
      ShareOut(t, teacher, k, lane, share);
      if (kTeam > 32 && lane == 0) {
        flags[0] = teacher.some;
        flags[1] = teacher.wrong;
      }
    }
    TeamSync<kTeam>();
    if (kTeam > 32) {
      teacher.some = flags[0];
      teacher.wrong = flags[1];
    }
    if (!teacher.some) {
      WriteZeros(out, rows.classes, first, zeros_end, tid, kTeam);
      TeamSync<kTeam>();
      continue;
    }
    const float4 n = norm[r];
    const float times = scale * up.grad[at.o * up.outer + at.i * up.inner];
    const float inverse = n.y == 0.0f ? 0.0f : 1.0f / n.y;
    const float spread = teacher.wrong ? NAN : inverse * times;
    const bool aligned = (((uintptr_t)out ^ (uintptr_t)span.row) & 15) == 0;
    for (int32_t tile = first; tile < last; tile += kTeam * kTile) {
      if (tile != first) LoadTile<kTeam, kTile>(v, span, tile, last, tid);
#pragma unroll
      for (int i = 0; i < kTile; ++i) {
        const int32_t j = tile + i * kTeam + tid;
        if (j >= last) continue;
        float f[kPer<T>];
        Unpack(Packed(v[i]), f, span.row);
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e) f[e] = Exp2((f[e] - n.x) * k) * spread;
        Store(out, span, aligned, j, f);
      }
    }
    TeamSync<kTeam>();
    if (!teacher.wrong)
      WriteNamed(rows, span.row, out, max(0, span.Column(first)),
                 min(span.classes, span.Column(last)), t.entries, token, share, tid, kTeam, n.x,
                 k, inverse, times);
    TeamSync<kTeam>();  // the next row's entries come to the same place
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

// Whether the rows that count are known to the device alone.
bool CountedThere(const k2b200_class_rows *rows, const k2b200_teacher *t) {
  return t->reduction == 2 && rows->lengths != nullptr;
}

DistilBy ByOf(const k2b200_class_rows *rows, const k2b200_teacher *t, const void *workspace) {
  DistilBy by = {};
  if (CountedThere(rows, t)) {
    by.device = static_cast<const DistilScale *>(workspace);
    return by;
  }
  const int64_t n = t->reduction == 2 ? std::max<int64_t>(1, rows->outer * rows->inner) : 1;
  by.host.exact = (double)t->weight / (double)n;
  by.host.rounded = (float)by.host.exact;
  return by;
}

template <typename T>
int32_t LaunchDistil(const k2b200_class_rows *rows, const k2b200_teacher *t, float *loss,
                     float *norm, void *grad, int64_t outer_stride, int64_t inner_stride,
                     void *workspace, cudaStream_t s) {
  const Rows<T> r = RowsOf<T>(rows);
  const Teacher teacher = {t->tokens, t->scores, t->tokens_64, t->type, t->entries,
                           t->temperature};
  const DistilBy by = ByOf(rows, t, workspace);
  double *partial = reinterpret_cast<double *>(static_cast<char *>(workspace) + kDistilHead);
  const RowPlan p = PlanRows(r);
  const int64_t groups = p.team == 32 ? CeilDiv(r.count, p.rows_per_block) : r.count;
  if (by.device) {
    DistilCount<<<1, 1024, 0, s>>>(rows->lengths, rows->lengths_64, rows->outer, rows->inner,
                                   t->weight, static_cast<DistilScale *>(workspace));
    NoteLaunch();
  }
  if (r.count > 0) {
    auto kernel = p.team == 32    ? (p.vectors == 1   ? Distil<T, 32, 1, false>
                                     : p.vectors == 2 ? Distil<T, 32, 2, false>
                                     : p.vectors == 4 ? Distil<T, 32, 4, false>
                                                      : Distil<T, 32, 8, false>)
                  : p.team == 128 ? (p.vectors == 4 ? Distil<T, 128, 4, false>
                                                    : Distil<T, 128, 8, false>)
                  : p.again       ? Distil<T, 256, 16, true>
                  : p.vectors == 4 ? Distil<T, 256, 4, false>
                  : p.vectors == 8 ? Distil<T, 256, 8, false>
                                   : Distil<T, 256, 16, false>;
    const size_t smem = (sizeof(int32_t) + sizeof(float)) * t->entries *
                        (p.team == 32 ? p.rows_per_block : 1);
    K2B_CUDA_OK(LaunchRows(kernel, groups * p.cluster, p.block, smem, p.cluster,
                           by.device != nullptr, s, r, teacher, reinterpret_cast<float4 *>(norm),
                           t->reduction == 0 ? loss : nullptr, partial, static_cast<T *>(grad),
                           outer_stride, inner_stride, by));
    NoteLaunch();
  }
  if (t->reduction != 0) {
    K2B_CUDA_OK(LaunchRows(DistilLoss, 1, 1024, 0, 1, r.count > 0, s, partial, (int32_t)groups,
                           by, loss));
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
  const Rows<T> r = RowsOf<T>(rows);
  const Teacher teacher = {t->tokens, t->scores, t->tokens_64, t->type, t->entries,
                           t->temperature};
  const RowPlan p = PlanRows(r);
  // vectors of a row, wherever it begins, in parts of a block's four per thread
  const int32_t part = 1024, parts = CeilDiv((int64_t)r.classes + kPer<T> - 1, kPer<T>) + 1;
  const int32_t row_parts = p.team == 32 ? 1 : CeilDiv(parts, part);
  const int64_t items = p.team == 32 ? CeilDiv(r.count, p.rows_per_block)
                                     : (int64_t)r.count * row_parts;
  const int64_t blocks = std::min<int64_t>(items, 8 * (int64_t)NumSms());
  auto kernel = p.team == 32 ? DistilBackward<T, 32> : DistilBackward<T, 256>;
  const int32_t threads = p.team == 32 ? p.block : 256;
  const size_t smem =
      (sizeof(int32_t) + sizeof(float)) * t->entries * (p.team == 32 ? p.rows_per_block : 1);
  kernel<<<(uint32_t)blocks, threads, smem, s>>>(
      r, teacher, reinterpret_cast<const float4 *>(norm), static_cast<T *>(grad), outer_stride,
      inner_stride, ByOf(rows, t, workspace), *up, unless_one, items, row_parts, part);
  NoteLaunch();
  K2B_CUDA_OK(cudaGetLastError());
  return kOk;
}

}  // namespace

extern "C" {

size_t k2b200_distillation_workspace_bytes(const k2b200_class_rows *rows) {
  return rows ? kDistilHead + sizeof(double) * (size_t)(rows->outer * rows->inner) : 0;
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
