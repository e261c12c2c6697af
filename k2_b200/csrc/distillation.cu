// Divergence of rows of scores from a teacher's distribution over its top classes, and its
// gradient.
//
// With q = softmax(t / T) over a row's entries and p = softmax(x / T) over its classes, the loss is
// T^2 sum_j q_j (log q_j - log p_j) and its gradient T (p_c - sum_j q_j [c = j]).  Distil hold the
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

// A teacher's row, by one warp, in two steps: tokens (-1 where there is none) and scores to shared
// memory, then the scores' shares q in their place.
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
    float score = TeacherScore(t, at);
    const bool there = c >= 0 && c < classes;
    wrong |= c < -1 || c >= classes || (there && !(score < INFINITY));
    if (!there) score = -INFINITY;
    best = fmaxf(best, score);
    token[j] = there ? (int32_t)c : -1;
    share[j] = score;
  }
  row.wrong = __any_sync(0xffffffffu, wrong);
  row.best = WarpMaxF(best);
  row.some = row.best > -INFINITY || row.wrong;
  row.mass = 0.0f;
  return row;
}
// k: log2 e / T.  Returns sum_j q_j ((t_j - best) - (x_j - high)), of which, over T, the loss is
// made (RowLoss).
template <typename T>
__device__ __forceinline__ float ShareOut(const Teacher &t, TeacherRow &row, const T *x, float k,
                                          float high, int32_t lane, const int32_t *token,
                                          float *share) {
  float mass = 0.0f, term = 0.0f;
  for (int32_t j = lane; j < t.entries; j += 32) {
    const float d = row.best > -INFINITY ? share[j] - row.best : -INFINITY, part = Exp2(d * k);
    mass += part;
    if (part != 0.0f) term += part * (d - (ToFloat(x[token[j]]) - high));
    share[j] = part;
  }
  const float2 both = WarpSum2F(mass, term);
  row.mass = both.x;
  const float by = row.best > -INFINITY ? 1.0f / row.mass : 0.0f;
  for (int32_t j = lane; j < t.entries; j += 32) share[j] *= by;
  return both.y * by;
}
// T^2 sum_j q_j (log q_j - log p_j), with log q_j = (t_j - best) / T - log mass and log p_j =
// (x_j - high) / T - log sum.
__device__ __forceinline__ float RowLoss(float temperature, const TeacherRow &row, float sum,
                                         float term) {
  if (row.wrong || (row.some && sum != sum)) return NAN;
  if (!row.some) return 0.0f;
  if (sum == 0.0f) return INFINITY;  // the student rules out every class
  return temperature * fmaf(temperature, logf(sum) - logf(row.mass), term);
}

// The teacher's classes among [begin, end) of a row, behind the stores of all others: a class that
// comes several times has the sum of its shares, whoever writes it.
template <typename T>
__device__ __forceinline__ void WriteNamed(const T *x, T *out, int32_t begin, int32_t end,
                                           int32_t entries, const int32_t *token,
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
// The same by one warp for up to 32 entries: most rows have no class twice, which one comparison of
// all lanes finds out.
template <typename T>
__device__ __forceinline__ void WriteNamedFew(const T *x, T *out, int32_t entries,
                                              const int32_t *token, const float *share,
                                              int32_t lane, float high, float k, float inverse,
                                              float by) {
  const int32_t c = lane < entries ? token[lane] : -1;
  const uint32_t same = __match_any_sync(0xffffffffu, c);
  float hit = c >= 0 ? share[lane] : 0.0f;
  if (__any_sync(0xffffffffu, c >= 0 && (same & (same - 1)) != 0)) {
    hit = 0.0f;
    for (int32_t o = 0; o < entries; ++o) hit += token[o] == c ? share[o] : 0.0f;
  }
  if (c >= 0)
    out[c] = FromFloat<T>((Exp2((ToFloat(x[c]) - high) * k) * inverse - hit) * by);
}

// p_c * by for the classes of a vector, p_c = 2^((x_c - high) * k) / sum with 1 / sum in `by`.
template <typename T>
__device__ __forceinline__ void Spread(const uint4 &v, const T *type, float high, float k,
                                       float by, float (&f)[kPer<T>]) {
  const Two minus = MakeTwo(-high, -high), times = MakeTwo(k, k), scale = MakeTwo(by, by);
  EachPair(v, type, [&](float2 x, int pair) {
    const float2 d = Split(Mul(Add(MakeTwo(x.x, x.y), minus), times));
    const float2 p = Split(Mul(MakeTwo(Exp2(d.x), Exp2(d.y)), scale));
    f[2 * pair] = p.x;
    f[2 * pair + 1] = p.y;
  });
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

// Rows of up to 4 KB: a warp takes `per_warp` of them one after the other.  Lane q knows where the
// q-th of them is and computes its loss.  loss: of the rows, or NULL and `partial` has the sum of
// each block's rows.
template <typename T, int kVectors>
__global__ void __launch_bounds__(128, kVectors >= 8 ? 6 : 8)
DistilWarps(Rows<T> rows, Teacher t, float4 *norm, float *loss, double *partial, T *grad,
            int64_t outer_stride, int64_t inner_stride, DistilBy by, int32_t per_warp) {
  extern __shared__ int32_t all_entries[];
  __shared__ double losses[4];
  LetNextStart();
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int32_t *token = all_entries + warp * 2 * t.entries;
  float *share = reinterpret_cast<float *>(token + t.entries);
  const int32_t first = (int32_t)(blockIdx.x * (blockDim.x >> 5) + warp) * per_warp,
                mine = first + lane, taken = min(per_warp, rows.count - first);
  const T *my_row = nullptr;
  T *my_out = nullptr;
  if (lane < taken) {
    const RowPlace at = PlaceOf(rows, mine);
    if (at.counts) my_row = rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride;
    if (grad) my_out = grad + at.o * outer_stride + at.i * inner_stride;
  }
  const float k = kLog2e / t.temperature;
  float my_high = 0.0f, my_sum = 0.0f, my_term = 0.0f;
  TeacherRow my_teacher = {};
  for (int32_t q = 0; q < taken; ++q) {
    const T *row = reinterpret_cast<const T *>(
        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_row), q));
    T *out = reinterpret_cast<T *>(
        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_out), q));
    if (row == nullptr) {
      if (out) WriteZeros(out, rows.classes, 0, INT32_MAX, lane, 32);
      continue;
    }
    const RowSpan<T> span(row, rows.classes);
    uint4 v[kVectors];
    LoadTile<32, kVectors>(v, span, rows, 0, span.vectors, lane);
    TeacherRow teacher = ReadTeacher(t, first + q, rows.classes, lane, token, share);
    float high = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) high = fmaxf(high, VectorMax(Packed(v[i]), row));
    high = WarpMaxF(high);
    const float from = high == -INFINITY ? 0.0f : high;
    Two sums[2] = {}, none;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      After(v[i], sums[i & 1]);
      AddVector<false>(v[i], row, from, k, sums[i & 1], none);
    }
    const float2 s = Split(Add(sums[0], sums[1]));
    const float sum = WarpSumF(s.x + s.y);
    const float term = ShareOut(t, teacher, row, k, from, lane, token, share);
    if (lane == q) {
      my_high = from;
      my_sum = sum;
      my_term = term;
      my_teacher = teacher;
    }
    if (out && !teacher.some) {
      WriteZeros(out, rows.classes, 0, INT32_MAX, lane, 32);
    } else if (out) {
      if (by.device) WaitForPrevious();
      const float times = t.temperature * (by.device ? by.device->rounded : by.host.rounded);
      const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
      const float spread = teacher.wrong ? NAN : inverse * times;
      const bool aligned = (((uintptr_t)out ^ (uintptr_t)row) & 15) == 0;
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        const int32_t j = i * 32 + lane;
        if (j >= span.vectors) continue;
        float f[kPer<T>];
        Spread(Packed(v[i]), row, from, k, spread, f);
        Store(out, span, aligned, j, f);
      }
      __syncwarp();
      if (!teacher.wrong) {
        if (t.entries <= 32)
          WriteNamedFew(row, out, t.entries, token, share, lane, from, k, inverse, times);
        else
          WriteNamed(row, out, 0, rows.classes, t.entries, token, share, lane, 32, from, k,
                     inverse, times);
      }
    }
    __syncwarp();  // the next row's entries come to the same place
  }
  float row_loss = 0.0f;
  if (lane < taken) {
    if (my_row) row_loss = RowLoss(t.temperature, my_teacher, my_sum, my_term);
    if (norm) norm[mine] = make_float4(my_high, my_sum, 0.0f, 0.0f);
    if (loss) loss[mine] = row_loss * by.host.rounded;
  }
  if (loss) return;
  // (the next kernel reads the scale too, and waits for nothing but this one's end)
  if (by.device) WaitForPrevious();
  double all = row_loss;
  for (int32_t d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
  if (lane == 0) losses[warp] = all;
  __syncthreads();
  if (threadIdx.x == 0) {
    all = 0.0;
    for (uint32_t w = 0; w < blockDim.x / 32; ++w) all += losses[w];
    partial[blockIdx.x] = all;
  }
}

template <int kTeam>
struct DistilShared {
  float high[kTeam / 32], sum[kTeam / 32];
  float all_high, all_sum;  // of a block, for its cluster
  int32_t some, wrong;
};

// A block of kTeam threads per row with kVectors vectors each; kAgain: the row does not fit and is
// read again for each pass.  Rows of a cluster of blocks (kTeam 256) are dealt out in slices.
template <typename T, int kTeam, int kVectors, bool kAgain>
__global__ void __launch_bounds__(kTeam, MinBlocks(kTeam, kVectors))
DistilBlocks(Rows<T> rows, Teacher t, float4 *norm, float *loss, double *partial, T *grad,
             int64_t outer_stride, int64_t inner_stride, DistilBy by) {
  extern __shared__ int32_t token[];
  __shared__ DistilShared<kTeam> sh;
  float *share = reinterpret_cast<float *>(token + t.entries);
  LetNextStart();
  const int32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t cluster = kTeam == 256 ? ClusterSize() : 1,
                 rank = kTeam == 256 ? ClusterRank() : 0;
  const int32_t r = (int32_t)(blockIdx.x / cluster);
  const RowPlace at = PlaceOf(rows, r);
  T *out = grad ? grad + at.o * outer_stride + at.i * inner_stride : nullptr;
  const RowSpan<T> span(rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride,
                        rows.classes);
  const int32_t slice = (span.vectors + (int32_t)cluster - 1) / (int32_t)cluster;
  const int32_t first = min(span.vectors, (int32_t)rank * slice),
                last = min(span.vectors, first + slice);
  // (a row of the gradient may lie otherwise and have a vector more)
  const int32_t zeros_first = (int32_t)rank * slice,
                zeros_last = rank + 1 == cluster ? INT32_MAX : ((int32_t)rank + 1) * slice;
  float row_loss = 0.0f;
  if (!at.counts) {
    if (out) WriteZeros(out, rows.classes, zeros_first, zeros_last, tid, kTeam);
    if (norm && rank == 0 && tid == 0) norm[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  } else {
    uint4 v[kVectors];
    const auto each = [&](auto &&f) {
      if constexpr (kAgain) {
        for (int32_t tile = first; tile < last; tile += kTeam * kVectors) {
          LoadTile<kTeam, kVectors>(v, span, rows, tile, last, tid);
#pragma unroll
          for (int i = 0; i < kVectors; ++i) f(i, tile + i * kTeam + tid);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) f(i, first + i * kTeam + tid);
      }
    };
    if (!kAgain) LoadTile<kTeam, kVectors>(v, span, rows, first, last, tid);
    const float k = kLog2e / t.temperature;
    TeacherRow teacher = {};
    if (warp == 0) {
      teacher = ReadTeacher(t, r, rows.classes, lane, token, share);
      if (lane == 0) {
        sh.some = teacher.some;
        sh.wrong = teacher.wrong;
      }
    }
    // the largest score and the sum of each warp
    float high = -INFINITY;
    each([&](int i, int32_t) { high = fmaxf(high, VectorMax(Packed(v[i]), span.row)); });
    high = WarpMaxF(high);
    float from = high == -INFINITY ? 0.0f : high;
    Two sums[2] = {}, none;
    each([&](int i, int32_t) {
      After(v[i], sums[i & 1]);
      AddVector<false>(v[i], span.row, from, k, sums[i & 1], none);
    });
    const float2 s = Split(Add(sums[0], sums[1]));
    const float warp_sum = WarpSumF(s.x + s.y);
    if (lane == 0) {
      sh.high[warp] = high;
      sh.sum[warp] = warp_sum;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kTeam / 32; ++w) high = fmaxf(high, sh.high[w]);
    from = high == -INFINITY ? 0.0f : high;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kTeam / 32; ++w)
      sum = fmaf(sh.sum[w], Exp2((sh.high[w] - from) * k), sum);
    teacher.some = sh.some;
    teacher.wrong = sh.wrong;
    if (kTeam == 256 && cluster > 1) {
      if (tid == 0) {
        sh.all_high = high;
        sh.all_sum = sum;
      }
      ClusterSync();
      for (uint32_t b = 0; b < cluster; ++b) high = fmaxf(high, ReadFrom(&sh.all_high, b));
      from = high == -INFINITY ? 0.0f : high;
      sum = 0.0f;
      for (uint32_t b = 0; b < cluster; ++b)
        sum = fmaf(ReadFrom(&sh.all_sum, b), Exp2((ReadFrom(&sh.all_high, b) - from) * k), sum);
      ClusterSync();  // nobody goes on while others read its memory
    }
    if (warp == 0) {
      const float term = ShareOut(t, teacher, span.row, k, from, lane, token, share);
      if (rank == 0) {
        row_loss = RowLoss(t.temperature, teacher, sum, term);
        if (norm && lane == 0) norm[r] = make_float4(from, sum, 0.0f, 0.0f);
      }
    }
    if (out && !teacher.some) {
      WriteZeros(out, rows.classes, zeros_first, zeros_last, tid, kTeam);
    } else if (out) {
      if (by.device) WaitForPrevious();
      const float times = t.temperature * (by.device ? by.device->rounded : by.host.rounded);
      const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
      const bool aligned = (((uintptr_t)out ^ (uintptr_t)span.row) & 15) == 0;
      const float spread = teacher.wrong ? NAN : inverse * times;
      each([&](int i, int32_t j) {
        if (j >= last) return;
        float f[kPer<T>];
        Spread(Packed(v[i]), span.row, from, k, spread, f);
        Store(out, span, aligned, j, f);
      });
      __syncthreads();
      if (!teacher.wrong)
        WriteNamed(span.row, out, max(0, span.Column(first)),
                   min(span.classes, span.Column(last)), t.entries, token, share, tid, kTeam,
                   from, k, inverse, times);
    }
  }
  if (loss) {
    if (rank == 0 && tid == 0) loss[r] = row_loss * by.host.rounded;
    return;
  }
  // (the next kernel reads the scale too, and waits for nothing but this one's end)
  if (by.device) WaitForPrevious();
  if (rank == 0 && tid == 0) partial[r] = row_loss;
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
// a row per warp (kTeam 32), dealt out to the blocks there are.  unless_one: what is there stays where
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
    LoadTile<kTeam, kTile>(v, span, rows, first, last, tid);
    TeacherRow teacher = {};
    if (kTeam == 32 || warp == 0) {
      teacher = ReadTeacher(t, r, rows.classes, lane, token, share);
      ShareOut(t, teacher, span.row, k, 0.0f, lane, token, share);
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
      if (tile != first) LoadTile<kTeam, kTile>(v, span, rows, tile, last, tid);
#pragma unroll
      for (int i = 0; i < kTile; ++i) {
        const int32_t j = tile + i * kTeam + tid;
        if (j >= last) continue;
        float f[kPer<T>];
        Spread(Packed(v[i]), span.row, n.x, k, spread, f);
        Store(out, span, aligned, j, f);
      }
    }
    TeamSync<kTeam>();
    if (!teacher.wrong)
      WriteNamed(span.row, out, max(0, span.Column(first)),
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
    const size_t entry = sizeof(int32_t) + sizeof(float);
    float4 *norms = reinterpret_cast<float4 *>(norm);
    float *row_losses = t->reduction == 0 ? loss : nullptr;
    if (p.team == 32) {
      auto kernel = p.vectors == 1   ? DistilWarps<T, 1>
                    : p.vectors == 2 ? DistilWarps<T, 2>
                    : p.vectors == 4 ? DistilWarps<T, 4>
                                     : DistilWarps<T, 8>;
      K2B_CUDA_OK(LaunchRows(kernel, groups, p.block, entry * t->entries * (p.block / 32), 1,
                             by.device != nullptr, s, r, teacher, norms, row_losses, partial,
                             static_cast<T *>(grad), outer_stride, inner_stride, by,
                             p.rows_per_warp));
    } else {
      auto kernel = p.team == 128   ? (p.vectors == 4 ? DistilBlocks<T, 128, 4, false>
                                                      : DistilBlocks<T, 128, 8, false>)
                    : p.again        ? DistilBlocks<T, 256, 16, true>
                    : p.vectors == 4 ? DistilBlocks<T, 256, 4, false>
                    : p.vectors == 8 ? DistilBlocks<T, 256, 8, false>
                                     : DistilBlocks<T, 256, 16, false>;
      K2B_CUDA_OK(LaunchRows(kernel, groups * p.cluster, p.block, entry * t->entries, p.cluster,
                             by.device != nullptr, s, r, teacher, norms, row_losses, partial,
                             static_cast<T *>(grad), outer_stride, inner_stride, by));
    }
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
  const int64_t items = p.team == 32 ? CeilDiv(r.count, p.block / 32)
                                     : (int64_t)r.count * row_parts;
  const int64_t blocks = std::min<int64_t>(items, 8 * (int64_t)NumSms());
  auto kernel = p.team == 32 ? DistilBackward<T, 32> : DistilBackward<T, 256>;
  const int32_t threads = p.team == 32 ? p.block : 256;
  const size_t smem =
      (sizeof(int32_t) + sizeof(float)) * t->entries * (p.team == 32 ? p.block / 32 : 1);
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
