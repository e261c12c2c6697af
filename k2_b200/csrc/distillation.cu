// Divergence of rows of scores from a teacher's distribution over its top classes, and its
// gradient.
//
// With q = softmax(t / T) over a row's entries and p = softmax(x / T) over its classes, the loss is
// T^2 sum_j q_j (log q_j - log p_j) and its gradient T (p_c - sum_j q_j [c = j]).  DistilWarps (rows
// up to 4 KB) and DistilRing have the row on the chip, so that loss and gradient take one read and one
// write of it; the gradient is for an upstream of 1, and DistilBackward makes it again for another
// one.  All classes are written as if the teacher had named none, whole vectors at a time, and its
// classes again behind them.
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
__global__ void __launch_bounds__(256)
DistilCount(const void *lengths, int32_t lengths_64, int64_t outer, int64_t inner, double weight,
            DistilScale *scale) {
  LetNextStart();
  __shared__ long long counted[8];
  long long mine = 0;
  for (int64_t o = threadIdx.x; o < outer; o += 256) {
    const int64_t n = IntAt(lengths, lengths_64, o);
    mine += n < 0 ? 0 : n > inner ? inner : n;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  if ((threadIdx.x & 31) == 0) counted[threadIdx.x >> 5] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) mine += counted[w];
    scale->exact = weight / (double)(mine > 1 ? mine : 1);
    scale->rounded = (float)scale->exact;
  }
}

// The first 32 * kAhead entries of a teacher's row, read by a warp ahead of time; and the student's
// scores of their classes.
template <int kAhead>
struct TeacherAhead {
  int32_t token[kAhead];
  float score[kAhead], x[kAhead];
};
// -1 for none, kNoClass for a number that is no class of 2^30.
constexpr int32_t kNoClass = INT32_MAX;
__device__ __forceinline__ int32_t EntryToken(const Teacher &t, int64_t at) {
  const int64_t c = IntAt(t.tokens, t.tokens_64, at);
  return c < -1 || c > kMaxClasses ? kNoClass : (int32_t)c;
}
template <int kAhead>
__device__ __forceinline__ void ReadAhead(TeacherAhead<kAhead> &e, const Teacher &t, int64_t r,
                                          int32_t lane) {
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int32_t j = lane + 32 * i;
    if (j < t.entries) {
      e.token[i] = EntryToken(t, r * t.entries + j);
      e.score[i] = TeacherScore(t, r * t.entries + j);
    }
  }
}

template <int kAhead, typename T>
__device__ __forceinline__ void ReadScores(TeacherAhead<kAhead> &e, const Teacher &t,
                                           int32_t classes, const T *x, int32_t lane) {
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (lane + 32 * i < t.entries && e.token[i] >= 0 && e.token[i] < classes)
      e.x[i] = ToFloat(x[e.token[i]]);
}

// A row of the teacher as a warp has it in shared memory: classes (-1 where there is none), scores
// that become shares q, and the student's scores of the classes.  Each lane has its entries to
// itself until they are shared out.
struct TeacherRow {
  int32_t *token;
  float *share, *x;
  float best, mass;
  bool some, wrong;  // wrong: a class that is none, or a score that is no number
};
constexpr int32_t kEntryBytes = 12;
__device__ __forceinline__ TeacherRow TeacherAt(void *memory, int32_t entries) {
  TeacherRow row;
  row.token = static_cast<int32_t *>(memory);
  row.share = reinterpret_cast<float *>(row.token + entries);
  row.x = row.share + entries;
  row.best = row.mass = 0.0f;
  row.some = row.wrong = false;
  return row;
}
// x: the student's row, for entries that were not read ahead.
template <int kAhead, typename T>
__device__ __forceinline__ void ReadTeacher(TeacherRow &row, const TeacherAhead<kAhead> &ahead,
                                            const Teacher &t, int64_t r, int32_t classes,
                                            const T *x, int32_t lane) {
  bool wrong = false;
  float best = -INFINITY;
  const auto entry = [&](int32_t j, int32_t c, float score, float of_student) {
    const bool there = c >= 0 && c < classes;
    wrong |= c >= classes || (there && !(score < INFINITY));
    if (!there) score = -INFINITY;
    best = fmaxf(best, score);
    row.token[j] = there ? c : -1;
    row.share[j] = score;
    row.x[j] = of_student;
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (lane + 32 * i < t.entries)
      entry(lane + 32 * i, ahead.token[i], ahead.score[i], ahead.x[i]);
  for (int32_t j = lane + 32 * kAhead; j < t.entries; j += 32) {
    const int32_t c = EntryToken(t, r * t.entries + j);
    entry(j, c, TeacherScore(t, r * t.entries + j),
          c >= 0 && c < classes ? ToFloat(x[c]) : 0.0f);
  }
  row.wrong = __any_sync(0xffffffffu, wrong);
  row.best = WarpMaxF(best);
  row.some = row.best > -INFINITY || row.wrong;
}
// The scores become shares.  k: log2 e / T.  Returns sum_j q_j ((t_j - best) - (x_j - high)), of
// which, over T, the loss is made (RowLoss).
__device__ __forceinline__ float ShareOut(TeacherRow &row, const Teacher &t, float k, float high,
                                          int32_t lane) {
  float mass = 0.0f, term = 0.0f;
  for (int32_t j = lane; j < t.entries; j += 32) {
    const float d = row.best > -INFINITY ? row.share[j] - row.best : -INFINITY, part = Exp2(d * k);
    mass += part;
    if (part != 0.0f) term = fmaf(part, d - (row.x[j] - high), term);
    row.share[j] = part;
  }
  const float2 both = WarpSum2F(mass, term);
  row.mass = both.x;
  const float by = row.best > -INFINITY ? 1.0f / row.mass : 0.0f;
  for (int32_t j = lane; j < t.entries; j += 32) row.share[j] *= by;
  return both.y * by;
}
// T^2 sum_j q_j (log q_j - log p_j), with log q_j = (t_j - best) / T - log mass and log p_j =
// (x_j - high) / T - log sum.  In 32 bits: each term is a difference of 32-bit numbers already, and
// there are 128 at most.  Rows are added up in 64.
__device__ __forceinline__ float RowLoss(float temperature, bool some, bool wrong, float mass,
                                         float sum, float term) {
  if (wrong || (some && sum != sum)) return NAN;
  if (!some) return 0.0f;
  if (sum == 0.0f) return INFINITY;  // the student rules out every class
  return temperature * fmaf(temperature, logf(sum) - logf(mass), term);
}

// The teacher's classes among [begin, end) of a row, behind the stores of all others.  A class that
// comes several times has the sum of its shares, whoever writes it; of up to 32 entries one warp
// finds out by a comparison of all lanes whether there is any.  More are compared one by one, which
// costs their square: 64000 rows of 500 bf16 classes take 60 us with 32 entries, 95 with 33, 120 with
// 64 and 321 with 128, cold.
template <typename T>
__device__ __forceinline__ void WriteNamed(const TeacherRow &row, const Teacher &t, T *out,
                                           int32_t begin, int32_t end, int32_t tid, int32_t team,
                                           float high, float k, float inverse, float by) {
  bool alone = false;
  if (t.entries <= 32) {
    if (tid >= 32) return;
    const int32_t c = tid < t.entries ? row.token[tid] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, c);
    alone = !__any_sync(0xffffffffu, c >= 0 && (same & (same - 1)) != 0);
  }
  for (int32_t j = tid; j < t.entries; j += team) {
    const int32_t c = row.token[j];
    if (c < begin || c >= end) continue;
    float hit = 0.0f;
    if (alone)
      hit = row.share[j];
    else
      for (int32_t o = 0; o < t.entries; ++o) hit += row.token[o] == c ? row.share[o] : 0.0f;
    out[c] = FromFloat<T>((Exp2((row.x[j] - high) * k) * inverse - hit) * by);
  }
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

// The gradient of a thread's vectors.
template <int kTeam, int kVectors, typename T>
__device__ __forceinline__ void WriteGrad(uint4 (&v)[kVectors], const RowPart<T> &part, T *out,
                                          float high, float k, float by) {
  const bool aligned = (((uintptr_t)out ^ (uintptr_t)part.span.row) & 15) == 0;
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    if (i >= part.mine) continue;
    float f[kPer<T>];
    Spread(Packed(v[i]), part.span.row, high, k, by, f);
    Store(out, part.span, aligned, part.first + i * kTeam, f);
  }
}

// The same for vectors in shared memory: whole ones in a loop of few instructions, the row's ends
// by themselves.
template <int kTeam, typename T>
__device__ __forceinline__ void WriteGradRow(const uint4 *slot, const RowPart<T> &part, T *out,
                                             float high, float k, float by) {
  const RowSpan<T> &span = part.span;
  const bool aligned = (((uintptr_t)out ^ (uintptr_t)span.row) & 15) == 0;
  int32_t begin = 0, end = part.mine;
  if (aligned) {
    if (part.mine > 0 && !span.Whole(span.Column(part.first))) begin = 1;
    if (end > begin && !span.Whole(span.Column(part.first + (end - 1) * kTeam))) --end;
    uint4 *to = reinterpret_cast<uint4 *>(out - span.shift) + part.first;
#pragma unroll 2
    for (int32_t i = begin; i < end; ++i) {
      float f[kPer<T>];
      Spread(slot[i * kTeam], span.row, high, k, by, f);
      to[i * kTeam] = Pack(f, out);
    }
  }
  // (what is left: one or two vectors, or all)
#pragma unroll 1
  for (int32_t i = 0; i < part.mine; ++i) {
    if (aligned && i >= begin && i < end) i = end;
    if (i >= part.mine) break;
    float f[kPer<T>];
    Spread(slot[i * kTeam], span.row, high, k, by, f);
    Store(out, span, false, part.first + i * kTeam, f);
  }
}

// Short rows: each warp is a team.  It takes 32 rows at a time, a whole grid of warps apart; lane q
// knows where the q-th of them is and computes its loss.  loss: of the rows, or NULL and `partial`
// has the sum of each block's rows.  Bound by instructions (690 a row, 72% of the issue slots): 64 x
// 1000 rows of 500 bf16 classes with 16 entries, a fifth beyond their lengths, 48 us, 2.5 TB/s.
template <typename T, int kVectors>
__global__ void __launch_bounds__(128, ResidentBlocks(kVectors))
DistilWarps(Rows<T> rows, Teacher t, float4 *norm, float *loss, double *partial, T *grad,
            int64_t outer_stride, int64_t inner_stride, DistilBy by) {
  extern __shared__ uint4 shared[];
  __shared__ double losses[4];
  LetNextStart();
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  uint4 *slot = shared + warp * 32 * kVectors + lane;
  TeacherRow teacher = TeacherAt(reinterpret_cast<char *>(shared + warps * 32 * kVectors) +
                                     warp * t.entries * kEntryBytes,
                                 t.entries);
  const int32_t apart = (int32_t)gridDim.x * warps;
  const float k = kLog2e / t.temperature;
  bool waited = by.device == nullptr;
  float scale = by.host.rounded;
  double all_losses = 0.0;
  for (int32_t base = (int32_t)blockIdx.x * warps + warp; base < rows.count; base += 32 * apart) {
    const int32_t mine = base + lane * apart,
                  taken = min(32, (rows.count - base + apart - 1) / apart);
    const T *my_row = nullptr;
    T *my_out = nullptr;
    if (lane < taken) {
      const RowPlace at = PlaceOf(rows, mine);
      if (at.counts) my_row = rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride;
      if (grad) my_out = grad + at.o * outer_stride + at.i * inner_stride;
    }
    const auto row_of = [&](int32_t q) {
      return reinterpret_cast<const T *>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_row), q & 31));
    };
    const T *next = row_of(0);
    TeacherAhead<1> ahead;
    if (next != nullptr) {
      const RowSpan<T> span(next, rows.classes);
      SendFor<32, kVectors>(slot, RowPart<T>(span, 0, span.vectors, lane, 32), rows);
      ReadAhead(ahead, t, base, lane);
    }
    float my_high = 0.0f, my_sum = 0.0f, my_term = 0.0f, my_mass = 0.0f;
    bool my_some = false, my_wrong = false;
    for (int32_t q = 0; q < taken; ++q) {
      const T *row = next;
      T *out = reinterpret_cast<T *>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_out), q));
      const RowSpan<T> span(row, rows.classes);
      const RowPart<T> part(span, 0, span.vectors, lane, 32);
      uint4 v[kVectors];
      if (row != nullptr) {
        WaitForAll();
        CutEnds<32>(slot, part);
        Take<32, kVectors>(v, slot, part);
        __syncwarp();  // (and the entries of the row before have been read)
        // the scores of the teacher's classes, while the row is there
        const T *here = reinterpret_cast<const T *>(slot - lane) + span.shift;
        ReadScores(ahead, t, rows.classes, here, lane);
        ReadTeacher(teacher, ahead, t, base + q * apart, rows.classes, here, lane);
        __syncwarp();
      }
      next = row_of(q + 1);
      if (q + 1 < taken && next != nullptr) {
        const RowSpan<T> coming(next, rows.classes);
        SendFor<32, kVectors>(slot, RowPart<T>(coming, 0, coming.vectors, lane, 32), rows);
        ReadAhead(ahead, t, base + (q + 1) * apart, lane);
      }
      if (row == nullptr) {
        if (out) WriteZeros(out, rows.classes, 0, INT32_MAX, lane, 32);
        continue;
      }
      const float2 half = Highest(v, row);
      const float high = WarpMaxF(fmaxf(half.x, half.y)), from = high == -INFINITY ? 0.0f : high;
      const float sum = WarpSumF(SumUp<false>(v, row, from, k).x);
      const float term = ShareOut(teacher, t, k, from, lane);
      if (lane == q) {
        my_high = from;
        my_sum = sum;
        my_term = term;
        my_mass = teacher.mass;
        my_some = teacher.some;
        my_wrong = teacher.wrong;
      }
      if (out && !teacher.some) {
        WriteZeros(out, rows.classes, 0, INT32_MAX, lane, 32);
      } else if (out) {
        if (!waited) {
          WaitForPrevious();
          waited = true;
          scale = by.device->rounded;
        }
        const float times = t.temperature * scale, inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        WriteGrad<32>(v, part, out, from, k, teacher.wrong ? NAN : inverse * times);
        __syncwarp();
        if (!teacher.wrong)
          WriteNamed(teacher, t, out, 0, rows.classes, lane, 32, from, k, inverse, times);
      }
    }
    float row_loss = 0.0f;
    if (lane < taken) {
      if (my_row) row_loss = RowLoss(t.temperature, my_some, my_wrong, my_mass, my_sum, my_term);
      if (norm) norm[mine] = make_float4(my_high, my_sum, 0.0f, 0.0f);
      if (loss) loss[mine] = row_loss * by.host.rounded;
    }
    all_losses += row_loss;
  }
  if (loss) return;
  // (the next kernel reads the scale too, and waits for nothing but this one's end)
  if (!waited) WaitForPrevious();
  for (int32_t d = 16; d > 0; d >>= 1) all_losses += __shfl_xor_sync(0xffffffffu, all_losses, d);
  if (lane == 0) losses[warp] = all_losses;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int32_t w = 1; w < warps; ++w) all_losses += losses[w];
    partial[blockIdx.x] = all_losses;
  }
}

template <int kTeam>
struct DistilShared {
  float high[2][kTeam / 32], sum[2][kTeam / 32];
  int32_t some[2], wrong[2];
  float all_high, all_sum;  // of a block, for its cluster
};

// Rows whose entries a team has in shared memory at a time: of a block's last row, whose classes are
// yet to be written, of the one at hand, and of one that a warp ahead of the others comes to.
template <int kTeam>
constexpr int32_t kHeld = kTeam == 32 ? 1 : 3;

// Longer rows: a warp (kTeam 32, several to a block) or a block is a team, or a cluster of blocks
// (kTeam 512), to which a row's vectors are dealt out in slices.  Rows come 32 at a time, as in
// DistilWarps; each block's first warp reads the teacher, and that of a row's first block computes
// the losses.  A block has one barrier per row: behind it, the sums of all warps are there, and the
// gradient of the row before has been stored, so that the teacher's classes can be written into it.
// tiles > 1: a slice does not fit, and is read again, part by part, for each pass.  16000 x 5000 fp16
// with 32 entries, a quarter beyond their lengths: 66 us, 4.3 TB/s; 4096 x 50021 bf16 with 64: 190 us,
// 4.3 TB/s, with two blocks of 100 KB to an SM, whose 16 warps issue in 43% of the cycles.
template <typename T, int kTeam>
__global__ void
__launch_bounds__(kTeam == 32 ? 128 : kTeam, kTeam == 32 ? 5 : kTeam == 128 ? 4 : kTeam == 256 ? 2 : 1)
DistilRing(Rows<T> rows, Teacher t, float4 *norm, float *loss, double *partial, T *grad,
           int64_t outer_stride, int64_t inner_stride, DistilBy by, int32_t vectors,
           int32_t tiles) {
  extern __shared__ uint4 shared[];
  __shared__ DistilShared<kTeam> sh;
  __shared__ double losses[4];
  LetNextStart();
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31,
                teams = kTeam == 32 ? (int32_t)blockDim.x / 32 : 1,
                team = kTeam == 32 ? warp : 0,
                tid = kTeam == 32 ? lane : (int32_t)threadIdx.x;
  const bool leads = kTeam == 32 || warp == 0;
  const uint32_t cluster = kTeam == 512 ? ClusterSize() : 1,
                 rank = kTeam == 512 ? ClusterRank() : 0;
  const int32_t stage = kTeam * vectors;
  uint4 *slot = shared + team * stage + tid;
  char *entries = reinterpret_cast<char *>(shared + teams * stage) +
                  team * kHeld<kTeam> * t.entries * kEntryBytes;
  const int32_t apart = (int32_t)(gridDim.x / cluster) * teams;
  const float k = kLog2e / t.temperature;
  bool waited = by.device == nullptr;
  float scale = by.host.rounded;
  double all_losses = 0.0;
  int32_t parity = 0, held = 0;
  // the row whose classes are yet to be written
  struct {
    T *out = nullptr;
    int32_t begin, end, held;
    float from, inverse, times;
  } last_row;
  const auto name = [&]() {
    if (last_row.out == nullptr) return;
    // (a block's last warps: the first one has the teacher to read)
    WriteNamed(TeacherAt(entries + last_row.held * t.entries * kEntryBytes, t.entries), t,
               last_row.out, last_row.begin, last_row.end, kTeam - 1 - tid, kTeam, last_row.from, k,
               last_row.inverse, last_row.times);
    last_row.out = nullptr;
  };
  for (int32_t base = (int32_t)(blockIdx.x / cluster) * teams + team; base < rows.count;
       base += 32 * apart) {
    const int32_t mine = base + lane * apart,
                  taken = min(32, (rows.count - base + apart - 1) / apart);
    const T *my_row = nullptr;
    T *my_out = nullptr;
    if (lane < taken) {
      const RowPlace at = PlaceOf(rows, mine);
      if (at.counts) my_row = rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride;
      if (grad) my_out = grad + at.o * outer_stride + at.i * inner_stride;
    }
    const auto row_of = [&](int32_t q) {
      const T *row = reinterpret_cast<const T *>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_row), q & 31));
      return q < taken ? row : nullptr;
    };
    // this thread's part of this block's slice of a row
    const auto part_of = [&](const T *row) {
      const RowSpan<T> span(row, rows.classes);
      const int32_t slice = (span.vectors + (int32_t)cluster - 1) / (int32_t)cluster;
      const int32_t first = min(span.vectors, (int32_t)rank * slice),
                    last = min(span.vectors, first + slice);
      return RowPart<T>(span, first, last, tid, kTeam);
    };
    const T *next = row_of(0);
    if (tiles == 1 && next != nullptr) SendFor<kTeam, 0>(slot, part_of(next), rows);
    // the teacher's entries of the next row; a block's with the student's scores, which its first
    // warp has no other way to, and those of the row behind
    constexpr int kAhead = kTeam == 32 ? 1 : K2B200_MAX_TOP / 32;
    TeacherAhead<kAhead> ahead, behind;
    if (leads && next != nullptr) {
      ReadAhead(ahead, t, base, lane);
      if (kTeam > 32) ReadScores(ahead, t, rows.classes, next, lane);
    }
    if (kTeam > 32 && leads && row_of(1) != nullptr) ReadAhead(behind, t, base + apart, lane);
    float my_high = 0.0f, my_sum = 0.0f, my_term = 0.0f, my_mass = 0.0f;
    bool my_some = false, my_wrong = false;
    for (int32_t q = 0; q < taken; ++q) {
      const int32_t r = base + q * apart;
      const T *row = next;
      next = row_of(q + 1);
      T *out = reinterpret_cast<T *>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_out), q));
      const RowPart<T> whole = part_of(row), coming = part_of(next);
      const RowPart<T> *const then = tiles == 1 && next != nullptr ? &coming : nullptr;
      if (row != nullptr) held = held + 1 < kHeld<kTeam> ? held + 1 : 0;
      TeacherRow teacher = TeacherAt(entries + held * t.entries * kEntryBytes, t.entries);
      if (kTeam > 32 && leads) {
        if (row != nullptr) ReadTeacher(teacher, ahead, t, r, rows.classes, row, lane);
        ahead = behind;
        if (next != nullptr) ReadScores(ahead, t, rows.classes, next, lane);
        if (row_of(q + 2) != nullptr) ReadAhead(behind, t, r + 2 * apart, lane);
      }
      // (a row of the gradient may lie otherwise and have a vector more)
      const auto zero = [&]() {
        const RowSpan<T> zeros(out, rows.classes);
        const int32_t slice = (zeros.vectors + (int32_t)cluster - 1) / (int32_t)cluster;
        WriteZeros(out, rows.classes, (int32_t)rank * slice, ((int32_t)rank + 1) * slice, tid,
                   kTeam);
      };
      if (row == nullptr) {
        if (out) zero();
        if (then) SendFor<kTeam, 0>(slot, coming, rows);
        if (kTeam == 32 && next != nullptr) ReadAhead(ahead, t, r + apart, lane);
        continue;  // (all blocks of the cluster)
      }
      WaitForAll();
      if (kTeam == 32) {
        __syncwarp();  // the row as the other lanes have it
        const T *here = reinterpret_cast<const T *>(slot - lane) + whole.span.shift;
        ReadScores(ahead, t, rows.classes, here, lane);
        ReadTeacher(teacher, ahead, t, r, rows.classes, here, lane);
        if (next != nullptr) ReadAhead(ahead, t, r + apart, lane);
        __syncwarp();
      }
      const RowSpan<T> &span = whole.span;
      const int32_t first = whole.first - tid, last = whole.last;
      // f(part) for each part of the slice, which is there
      const auto each = [&](auto &&f) {
        if (tiles == 1) {
          f(whole);
          return;
        }
        for (int32_t tile = first; tile < last; tile += stage) {
          const RowPart<T> part(span, tile, min(last, tile + stage), tid, kTeam);
          SendFor<kTeam, 0>(slot, part, rows);
          WaitForAll();
          CutEnds<kTeam>(slot, part);
          f(part);
        }
      };
      if (tiles == 1) CutEnds<kTeam>(slot, whole);
      // the largest score and the sum of each warp
      Sums sums = NoSums();
      each([&](const RowPart<T> &part) {
        AddRow<false, kTeam>(sums, slot, part.most, row, k, NoRefill());
      });
      float high, sum = WarpSums<false>(sums, k, &high).x;
      bool some = teacher.some, wrong = teacher.wrong;
      if (kTeam > 32) {
        // (a warp is at most one barrier ahead: the values of the row before are still read)
        parity ^= 1;
        if (lane == 0) {
          sh.high[parity][warp] = high;
          sh.sum[parity][warp] = sum;
          if (warp == 0) {
            sh.some[parity] = some;
            sh.wrong[parity] = wrong;
          }
        }
        __syncthreads();
        some = sh.some[parity];
        wrong = sh.wrong[parity];
        const bool one = lane < kTeam / 32;
        const float h = one ? sh.high[parity][lane] : -INFINITY;
        high = WarpMaxF(h);
        sum = WarpSumF(one ? sh.sum[parity][lane] *
                                 Exp2((h - (high == -INFINITY ? 0.0f : high)) * k)
                           : 0.0f);
        name();
      }
      if (kTeam == 512 && cluster > 1) {
        if (tid == 0) {
          sh.all_high = high;
          sh.all_sum = sum;
        }
        ClusterSync();
        const bool one = lane < (int32_t)cluster;
        const float h = one ? ReadFrom(&sh.all_high, lane) : -INFINITY,
                    part = one ? ReadFrom(&sh.all_sum, lane) : 0.0f;
        high = WarpMaxF(h);
        sum = WarpSumF(one ? part * Exp2((h - (high == -INFINITY ? 0.0f : high)) * k) : 0.0f);
        ClusterSync();  // nobody goes on while others read its memory
      }
      const float from = high == -INFINITY ? 0.0f : high;
      if (leads) {
        const float term = ShareOut(teacher, t, k, from, lane);
        if (lane == q) {
          my_high = from;
          my_sum = sum;
          my_term = term;
          my_mass = teacher.mass;
          my_some = some;
          my_wrong = wrong;
        }
      }
      if (out && some) {
        if (!waited) {
          WaitForPrevious();
          waited = true;
          scale = by.device->rounded;
        }
        const float times = t.temperature * scale, inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        each([&](const RowPart<T> &part) {
          WriteGradRow<kTeam>(slot, part, out, from, k, wrong ? NAN : inverse * times);
        });
        if (then) SendFor<kTeam, 0>(slot, coming, rows);
        if (!wrong) {
          last_row.out = out;
          last_row.begin = max(0, span.Column(first));
          last_row.end = min(span.classes, span.Column(last));
          last_row.held = held;
          last_row.from = from;
          last_row.inverse = inverse;
          last_row.times = times;
        }
      } else {
        if (out) zero();
        if (then) SendFor<kTeam, 0>(slot, coming, rows);
      }
      if (kTeam == 32) {
        __syncwarp();
        name();
        __syncwarp();  // the next row's entries come to the same place
      }
    }
    if (!leads || rank != 0) continue;
    float row_loss = 0.0f;
    if (lane < taken) {
      if (my_row) row_loss = RowLoss(t.temperature, my_some, my_wrong, my_mass, my_sum, my_term);
      if (norm) norm[mine] = make_float4(my_high, my_sum, 0.0f, 0.0f);
      if (loss) loss[mine] = row_loss * by.host.rounded;
    }
    all_losses += row_loss;
  }
  if (kTeam > 32) {
    __syncthreads();
    name();
  }
  if (loss) return;
  // (the next kernel reads the scale too, and waits for nothing but this one's end)
  if (!waited) WaitForPrevious();
  for (int32_t d = 16; d > 0; d >>= 1) all_losses += __shfl_xor_sync(0xffffffffu, all_losses, d);
  if (kTeam > 32) {
    if (rank == 0 && tid == 0) partial[blockIdx.x / cluster] = all_losses;
  } else {
    if (lane == 0) losses[warp] = all_losses;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int32_t w = 1; w < teams; ++w) all_losses += losses[w];
      partial[blockIdx.x] = all_losses;
    }
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
// a row per warp (kTeam 32), dealt out to the blocks there are.  unless_one: what is there stays where
// the upstream is 1.  64000 rows of 500 bf16 classes with 32 entries: 92 us, a warp going through its
// row's teacher and classes one after the other; 4096 of 32001 with 64: 128 us, 4.1 TB/s.
template <typename T, int kTeam>
__global__ void __launch_bounds__(256)
DistilBackward(Rows<T> rows, Teacher t, const float4 *norm, T *grad, int64_t outer_stride,
               int64_t inner_stride, DistilBy by, k2b200_row_grad up, int32_t unless_one,
               int64_t items, int32_t parts, int32_t part) {
  constexpr int kTile = 4;
  extern __shared__ uint4 shared[];
  __shared__ int32_t flags[2];
  if (unless_one && up.grad[0] == 1.0f) return;
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t tid = kTeam == 32 ? lane : (int32_t)threadIdx.x;
  const float k = kLog2e / t.temperature;
  const float scale = t.temperature * (by.device ? by.device->rounded : by.host.rounded);
  TeacherRow teacher = TeacherAt(
      reinterpret_cast<char *>(shared) + (kTeam == 32 ? warp * t.entries * kEntryBytes : 0),
      t.entries);
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
    TeamSync<kTeam>();  // the entries of the row before have been read
    if (kTeam == 32 || warp == 0) {
      TeacherAhead<1> ahead;
      ReadAhead(ahead, t, r, lane);
      ReadScores(ahead, t, rows.classes, span.row, lane);
      ReadTeacher(teacher, ahead, t, r, rows.classes, span.row, lane);
      ShareOut(teacher, t, k, 0.0f, lane);
      if (kTeam > 32 && lane == 0) {
        flags[0] = teacher.some;
        flags[1] = teacher.wrong;
      }
    }
    TeamSync<kTeam>();
    const bool some = kTeam > 32 ? flags[0] : teacher.some,
               wrong = kTeam > 32 ? flags[1] : teacher.wrong;
    if (!some) {
      WriteZeros(out, rows.classes, first, zeros_end, tid, kTeam);
      continue;
    }
    const float4 n = norm[r];
    const float times = scale * up.grad[at.o * up.outer + at.i * up.inner];
    const float inverse = n.y == 0.0f ? 0.0f : 1.0f / n.y;
    const float spread = wrong ? NAN : inverse * times;
    const bool aligned = (((uintptr_t)out ^ (uintptr_t)span.row) & 15) == 0;
    // vectors [from, to) are whole
    const int32_t from = first < last && !span.Whole(span.Column(first)) ? first + 1 : first,
                  to = last > from && !span.Whole(span.Column(last - 1)) ? last - 1 : last;
    const uint4 *in = reinterpret_cast<const uint4 *>(span.row - span.shift);
    const auto store = [&](int32_t j, const uint4 &x, bool whole) {
      float f[kPer<T>];
      Spread(x, span.row, n.x, k, spread, f);
      if (whole)
        *reinterpret_cast<uint4 *>(out + span.Column(j)) = Pack(f, out);
      else
        Store(out, span, false, j, f);
    };
    uint4 v[kTile];
    const auto load = [&](int32_t tile) {
#pragma unroll
      for (int i = 0; i < kTile; ++i)
        if (tile + i * kTeam < to) v[i] = in[tile + i * kTeam];
    };
    load(from + tid);
    for (int32_t tile = from + tid; tile < to; tile += kTeam * kTile) {
      uint4 x[kTile];
#pragma unroll
      for (int i = 0; i < kTile; ++i) x[i] = v[i];
      load(tile + kTeam * kTile);
      if (aligned) {
#pragma unroll
        for (int i = 0; i < kTile; ++i)
          if (tile + i * kTeam < to) store(tile + i * kTeam, x[i], true);
      } else {
#pragma unroll 1
        for (int32_t j = tile; j < min(to, tile + kTeam * kTile); j += kTeam)
          store(j, in[j], false);
      }
    }
    // the row's ends
    if (tid < 2) {
      const int32_t j = tid == 0 ? first : last - 1;
      if ((j < from || j >= to) && j < last && (tid == 0 || j > first))
        store(j, span.Edge(j), false);
    }
    TeamSync<kTeam>();
    if (!wrong)
      WriteNamed(teacher, t, out, max(0, span.Column(first)),
                 min(span.classes, span.Column(last)), tid, kTeam, n.x, k, inverse, times);
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
  K2B_REQUIRE(Aligned(t->tokens, IntSize(t->tokens_64)) && Aligned(t->scores, FloatSize(t->type)),
              "a teacher's tokens or scores that are not aligned to their type");
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
  double *partial =
      workspace ? reinterpret_cast<double *>(static_cast<char *>(workspace) + kDistilHead) : nullptr;
  if (by.device) {
    DistilCount<<<1, 256, 0, s>>>(rows->lengths, rows->lengths_64, rows->outer, rows->inner,
                                   t->weight, static_cast<DistilScale *>(workspace));
    NoteLaunch();
  }
  int32_t parts = 0;
  if (r.count > 0) {
    const int32_t held = t->entries * kEntryBytes;
    const RowPlan p = PlanRows(r, kHeld<32> * held, kHeld<512> * held);
    const size_t smem =
        (size_t)p.ring + (size_t)(p.team == 32 ? kHeld<32> : kHeld<512>) * held * (p.block / p.team);
    parts = (int32_t)(p.blocks / p.cluster);
    float4 *norms = reinterpret_cast<float4 *>(norm);
    float *row_losses = t->reduction == 0 ? loss : nullptr;
    const auto launch = [&](auto kernel, auto... how) {
      const cudaError_t e = AllowShared(kernel, smem);
      if (e != cudaSuccess) return e;
      return LaunchRows(kernel, p.blocks, p.block, smem, p.cluster, by.device != nullptr, s, r,
                        teacher, norms, row_losses, partial, static_cast<T *>(grad),
                        outer_stride, inner_stride, by, how...);
    };
    K2B_CUDA_OK(p.in_registers ? launch(p.vectors == 1   ? DistilWarps<T, 1>
                                        : p.vectors == 2 ? DistilWarps<T, 2>
                                        : p.vectors == 4 ? DistilWarps<T, 4>
                                                         : DistilWarps<T, 8>)
                               : launch(p.team == 32    ? DistilRing<T, 32>
                                        : p.team == 128 ? DistilRing<T, 128>
                                        : p.team == 256 ? DistilRing<T, 256>
                                                        : DistilRing<T, 512>,
                                        p.vectors, p.tiles));
    NoteLaunch();
  }
  if (t->reduction != 0) {
    K2B_CUDA_OK(LaunchRows(DistilLoss, 1, 1024, 0, 1, r.count > 0, s, partial, parts, by, loss));
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
  // vectors of a row, wherever it begins: up to 256 of them are a warp's; more are dealt out to
  // blocks in parts as in the backward pass of token scores
  const int32_t vectors = CeilDiv((int64_t)r.classes + kPer<T> - 1, kPer<T>) + 1;
  const bool few = vectors <= 256;
  const int32_t part = CeilDiv(vectors, 4096) * (int64_t)r.count >= 2 * NumSms() ? 4096 : 1024,
                parts = few ? 1 : CeilDiv(vectors, part);
  const int32_t warps =
      few ? (int32_t)std::min<int64_t>(8, std::max<int64_t>(1, r.count / NumSms())) : 1;
  const int64_t items = few ? CeilDiv(r.count, warps) : (int64_t)r.count * parts;
  const int64_t blocks = std::min<int64_t>(items, 8 * (int64_t)NumSms());
  auto kernel = few ? DistilBackward<T, 32> : DistilBackward<T, 256>;
  kernel<<<(uint32_t)blocks, few ? 32 * warps : 256, (size_t)t->entries * kEntryBytes * warps, s>>>(
      r, teacher, reinterpret_cast<const float4 *>(norm), static_cast<T *>(grad), outer_stride,
      inner_stride, ByOf(rows, t, workspace), *up, unless_one, items, parts, part);
  NoteLaunch();
  K2B_CUDA_OK(cudaGetLastError());
  return kOk;
}

}  // namespace

extern "C" {

size_t k2b200_distillation_workspace_bytes(const k2b200_class_rows *rows) {
  if (rows == nullptr) return 0;
  // (a loss per block: PlanRows has at most 64 of them on an SM)
  return kDistilHead + sizeof(double) * (size_t)std::min<int64_t>(rows->outer * rows->inner,
                                                                  64 * (int64_t)NumSms());
}

int32_t k2b200_distillation(const k2b200_class_rows *rows, const k2b200_teacher *teacher,
                            float *loss, float *norm, void *grad_scores,
                            int64_t grad_outer_stride, int64_t grad_inner_stride,
                            void *workspace, size_t workspace_bytes, void *stream) {
  K2B_FORWARD(CheckRows(rows));
  K2B_REQUIRE(Aligned(norm, 16) && Aligned(workspace, sizeof(double)),
              "norm or workspace that are not aligned to 16 and 8 bytes");
  K2B_REQUIRE(Aligned(grad_scores, FloatSize(rows->type)) && Aligned(loss, 4),
              "a loss or gradient that is not aligned to its type");
  K2B_FORWARD(CheckTeacher(teacher, rows));
  K2B_REQUIRE(!grad_scores || teacher->reduction != 0,
              "the gradient of row losses needs their upstream");
  const size_t need =
      teacher->reduction == 0 ? 0 : k2b200_distillation_workspace_bytes(rows);
  K2B_REQUIRE(workspace || need == 0, "NULL pointer");
  K2B_REQUIRE(loss || (teacher->reduction == 0 && rows->outer * rows->inner == 0),
              "NULL pointer");
  if (workspace_bytes < need) {
    SetError("workspace of %zu bytes, %zu are needed", workspace_bytes, need);
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
  K2B_REQUIRE(Aligned(norm, 16) && Aligned(workspace, sizeof(double)),
              "norm or workspace that are not aligned to 16 and 8 bytes");
  K2B_REQUIRE(Aligned(grad_scores, FloatSize(rows->type)) && Aligned(upstream ? upstream->grad : nullptr, 4),
              "a gradient that is not aligned to its type");
  K2B_FORWARD(CheckTeacher(teacher, rows));
  if (rows->outer * rows->inner == 0) return kOk;
  const size_t need = teacher->reduction == 0 ? 0 : kDistilHead;
  K2B_REQUIRE(norm && upstream && upstream->grad && grad_scores && (workspace || need == 0),
              "NULL pointer");
  if (workspace_bytes < need) {
    SetError("workspace of %zu bytes, %zu are needed", workspace_bytes, need);
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
