// Rows of class scores as the kernels of token_scores.cu and distillation.cu hold them.
//
// A team of threads - a warp, a block, or the blocks of a cluster - has a row at a time, as aligned
// vectors of 16 bytes that each thread copies to shared memory for itself: no barrier stands between
// a copy and its use, only cp.async's own wait, and other rows are on their way meanwhile.  Short
// rows (up to 4 KB: a warp's 8 vectors per lane) go on to registers, and their place is free for the
// warp's next row at once; longer ones are read from shared memory as often as they are needed, by
// loops whose code stays in the instruction cache (unrolled over 20 vectors of a thread it did not:
// 16000 x 5000 fp16 rows with their gradient took 120 us, most of it waiting for instructions).
// Where a row begins inside a vector (any alignment of an element will do) the first and the last
// vector are shared with its neighbours: what is not the row's is -inf.
//
//   p_c = 2^((x_c - high) * log2 e) / sum   high the largest score, sum over all classes
//
// Everything is computed in 32 bits, whatever the type of the scores.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/k2b200.h"
#include "common.cuh"
#include "cp_async.cuh"

namespace k2b {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// (columns of a vector stay within 32 bits)
constexpr int32_t kMaxClasses = 1 << 30;

// What a kernel needs of k2b200_class_rows.
template <typename T>
struct Rows {
  const T *scores;
  int32_t classes, count;
  uint32_t inner, inverse, shift;  // r / inner = r * inverse >> shift for r < 2^28
  int64_t outer_stride, inner_stride;
  const T *begin, *end;  // the first class of all rows, and behind the last one
  const void *lengths;
  int32_t lengths_64;
};

struct RowPlace {
  int64_t o, i;
  bool counts;
};

// An element of an array of int32 or int64, as int64.
__device__ __forceinline__ int64_t IntAt(const void *ints, int32_t is_64, int64_t k) {
  return is_64 ? static_cast<const int64_t *>(ints)[k]
               : (int64_t)static_cast<const int32_t *>(ints)[k];
}

template <typename T>
__device__ __forceinline__ RowPlace PlaceOf(const Rows<T> &rows, int32_t r) {
  RowPlace p;
  const uint32_t o = (uint32_t)((uint64_t)(uint32_t)r * rows.inverse >> rows.shift);
  p.o = o;
  p.i = (uint32_t)r - o * rows.inner;
  p.counts = rows.lengths == nullptr || p.i < IntAt(rows.lengths, rows.lengths_64, p.o);
  return p;
}

// ---------------------------------------------------------------------------
// numbers
// ---------------------------------------------------------------------------
__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T FromFloat(float v);
template <>
__device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// 2^x, off by at most 2 units of the last place and 0 below 2^-126: a class of that share is one
// that has none.
__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two numbers in one instruction each, rounded as by single ones.
struct Two {
  uint64_t bits;
};
__device__ __forceinline__ Two MakeTwo(float a, float b) {
  Two t;
  asm("mov.b64 %0, {%1, %2};" : "=l"(t.bits) : "f"(a), "f"(b));
  return t;
}
__device__ __forceinline__ float2 Split(Two t) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(t.bits));
  return f;
}
__device__ __forceinline__ Two Add(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two Mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two Fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r.bits)
      : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}

// Order of scores: an unsigned number that grows with the score, 0 for none.  NaN comes before all
// numbers and -0 equals +0.  With the class below it, two keys of a row are never equal.
__device__ __forceinline__ uint32_t OrderOf(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  if (v != v) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float ScoreOf(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t KeyOf(float v, int32_t c) {
  return (uint64_t)OrderOf(v) << 32 | (uint32_t)~c;
}

__device__ __forceinline__ float WarpMaxF(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ float WarpSumF(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// Both sums at once: the halves of the warp take one each.
__device__ __forceinline__ float2 WarpSum2F(float a, float b) {
  const bool high = threadIdx.x & 16;
  float mine = high ? b : a;
  mine += __shfl_xor_sync(0xffffffffu, high ? a : b, 16);
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  const float other = __shfl_xor_sync(0xffffffffu, mine, 16);
  return high ? make_float2(other, mine) : make_float2(mine, other);
}

// ---------------------------------------------------------------------------
// vectors of 16 bytes
// ---------------------------------------------------------------------------
template <typename T>
constexpr int kPer = 16 / (int)sizeof(T);

// Scores 2k and 2k + 1 of a vector.
template <int kPair>
__device__ __forceinline__ float2 PairOf(const uint4 &v, const float *) {
  return kPair == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                    : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
}
template <int kPair>
__device__ __forceinline__ uint32_t WordOf(const uint4 &v) {
  return kPair == 0 ? v.x : kPair == 1 ? v.y : kPair == 2 ? v.z : v.w;
}
template <int kPair>
__device__ __forceinline__ float2 PairOf(const uint4 &v, const __nv_bfloat16 *) {
  const uint32_t w = WordOf<kPair>(v);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <int kPair>
__device__ __forceinline__ float2 PairOf(const uint4 &v, const __half *) {
  const uint32_t w = WordOf<kPair>(v);
  __half2 h;
  memcpy(&h, &w, 4);
  return __half22float2(h);
}
template <typename T>
__device__ __forceinline__ void Unpack(const uint4 &v, float (&f)[kPer<T>], const T *type) {
  const float2 a = PairOf<0>(v, type), b = PairOf<1>(v, type);
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
  if constexpr (kPer<T> == 8) {
    const float2 c = PairOf<2>(v, type), d = PairOf<3>(v, type);
    f[4] = c.x;
    f[5] = c.y;
    f[6] = d.x;
    f[7] = d.y;
  }
}
// f(pair, index) for the pairs of a vector.
template <typename T, typename F>
__device__ __forceinline__ void EachPair(const uint4 &v, const T *type, F &&f) {
  f(PairOf<0>(v, type), 0);
  f(PairOf<1>(v, type), 1);
  if constexpr (kPer<T> == 8) {
    f(PairOf<2>(v, type), 2);
    f(PairOf<3>(v, type), 3);
  }
}
__device__ __forceinline__ uint4 Pack(const float (&f)[4], const float *) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                    __float_as_uint(f[3]));
}
template <typename Pair, Pair (*kRound)(float, float)>
__device__ __forceinline__ uint4 PackPairs(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const Pair p = kRound(f[2 * k], f[2 * k + 1]);
    memcpy(&w[k], &p, 4);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 Pack(const float (&f)[8], const __half *) {
  return PackPairs<__half2, __floats2half2_rn>(f);
}
__device__ __forceinline__ uint4 Pack(const float (&f)[8], const __nv_bfloat16 *) {
  return PackPairs<__nv_bfloat162, __floats2bfloat162_rn>(f);
}

// Makes the compiler forget where a vector's words come from: it would keep a row unpacked between
// the passes over it, in twice the registers.
__device__ __forceinline__ uint4 &Packed(uint4 &v) {
  asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w));
  return v;
}
// ... and does not unpack it before `sum` is what it is here: it would unpack all of a row's vectors
// at once otherwise.
__device__ __forceinline__ void After(uint4 &v, Two &sum) {
  asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w), "+l"(sum.bits));
}

// The largest of a vector's scores; NaN are passed over.
__device__ __forceinline__ float VectorMax(uint4 v, const float *) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
               fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
template <typename Pair>
__device__ __forceinline__ Pair PairMax(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  Pair p[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) memcpy(&p[k], &w[k], 4);
  return __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
}
__device__ __forceinline__ float VectorMax(uint4 v, const __half *) {
  const float2 f = __half22float2(PairMax<__half2>(v));
  return fmaxf(f.x, f.y);
}
__device__ __forceinline__ float VectorMax(uint4 v, const __nv_bfloat16 *) {
  const float2 f = __bfloat1622float2(PairMax<__nv_bfloat162>(v));
  return fmaxf(f.x, f.y);
}
__device__ __forceinline__ uint4 LowestVector(const float *) {
  return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
}
__device__ __forceinline__ uint4 LowestVector(const __half *) {
  return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
}
__device__ __forceinline__ uint4 LowestVector(const __nv_bfloat16 *) {
  return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
}

// A row as aligned vectors: vector j holds the classes from Column(j) on, of which the first
// vector's first `shift` and the last one's last are none of the row's.
template <typename T>
struct RowSpan {
  const T *row;
  int32_t classes, shift, vectors;
  __device__ __forceinline__ RowSpan(const T *x, int32_t c) : row(x), classes(c) {
    shift = (int32_t)(((uintptr_t)x & 15) / sizeof(T));
    vectors = (shift + c + kPer<T> - 1) / kPer<T>;
  }
  __device__ __forceinline__ int32_t Column(int32_t j) const { return j * kPer<T> - shift; }
  __device__ __forceinline__ bool Whole(int32_t c0) const {
    return c0 >= 0 && c0 + kPer<T> <= classes;
  }
  // A vector that is not whole, element by element.
  __device__ __forceinline__ uint4 Edge(int32_t j) const {
    const int32_t c0 = Column(j);
    float f[kPer<T>];
#pragma unroll
    for (int k = 0; k < kPer<T>; ++k) {
      const int32_t c = c0 + k;
      f[k] = c >= 0 && c < classes ? ToFloat(row[c]) : -INFINITY;
    }
    return Pack(f, row);  // (exact)
  }
  __device__ __forceinline__ uint4 Vector(int32_t j) const {
    const int32_t c0 = Column(j);
    return Whole(c0) ? *reinterpret_cast<const uint4 *>(row + c0) : Edge(j);
  }
};

// Elements [begin, end) of a vector, -inf elsewhere.
__device__ __forceinline__ uint4 Keep(const uint4 &v, int32_t begin, int32_t end, const float *t,
                                      const uint4 &low) {
  return make_uint4(begin <= 0 && end > 0 ? v.x : low.x, begin <= 1 && end > 1 ? v.y : low.y,
                    begin <= 2 && end > 2 ? v.z : low.z, begin <= 3 && end > 3 ? v.w : low.w);
}
__device__ __forceinline__ uint4 Keep(const uint4 &v, int32_t begin, int32_t end, const float *t) {
  return Keep(v, begin, end, t, LowestVector(t));
}
template <typename T>
__device__ __forceinline__ uint4 Keep(const uint4 &v, int32_t begin, int32_t end, const T *t) {
  // (whole words where pairs of scores are aligned)
  if (((begin | end) & 1) == 0)
    return Keep(v, begin / 2, end / 2, static_cast<const float *>(nullptr), LowestVector(t));
  // (a shift by 32 or more leaves nothing)
  const auto word = [&](uint32_t w, int32_t k, uint32_t low) {
    uint32_t from, to;
    asm("shl.b32 %0, %1, %2;" : "=r"(from) : "r"(~0u), "r"(max(0, 16 * begin - 32 * k)));
    asm("shl.b32 %0, %1, %2;" : "=r"(to) : "r"(~0u), "r"(max(0, 16 * end - 32 * k)));
    const uint32_t keep = from & ~to;
    return (w & keep) | (low & ~keep);
  };
  const uint32_t low = LowestVector(t).x;
  return make_uint4(word(v.x, 0, low), word(v.y, 1, low), word(v.z, 2, low), word(v.w, 3, low));
}

// A thread's vectors of a row: first + i * team for those before `last`, at slot[i * team].
template <typename T>
struct RowPart {
  RowSpan<T> span;
  int32_t first, last, mine, most;  // mine: this thread's; most: any thread's
  __device__ __forceinline__ RowPart(const RowSpan<T> &row, int32_t from, int32_t to, int32_t tid,
                                     int32_t team)
      : span(row), first(from + tid), last(to) {
    mine = first < last ? (last - first + team - 1) / team : 0;
    most = (to - from + team - 1) / team;
  }
};

// Waits until what this thread has sent for is there.
__device__ __forceinline__ void WaitForAll() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Sends for them.  A vector that the row shares with others is copied as a whole where all of it
// lies between the first and the last class of all rows, and read element by element elsewhere.
// kVectors: what a thread has at most (0: any number).
template <int kTeam, int kVectors, typename T>
__device__ __forceinline__ void SendFor(uint4 *slot, const RowPart<T> &part, const Rows<T> &rows) {
  asm volatile("" ::: "memory");  // (behind the last use of what was there)
  const RowSpan<T> &span = part.span;
  const int32_t end = span.vectors - 1;
  const uint4 *at = reinterpret_cast<const uint4 *>(span.row - span.shift);
  const bool front = reinterpret_cast<const T *>(at) >= rows.begin,
             tail = reinterpret_cast<const T *>(at + span.vectors) <= rows.end;
  if (front && tail) {
    if (kVectors > 0) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
        if (i < part.mine) CpAsync16(slot + i * kTeam, at + part.first + i * kTeam);
    } else {
#pragma unroll 4
      for (int32_t i = 0; i < part.mine; ++i)
        CpAsync16(slot + i * kTeam, at + part.first + i * kTeam);
    }
  } else {
    for (int32_t i = 0; i < part.mine; ++i) {
      const int32_t j = part.first + i * kTeam;
      if ((j > 0 || front) && (j < end || tail))
        CpAsync16(slot + i * kTeam, at + j);
      else
        slot[i * kTeam] = span.Edge(j);
    }
  }
}
// The row behind the one at hand, whose vectors are sent for one by one, each as soon as its place
// is free.  A row that SendFor would not copy as a whole waits for the end (Rest).
template <int kTeam, typename T>
struct Refill {
  const uint4 *at;
  int32_t mine;  // this thread's that are sent for one by one
  __device__ __forceinline__ Refill(const RowPart<T> *part, const Rows<T> &rows)
      : at(nullptr), mine(0) {
    if (part == nullptr) return;
    const RowSpan<T> &span = part->span;
    const T *begin = span.row - span.shift;
    if (begin < rows.begin || begin + (int64_t)span.vectors * kPer<T> > rows.end) return;
    at = reinterpret_cast<const uint4 *>(begin) + part->first;
    mine = part->mine;
  }
  __device__ __forceinline__ void operator()(uint4 *slot, int32_t i) const {
    asm volatile("" ::: "memory");  // (behind the last use of what was there)
    if (i < mine) CpAsync16(slot + i * kTeam, at + i * kTeam);
  }
  // What places `done` and on are for.
  __device__ __forceinline__ void Rest(uint4 *slot, int32_t done, const RowPart<T> *part,
                                       const Rows<T> &rows) const {
    if (part == nullptr) return;
    if (at == nullptr)
      SendFor<kTeam, 0>(slot, *part, rows);
    else
      for (int32_t i = done; i < mine; ++i) (*this)(slot, i);
  }
};
struct NoRefill {
  __device__ __forceinline__ void operator()(uint4 *, int32_t) const {}
};

// -inf for what is not the row's, once they are there.
template <int kTeam, typename T>
__device__ __forceinline__ void CutEnds(uint4 *slot, const RowPart<T> &part) {
  const RowSpan<T> &span = part.span;
  const int32_t end = span.vectors - 1, rest = span.classes - span.Column(end);
  if (span.shift != 0 && part.first == 0 && part.mine > 0)
    slot[0] = Keep(slot[0], span.shift, kPer<T>, span.row);
  if (rest < kPer<T> && part.mine > 0 && part.first + (part.mine - 1) * kTeam == end) {
    uint4 &v = slot[(part.mine - 1) * kTeam];
    v = Keep(v, 0, rest, span.row);
  }
  // (as many for every thread, so that those of a warp go through a row together)
  if (part.mine < part.most) slot[part.mine * kTeam] = LowestVector(span.row);
}

// Sums of 2^d and of d 2^d over a vector, d = (x - high) * k.
template <bool kSlope, typename T>
__device__ __forceinline__ void AddVector(const uint4 &v, const T *type, float high, float k,
                                          Two &sum, Two &slope) {
  const Two minus = MakeTwo(-high, -high), by = MakeTwo(k, k);
  EachPair(v, type, [&](float2 x, int) {
    const float2 d = Split(Mul(Add(MakeTwo(x.x, x.y), minus), by));
    const Two e = MakeTwo(Exp2(d.x), Exp2(d.y));
    sum = Add(sum, e);
    // 0 and not 0 * -inf where p = 0
    if (kSlope) slope = Fma(e, MakeTwo(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)), slope);
  });
}

// A thread's vectors, from shared memory to registers.
template <int kTeam, int kVectors, typename T>
__device__ __forceinline__ void Take(uint4 (&v)[kVectors], const uint4 *slot,
                                     const RowPart<T> &part) {
#pragma unroll
  for (int i = 0; i < kVectors; ++i)
    v[i] = i < part.mine ? slot[i * kTeam] : LowestVector(part.span.row);
}

// The largest score of a thread's vectors, those of the first and of the second half apart.
template <int kVectors, typename T>
__device__ __forceinline__ float2 Highest(uint4 (&v)[kVectors], const T *type) {
  float half[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    float &g = half[2 * i / kVectors];
    g = fmaxf(g, VectorMax(Packed(v[i]), type));
  }
  return make_float2(half[0], half[1]);
}

// Sums of 2^d and of d 2^d over a thread's vectors, d = (x - high) * k: two vectors at a time.
template <bool kSlope, int kVectors, typename T>
__device__ __forceinline__ float2 SumUp(uint4 (&v)[kVectors], const T *type, float high, float k) {
  Two sum[2] = {}, slope[2] = {};
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    After(v[i], sum[i & 1]);
    AddVector<kSlope>(v[i], type, high, k, sum[i & 1], slope[i & 1]);
  }
  const float2 s = Split(Add(sum[0], sum[1]));
  if (!kSlope) return make_float2(s.x + s.y, 0.0f);
  const float2 t = Split(Add(slope[0], slope[1]));
  return make_float2(s.x + s.y, t.x + t.y);
}

// What a thread knows of a longer row's vectors: the largest score, of all and of every fourth
// vector, and the sums of 2^d and d 2^d against it.
struct Sums {
  float high, group[4];
  Two sum, slope;
};
__device__ __forceinline__ Sums NoSums() {
  return {-INFINITY, {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, {0}, {0}};
}
// The sums so far, against a larger score.
template <bool kSlope>
__device__ __forceinline__ void Raise(Sums &s, float high, float k) {
  if (!(high > s.high)) return;
  const float d = fmaxf((s.high - high) * k, -1e30f), e = Exp2(d);
  const Two by = MakeTwo(e, e);
  if (kSlope) s.slope = Mul(by, Fma(s.sum, MakeTwo(d, d), s.slope));
  s.sum = Mul(s.sum, by);
  s.high = high;
}
// then(slot, i): called behind the last use of vector i.
template <bool kSlope, int kTeam, typename T, typename F>
__device__ __forceinline__ void AddRow(Sums &s, uint4 *slot, int32_t mine, const T *type, float k,
                                       const F &then) {
  int32_t i = 0;
#pragma unroll 1
  for (; i + 4 <= mine; i += 4) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      v[u] = slot[(i + u) * kTeam];
      s.group[u] = fmaxf(s.group[u], VectorMax(v[u], type));
    }
    Raise<kSlope>(s, fmaxf(fmaxf(s.group[0], s.group[1]), fmaxf(s.group[2], s.group[3])), k);
    const float from = s.high == -INFINITY ? 0.0f : s.high;
    Two sum = {0}, slope = {0};  // of every second vector
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      After(v[u], u & 1 ? sum : s.sum);
      AddVector<kSlope>(v[u], type, from, k, u & 1 ? sum : s.sum, u & 1 ? slope : s.slope);
    }
    s.sum = Add(s.sum, sum);
    if (kSlope) s.slope = Add(s.slope, slope);
#pragma unroll
    for (int u = 0; u < 4; ++u) then(slot, i + u);
  }
#pragma unroll 1
  for (; i < mine; ++i) {
    const uint4 v = slot[i * kTeam];
    const float high = VectorMax(v, type);
    // (as many groups as there are: a loop does not choose a register)
    s.group[0] = (i & 3) == 0 ? fmaxf(s.group[0], high) : s.group[0];
    s.group[1] = (i & 3) == 1 ? fmaxf(s.group[1], high) : s.group[1];
    s.group[2] = (i & 3) == 2 ? fmaxf(s.group[2], high) : s.group[2];
    Raise<kSlope>(s, high, k);
    AddVector<kSlope>(v, type, s.high == -INFINITY ? 0.0f : s.high, k, s.sum, s.slope);
    then(slot, i);
  }
}
// A slice [first, last) of a row's vectors as a team of `team` threads reads it from memory: the whole
// ones, and the ends that the row shares with its neighbours, which threads 0 and 1 have.
template <typename T>
struct RowStream {
  RowSpan<T> span;
  const uint4 *in;
  int32_t first, last, from, to;
  __device__ __forceinline__ RowStream(const RowSpan<T> &row, int32_t begin, int32_t end)
      : span(row), in(reinterpret_cast<const uint4 *>(row.row - row.shift)), first(begin),
        last(end) {
    from = first < last && !span.Whole(span.Column(first)) ? first + 1 : first;
    to = last > from && !span.Whole(span.Column(last - 1)) ? last - 1 : last;
  }
  // The vector at an end that this thread has, or -1.
  __device__ __forceinline__ int32_t End(int32_t tid) const {
    if (tid == 0 && from > first) return first;
    if (tid == 1 && to < last && last - 1 >= from) return last - 1;
    return -1;
  }
};
// f(x, count, j): up to four of a thread's vectors at a time, j the first of them and a team's
// width apart.
template <int kTeam, typename T, typename F>
__device__ __forceinline__ void EachFour(const RowStream<T> &s, int32_t tid, F &&f) {
#pragma unroll 1
  for (int32_t j = s.from + tid; j < s.to; j += 4 * kTeam) {
    uint4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (j + u * kTeam < s.to) x[u] = s.in[j + u * kTeam];
    f(x, min(4, (s.to - j + kTeam - 1) / kTeam), j);
  }
}
template <bool kSlope, int kTeam, typename T>
__device__ __forceinline__ Sums SumStream(const RowStream<T> &stream, int32_t tid, float k) {
  Sums s = NoSums();
  const T *type = stream.span.row;
  const auto one = [&](const uint4 &x, int u) {
    const float high = VectorMax(x, type);
    s.group[u] = fmaxf(s.group[u], high);
    Raise<kSlope>(s, high, k);
    AddVector<kSlope>(x, type, s.high == -INFINITY ? 0.0f : s.high, k, s.sum, s.slope);
  };
  EachFour<kTeam>(stream, tid, [&](uint4 (&x)[4], int32_t count, int32_t) {
    if (count == 4) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s.group[u] = fmaxf(s.group[u], VectorMax(x[u], type));
      Raise<kSlope>(s, fmaxf(fmaxf(s.group[0], s.group[1]), fmaxf(s.group[2], s.group[3])), k);
      const float from = s.high == -INFINITY ? 0.0f : s.high;
      Two sum = {0}, slope = {0};  // of every second vector
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        After(x[u], u & 1 ? sum : s.sum);
        AddVector<kSlope>(x[u], type, from, k, u & 1 ? sum : s.sum, u & 1 ? slope : s.slope);
      }
      s.sum = Add(s.sum, sum);
      if (kSlope) s.slope = Add(s.slope, slope);
    } else {
#pragma unroll
      for (int u = 0; u < 3; ++u)
        if (u < count) one(x[u], u);
    }
  });
  const int32_t end = stream.End(tid);
  if (end >= 0) one(stream.span.Edge(end), 3);
  return s;
}

// A warp's sums against its largest score.
template <bool kSlope>
__device__ __forceinline__ float2 WarpSums(const Sums &s, float k, float *high) {
  *high = WarpMaxF(s.high);
  const float from = *high == -INFINITY ? 0.0f : *high;
  const float d = (s.high - from) * k, e = Exp2(d);
  const float2 sum = Split(s.sum);
  if (!kSlope) return make_float2(WarpSumF((sum.x + sum.y) * e), 0.0f);
  const float2 slope = Split(s.slope);
  return WarpSum2F((sum.x + sum.y) * e,
                   e * fmaf(sum.x + sum.y, fmaxf(d, -1e30f), slope.x + slope.y));
}

// Values for the classes of vector j into another row of the same length; `aligned`: both rows
// begin at the same place of a vector.  They do not where scores are a slice of padded classes and
// the gradient is contiguous: one by one then, 73 us and not 60 for the distillation of 64000 x 500
// bf16 classes of 512.
template <typename T>
__device__ __forceinline__ void Store(T *out, const RowSpan<T> &span, bool aligned, int32_t j,
                                      const float (&f)[kPer<T>]) {
  const int32_t c0 = span.Column(j);
  if (aligned && span.Whole(c0)) {
    *reinterpret_cast<uint4 *>(out + c0) = Pack(f, out);
    return;
  }
  // (words where pairs of scores are aligned)
  if (aligned && kPer<T> == 8 && ((span.shift | span.classes) & 1) == 0) {
    const uint4 v = Pack(f, out);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c0 + 2 * k >= 0 && c0 + 2 * k < span.classes)
        *reinterpret_cast<uint32_t *>(out + c0 + 2 * k) = w[k];
    return;
  }
#pragma unroll
  for (int k = 0; k < kPer<T>; ++k)
    if (c0 + k >= 0 && c0 + k < span.classes) out[c0 + k] = FromFloat<T>(f[k]);
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

// ---------------------------------------------------------------------------
// teams
// ---------------------------------------------------------------------------
// Sums that the lanes have against a score of their own (-inf: none), against the largest of them.
__device__ __forceinline__ float2 JoinWarp(float h, float2 sums, float *high) {
  *high = WarpMaxF(h);
  const float d = (h - (*high == -INFINITY ? 0.0f : *high)) * kLog2e, e = Exp2(d);
  return WarpSum2F(sums.x * e, e * fmaf(sums.x, fmaxf(d, -1e30f), sums.y));
}

template <int kTeam>
__device__ __forceinline__ void TeamSync() {
  if (kTeam == 32) __syncwarp(); else __syncthreads();
}

// This block's place in its cluster (0 of 1 without one).
__device__ __forceinline__ uint32_t ClusterRank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t ClusterSize() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
// All threads of all blocks of the cluster; what was written to shared memory before is seen
// behind it.
__device__ __forceinline__ void ClusterSync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}
// A shared variable of this block, in block `rank` of the cluster.
template <typename V>
__device__ __forceinline__ V ReadFrom(const V *mine, uint32_t rank) {
  static_assert(sizeof(V) == 4 || sizeof(V) == 8, "4 or 8 bytes");
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(mine);
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  V v;
  if (sizeof(V) == 4) {
    uint32_t w;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(there) : "memory");
    memcpy(&v, &w, 4);
  } else {
    uint64_t w;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(w) : "r"(there) : "memory");
    memcpy(&v, &w, 8);
  }
  return v;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// How the rows of a call are dealt out.
struct RowPlan {
  int32_t team;       // threads per row and block: 32, 128, 256 or, in clusters, 512
  int32_t vectors;    // per thread: of a short row 1, 2, 4 or 8, which are registers; at most of others
  bool in_registers;
  int32_t cluster;    // blocks per row
  int32_t tiles;      // parts of a row that does not fit: read again for each pass
  int32_t block;      // threads of a block: a team, or several warps that are a team each
  int32_t ring;       // bytes of a block's rows
  int64_t blocks;     // what the device holds at a time, or what the rows need
};

// Blocks of an SM that the kernels for short rows are compiled for.
constexpr int ResidentBlocks(int vectors) { return vectors > 4 ? 6 : 8; }

// more_warp, more_block: bytes of shared memory that a team takes besides.
template <typename T>
static inline RowPlan PlanRows(const Rows<T> &r, int32_t more_warp, int32_t more_block) {
  RowPlan p = {32, 1, true, 1, 1, 32, 0, 0};
  const int64_t rows = r.count, size = sizeof(T);
  // its vectors: one more where it does not begin with one
  const bool whole = ((uintptr_t)r.scores | (uint64_t)(r.outer_stride * size) |
                      (uint64_t)(r.inner_stride * size)) % 16 == 0;
  const int64_t vectors = (r.classes * size + (whole ? 0 : 16 - size) + 15) / 16;
  const int32_t sms = NumSms();
  constexpr int64_t kShared = 224 << 10;  // of an SM
  int64_t fit;
  if (vectors <= 32 * 8) {
    while (vectors > 32 * p.vectors) p.vectors *= 2;
    p.block = 32 * (int32_t)std::min<int64_t>(4, std::max<int64_t>(1, rows / sms));
    fit = (int64_t)ResidentBlocks(p.vectors) * (128 / p.block);
  } else {
    p.in_registers = false;
    // What a team does once per row, each of its warps does: few threads and many vectors each, as
    // long as enough rows fit an SM.  bf16 rows of 160 MB in all, us with 16 top classes / of a
    // distillation, by threads to a row:
    //           32         128        256        512
    //   12 KB   64 /  76   81 / 122  121 / 188  199 / 352
    //   24      79 /  87   66 /  87   83 / 122  116 / 198
    //   48       -         57 /  75   66 /  86   77 / 132
    //   80       -         73 /  96   59 /  77   63 / 105
    if (vectors <= 32 * 36 && rows >= 4 * (int64_t)sms) {
      p.block = 128;
    } else {
      p.team = p.block = vectors <= 128 * 28 ? 128 : 256;
      // over more SMs: rows that do not fit one, and few rows, down to 8 KB each
      while (p.cluster < 8 && (vectors * 16 > p.cluster * kShared * 7 / 8 ||
                               (rows * p.cluster * 2 <= sms && vectors > p.cluster * 2 * 512))) {
        p.cluster *= 2;
        p.team = p.block = 512;
      }
    }
    const int64_t threads = (int64_t)p.cluster * p.team;
    int64_t each = (vectors + threads - 1) / threads;
    const int64_t most = kShared * 7 / 8 / 16 / p.team;
    p.tiles = (int32_t)((each + most - 1) / most);
    p.vectors = (int32_t)std::min(each, most);
    fit = 2048 / p.block;
  }
  const int64_t teams = p.block / p.team;
  p.ring = p.block * p.vectors * 16;
  fit = std::min(fit, kShared / (p.ring + (p.team == 32 ? more_warp * teams : more_block) + 1024));
  p.blocks = std::min<int64_t>((rows + teams - 1) / teams * p.cluster,
                               sms * std::max<int64_t>(1, fit) / p.cluster * p.cluster);
  return p;
}

// Lets a kernel have more shared memory than the 48 KB that it has without asking (of which the
// kernels here name up to 17 themselves).  The limit is the kernel's, whichever thread of the host
// sets it: every call sets the same one, for the longest ring of PlanRows with what a team has
// besides, so that none takes away what another one is about to launch with.
constexpr size_t kMostShared = 204 << 10;
template <typename... Params>
static cudaError_t AllowShared(void (*kernel)(Params...), size_t bytes) {
  if (bytes <= 30 << 10) return cudaSuccess;
  if (bytes > kMostShared) return cudaErrorInvalidValue;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)kMostShared);
}

// A launch of `blocks` blocks in clusters; `behind`: see LaunchBehind (common.cuh).
template <typename... Params, typename... Args>
static cudaError_t LaunchRows(void (*kernel)(Params...), int64_t blocks, int32_t threads,
                              size_t smem, int32_t cluster, bool behind, cudaStream_t stream,
                              Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((uint32_t)blocks);
  cfg.blockDim = dim3((uint32_t)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (uint32_t)cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (behind) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Whether an array of elements of `size` bytes, if there is one, lies as the device reads it.
static inline bool Aligned(const void *array, size_t size) { return (uintptr_t)array % size == 0; }
static inline size_t IntSize(int32_t is_64) { return is_64 ? 8 : 4; }
static inline size_t FloatSize(int32_t type) { return type == K2B200_F32 ? 4 : 2; }

// What the entry points ask of a k2b200_class_rows.
static inline int32_t CheckRows(const k2b200_class_rows *rows) {
  K2B_REQUIRE(rows != nullptr, "NULL pointer");
  K2B_REQUIRE(rows->type >= K2B200_F32 && rows->type <= K2B200_BF16, "unknown type %d",
              rows->type);
  K2B_REQUIRE(rows->num_classes > 0 && rows->num_classes <= kMaxClasses,
              "rows of %d classes: 1 to 2^30", rows->num_classes);
  // (blocks of a cluster count too: 8 to a row at most)
  K2B_REQUIRE(rows->outer >= 0 && rows->inner >= 0 && rows->outer < ((int64_t)1 << 28) &&
                  rows->inner < ((int64_t)1 << 28) &&
                  rows->outer * rows->inner < ((int64_t)1 << 28),
              "%lld x %lld rows: fewer than 2^28", (long long)rows->outer,
              (long long)rows->inner);
  K2B_REQUIRE(rows->scores != nullptr || rows->outer * rows->inner == 0, "NULL pointer");
  K2B_REQUIRE(Aligned(rows->scores, FloatSize(rows->type)) &&
                  Aligned(rows->lengths, IntSize(rows->lengths_64)),
              "scores or lengths that are not aligned to their type");
  return kOk;
}

template <typename T>
static inline Rows<T> RowsOf(const k2b200_class_rows *rows) {
  Rows<T> r;
  r.scores = static_cast<const T *>(rows->scores);
  r.classes = rows->num_classes;
  r.count = (int32_t)(rows->outer * rows->inner);
  r.inner = (uint32_t)std::max<int64_t>(1, rows->inner);
  // with 2^28 times the next power of two over it, r * the error of the quotient stays below 1
  r.shift = 28;
  while ((1u << (r.shift - 28)) < r.inner) ++r.shift;
  r.inverse = (uint32_t)((((uint64_t)1 << r.shift) + r.inner - 1) / r.inner);
  r.begin = r.end = r.scores;
  for (int64_t o : {(int64_t)0, rows->outer - 1})
    for (int64_t i : {(int64_t)0, rows->inner - 1}) {
      const T *x = r.scores + o * rows->outer_stride + i * rows->inner_stride;
      r.begin = std::min(r.begin, x);
      r.end = std::max(r.end, x + r.classes);
    }
  r.outer_stride = rows->outer_stride;
  r.inner_stride = rows->inner_stride;
  r.lengths = rows->lengths;
  r.lengths_64 = rows->lengths_64;
  return r;
}

}  // namespace k2b
