// Rows of class scores as the kernels of token_scores.cu and distillation.cu hold them.
//
// A row is read once, as aligned vectors of 16 bytes, into the registers of a team of threads: a
// warp up to 4 KB, 128 threads up to 16, 256 up to 64, and a cluster of up to 8 such blocks up to
// 512.  Where the row begins inside a vector (any alignment of an element will do) the elements of
// the first and the last vector are read one by one, and what lies outside the row is -inf there.
// What a kernel needs of the row more than once it takes from the registers.  Longer rows are read
// again, tile by tile.
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

// 2^x, off by at most 2 units of the last place and 0 below 2^-126.
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
    return Packed(f);  // (exact)
  }
  __device__ __forceinline__ uint4 Vector(int32_t j) const {
    const int32_t c0 = Column(j);
    return Whole(c0) ? *reinterpret_cast<const uint4 *>(row + c0) : Edge(j);
  }
  __device__ __forceinline__ static uint4 Packed(const float (&f)[kPer<T>]) {
    uint4 v = Pack(f, static_cast<const T *>(nullptr));
    return k2b::Packed(v);
  }
};

// Elements [begin, end) of a vector, -inf elsewhere.
__device__ __forceinline__ uint4 Keep(const uint4 &v, int32_t begin, int32_t end, const float *t) {
  const uint4 low = LowestVector(t);
  return make_uint4(begin <= 0 && end > 0 ? v.x : low.x, begin <= 1 && end > 1 ? v.y : low.y,
                    begin <= 2 && end > 2 ? v.z : low.z, begin <= 3 && end > 3 ? v.w : low.w);
}
template <typename T>
__device__ __forceinline__ uint4 Keep(const uint4 &v, int32_t begin, int32_t end, const T *t) {
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

// Vectors tile + i * kTeam + tid for i < kVectors of those before `last`.  A vector that the row
// shares with others is read as a whole where all of it lies between the first and the last class
// of all rows, and element by element elsewhere.
template <int kTeam, int kVectors, typename T>
__device__ __forceinline__ void LoadTile(uint4 (&v)[kVectors], const RowSpan<T> &span,
                                         const Rows<T> &rows, int32_t tile, int32_t last,
                                         int32_t tid) {
  const int32_t end = span.vectors - 1, rest = span.classes - span.Column(end);
  const uint4 *at = reinterpret_cast<const uint4 *>(span.row - span.shift);
  const bool front = span.shift != 0 && tile == 0,
             tail = rest < kPer<T> && end >= tile && end < min(last, tile + kTeam * kVectors);
  if ((!front || reinterpret_cast<const T *>(at) >= rows.begin) &&
      (!tail || reinterpret_cast<const T *>(at + span.vectors) <= rows.end)) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int32_t j = tile + i * kTeam + tid;
      v[i] = j < last ? at[j] : LowestVector(span.row);
    }
    if (front && tid == 0) v[0] = Keep(v[0], span.shift, kPer<T>, span.row);
    if (tail) {
      const int32_t slot = (end - tile) / kTeam;
      const bool mine = ((end - tile) & (kTeam - 1)) == tid;
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
        if (i == slot) {
          const uint4 kept = Keep(v[i], 0, rest, span.row);
          if (mine) v[i] = kept;
        }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int32_t j = tile + i * kTeam + tid;
      v[i] = j < last && span.Whole(span.Column(j)) ? at[j] : LowestVector(span.row);
    }
#pragma unroll 1
    for (int32_t both = 0; both < 2; ++both) {
      const int32_t j = both ? end : 0;
      if (j < tile || j >= min(last, tile + kTeam * kVectors) ||
          ((j - tile) & (kTeam - 1)) != tid || span.Whole(span.Column(j)))
        continue;
      const uint4 e = span.Edge(j);
      const int32_t slot = (j - tile) / kTeam;
#pragma unroll
      for (int i = 0; i < kVectors; ++i)
        if (i == slot) v[i] = e;
    }
  }
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

// Values for the classes of vector j into another row of the same length; `aligned`: both rows
// begin at the same place of a vector.
template <typename T>
__device__ __forceinline__ void Store(T *out, const RowSpan<T> &span, bool aligned, int32_t j,
                                      const float (&f)[kPer<T>]) {
  const int32_t c0 = span.Column(j);
  if (aligned && span.Whole(c0)) {
    *reinterpret_cast<uint4 *>(out + c0) = Pack(f, out);
    return;
  }
#pragma unroll
  for (int k = 0; k < kPer<T>; ++k)
    if (c0 + k >= 0 && c0 + k < span.classes) out[c0 + k] = FromFloat<T>(f[k]);
}

// ---------------------------------------------------------------------------
// teams
// ---------------------------------------------------------------------------
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

// Blocks of an SM that a kernel is compiled for: the registers are the row's and some 40 more.
constexpr int MinBlocks(int team, int vectors) {
  return (vectors >= 16 ? 2 : vectors >= 8 ? 3 : 4) * (team == 128 ? 2 : 1);
}

// Adds sums of 2^d and d 2^d whose d is by `by` * log2 e too high (-inf: there are none).
__device__ __forceinline__ void Join(float &sum, float &slope, float more, float more_slope,
                                     float by) {
  const float d = by * kLog2e, e = Exp2(d);
  sum = fmaf(more, e, sum);
  slope = fmaf(e, fmaf(more, fmaxf(d, -1e30f), more_slope), slope);
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
  int32_t team;     // threads per row and block: 32, 128, 256
  int32_t vectors;  // per thread
  int32_t cluster;  // blocks per row
  bool again;       // the row does not fit and is read again
  int32_t block;    // threads of a block: `team`, or several warps that are a team each
  int32_t rows_per_warp, rows_per_block;
};

template <typename T>
static inline RowPlan PlanRows(const Rows<T> &r) {
  RowPlan p = {32, 1, 1, false, 32, 1, 1};
  const int64_t rows = r.count, size = sizeof(T);
  // its vectors: one more where it does not begin with one
  const bool whole = ((uintptr_t)r.scores | (uint64_t)(r.outer_stride * size) |
                      (uint64_t)(r.inner_stride * size)) % 16 == 0;
  const int64_t bytes = r.classes * size + (whole ? 0 : 16 - size);
  const int32_t sms = NumSms();
  if (bytes <= 32 * 8 * 16) {
    while (bytes > 32 * 16 * p.vectors) p.vectors *= 2;
    // few rows: one to a warp, and warps to as many SMs as there are; many: four to a warp
    p.rows_per_warp = rows >= 16 * 4 * (int64_t)sms ? 4 : 1;
    p.block = 32 * (int32_t)std::min<int64_t>(4, std::max<int64_t>(1, rows / sms));
    p.rows_per_block = p.block / 32 * p.rows_per_warp;
    return p;
  }
  p.team = p.block = bytes <= 128 * 8 * 16 ? 128 : 256;
  if (p.team == 128) {
    p.vectors = bytes <= 128 * 4 * 16 ? 4 : 8;
    return p;
  }
  while (p.cluster < 8 && bytes > (int64_t)p.cluster * 256 * 16 * 16) p.cluster *= 2;
  // few rows: over more SMs, down to 8 KB of the row each
  while (p.cluster < 8 && rows * p.cluster * 2 <= sms && bytes > (int64_t)p.cluster * 2 * 8192)
    p.cluster *= 2;
  p.vectors = 4;
  while (p.vectors < 16 && bytes > (int64_t)p.cluster * 256 * 16 * p.vectors) p.vectors *= 2;
  p.again = bytes > (int64_t)p.cluster * 256 * 16 * p.vectors;
  return p;
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
