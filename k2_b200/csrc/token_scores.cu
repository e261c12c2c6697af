// Log-probs of given classes, entropies and top classes of rows of scores, and their gradient.
//
// With d_c = (x_c - high) log2 e and e_c = 2^d_c: log p_c = (x_c - high) - ln sum e, and the entropy is
// ln sum e - ln 2 (sum e d) / sum e.  Top classes: the threads' largest scores are themselves scores of
// the row, so that the k-th largest of them bounds the row's k-th largest from below, and few scores
// lie above it (of n threads about n ln(n / (n - k))) while k is well below n; those are collected in
// shared memory, and each one's place is the number of larger ones.  Where more lie above it than
// there is room for - ties, many large scores in one thread, or a k near n (TokenWarps has 64 groups
// of scores, TokenRing 128 or 256) - the bound is raised by bisection over (score, class), which no
// two classes share, from scores that are read again.  64000 rows of 500 bf16 classes: 57 us with 8
// top classes, 122 with 32, 306 with 48, 629 with 64, 858 with 65 to 128, cold.
//
// Kernels, by the length of a row (PlanRows): TokenWarps up to 4 KB, TokenRing with a warp per row up
// to 18 KB, then with blocks where top classes are asked for, and TokenStream where not; few long rows
// are dealt out to clusters.  TokenWarpsBackward and TokenBlocksBackward for the gradient.
#include "class_rows.cuh"

#include <type_traits>

namespace k2b {

struct TokenOut {
  const void *tokens;
  int32_t tokens_64, top_k, room;  // room: keys per team
  float *log_probs, *entropy, *top_log_probs;
  int32_t *top_tokens;
  float4 *norm;
};

// Keys that a team has room for: what lies above the bound, with some to spare.
static inline int32_t RoomFor(int32_t top_k) {
  return top_k == 0 ? 0 : top_k <= 8 ? 32 : top_k <= 16 ? 64 : top_k <= 32 ? 96
                                          : top_k <= 64 ? 160
                                                        : 288;
}

constexpr uint32_t kOrderOfNone = 0x007fffffu;  // OrderOf(-inf)

// The largest bound found that at least k of a warp's kGroups values per lane reach, where there
// are so many; -inf else.  By bisection, until no more than an eighth too many reach it.
template <int kGroups>
__device__ __forceinline__ uint32_t BoundOf(const uint32_t (&order)[kGroups], int32_t k) {
  uint32_t least = order[0], most = order[0];
#pragma unroll
  for (int g = 1; g < kGroups; ++g) {
    least = min(least, order[g]);
    most = max(most, order[g]);
  }
  if (k > 32 * kGroups) return kOrderOfNone;
  uint32_t low = __reduce_min_sync(0xffffffffu, least);
  uint32_t high = __reduce_max_sync(0xffffffffu, most) + 1;  // (NaN is not among them)
  while (high - low > 1) {
    const uint32_t mid = low + (high - low) / 2;
    int32_t reach = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) reach += __popc(__ballot_sync(0xffffffffu, order[g] >= mid));
    if (reach >= k) {
      low = mid;
      if (reach <= k + (k >> 3)) break;
    } else {
      high = mid;
    }
  }
  return low;
}

// The keys that a team collects: score and class in one number (OrderOf), which sorts as they do.
// A warp's rows have at most 32 * 36 * 8 classes, so that with a score of 16 bits a key is one of 32.
template <typename T, int kTeam>
struct Keys {
  using Key = uint64_t;
  __device__ __forceinline__ static Key Make(T x, int32_t c) { return KeyOf(ToFloat(x), c); }
  __device__ __forceinline__ static Key From(uint64_t key) { return key; }
  __device__ __forceinline__ static float Score(Key key) { return ScoreOf((uint32_t)(key >> 32)); }
  __device__ __forceinline__ static int32_t Class(Key key) { return (int32_t)~(uint32_t)key; }
};
struct ShortKeys {
  using Key = uint32_t;
  __device__ __forceinline__ static Key Make(uint32_t bits, uint32_t infinity, int32_t c) {
    uint32_t order = bits & 0x8000u ? ~bits & 0xffffu : bits | 0x8000u;
    if (bits == 0x8000u) order = 0x8000u;              // -0 is 0
    if ((bits & 0x7fffu) > infinity) order = 0xffffu;  // NaN
    return order << 16 | (~(uint32_t)c & 0xffffu);
  }
  __device__ __forceinline__ static uint16_t Bits(Key key) {
    return (uint16_t)(key & 0x80000000u ? key >> 16 & 0x7fffu : ~(key >> 16));
  }
  __device__ __forceinline__ static int32_t Class(Key key) { return (int32_t)(~key & 0xffffu); }
};
template <>
struct Keys<__half, 32> : ShortKeys {
  __device__ __forceinline__ static Key Make(__half x, int32_t c) {
    return ShortKeys::Make(__half_as_ushort(x), 0x7c00u, c);
  }
  __device__ __forceinline__ static Key From(uint64_t key) {
    return Make(__float2half_rn(ScoreOf((uint32_t)(key >> 32))), (int32_t)~(uint32_t)key);
  }
  __device__ __forceinline__ static float Score(Key key) {
    return __half2float(__ushort_as_half(Bits(key)));
  }
};
template <>
struct Keys<__nv_bfloat16, 32> : ShortKeys {
  __device__ __forceinline__ static Key Make(__nv_bfloat16 x, int32_t c) {
    return ShortKeys::Make(__bfloat16_as_ushort(x), 0x7f80u, c);
  }
  __device__ __forceinline__ static Key From(uint64_t key) {
    return Make(__float2bfloat16_rn(ScoreOf((uint32_t)(key >> 32))), (int32_t)~(uint32_t)key);
  }
  __device__ __forceinline__ static float Score(Key key) {
    return __uint_as_float((uint32_t)Bits(key) << 16);
  }
};

// Bit e is set where score e of a vector is not below `least` (NaN is not).
__device__ __forceinline__ uint32_t Reaching(const uint4 &v, float least, const float *) {
  return (!(__uint_as_float(v.x) < least) ? 1u : 0u) | (!(__uint_as_float(v.y) < least) ? 2u : 0u) |
         (!(__uint_as_float(v.z) < least) ? 4u : 0u) | (!(__uint_as_float(v.w) < least) ? 8u : 0u);
}
template <typename Pair>
__device__ __forceinline__ uint32_t ReachingPairs(const uint4 &v, Pair least) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    Pair p;
    memcpy(&p, &w[k], 4);
    // all bits of a half that reaches: of the low one bit 2k, of the high one bit 16 + 2k + 1
    bits |= __hgeu2_mask(p, least) & ((1u << 2 * k) | (1u << (17 + 2 * k)));
  }
  return (bits | bits >> 16) & 0xff;
}
__device__ __forceinline__ uint32_t Reaching(const uint4 &v, float least, const __half *) {
  return ReachingPairs(v, __half2half2(__float2half_rd(least)));
}
__device__ __forceinline__ uint32_t Reaching(const uint4 &v, float least, const __nv_bfloat16 *) {
  return ReachingPairs(v, __bfloat162bfloat162(__float2bfloat16_rd(least)));
}

// One more of what a team counts in shared memory; few lanes come here at a time, so that nothing is
// gained by adding theirs up first.
__device__ __forceinline__ int32_t Count(int32_t *found) {
  int32_t at;
  asm volatile("atom.shared.add.u32 %0, [%1], 1;"
               : "=r"(at)
               : "r"((uint32_t)__cvta_generic_to_shared(found))
               : "memory");
  return at;
}

// Puts the key of each score whose bit is set, of vectors i0 on, where there is room, and counts them
// all.
template <int kTeam, typename T, typename Key>
__device__ __forceinline__ void PutKeys(uint32_t bits, const uint4 *slot, const RowPart<T> &part,
                                        int32_t i0, Key *keys, int32_t room, int32_t *found) {
  while (bits) {
    const int32_t bit = __ffs(bits) - 1, i = i0 + bit / kPer<T>, e = bit % kPer<T>;
    bits &= bits - 1;
    const int32_t c = part.span.Column(part.first + i * kTeam) + e;
    // (beside the row there is nothing but -inf)
    if (i >= part.mine || c < 0 || c >= part.span.classes) continue;
    const int32_t at = Count(found);
    if (at < room)
      keys[at] = Keys<T, kTeam>::Make(reinterpret_cast<const T *>(slot + i * kTeam)[e], c);
  }
}

// The keys of a thread's scores that reach `least`: of vectors in registers (a score is told by its
// bit, but no register by a number: it is read from shared memory) ...
template <int kTeam, int kVectors, typename T, typename Key>
__device__ __forceinline__ void Collect(uint4 (&v)[kVectors], const uint4 *slot,
                                        const RowPart<T> &part, float least, Key *keys,
                                        int32_t room, int32_t *found) {
  constexpr int kWord = 32 / kPer<T>;  // vectors to a word of bits
#pragma unroll
  for (int i0 = 0; i0 < kVectors; i0 += kWord) {
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < kWord && i0 + u < kVectors; ++u)
      bits |= Reaching(Packed(v[i0 + u]), least, part.span.row) << (u * kPer<T>);
    PutKeys<kTeam>(bits, slot, part, i0, keys, room, found);
  }
}
// ... and of vectors in shared memory.
template <int kTeam, typename T, typename Key, typename F>
__device__ __forceinline__ void CollectRow(uint4 *slot, const RowPart<T> &part, float least,
                                           Key *keys, int32_t room, int32_t *found,
                                           const F &then) {
  constexpr int kWord = 32 / kPer<T>;
#pragma unroll 1
  for (int32_t i0 = 0; i0 < part.most; i0 += kWord) {
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < kWord; ++u)
      if (i0 + u < part.most)
        bits |= Reaching(slot[(i0 + u) * kTeam], least, part.span.row) << (u * kPer<T>);
    PutKeys<kTeam>(bits, slot, part, i0, keys, room, found);
#pragma unroll
    for (int u = 0; u < kWord; ++u)
      if (i0 + u < part.most) then(slot, i0 + u);
  }
}

// Keys of a row's classes [first, last) vectors by a team, read from memory: of those that reach
// `bound` the number, or each of them.
template <int kTeam, typename T, typename F>
__device__ __forceinline__ void EachKey(const RowSpan<T> &span, int32_t first, int32_t last,
                                        int32_t tid, uint64_t bound, F &&f) {
  for (int32_t j = first + tid; j < last; j += kTeam) {
    float x[kPer<T>];
    Unpack(span.Vector(j), x, span.row);
#pragma unroll
    for (int k = 0; k < kPer<T>; ++k) {
      const int32_t c = span.Column(j) + k;
      const uint64_t key = KeyOf(x[k], c);
      if (key >= bound && c >= 0 && c < span.classes) f(key);
    }
  }
}

// A bound that at least top_k and at most `room` keys reach, where too many reach `bound`: ties, or
// large scores side by side.  By bisection over score and class; no two keys are equal, so there is
// one.  count(key): how many of the team's row reach a key.
template <typename F>
__device__ __forceinline__ uint64_t RaiseBound(uint64_t bound, int32_t top_k, int32_t room,
                                               int32_t classes, F &&count) {
  uint64_t low = bound, far = ~0ull, mid = bound + (1ull << 32);
  // (halved 64 times at most; the limit is for scores that somebody else changes meanwhile)
  for (int32_t k = 0; k < 128; ++k) {
    const int32_t n = count(mid);
    if (n >= top_k && n <= room) return mid;
    if (n < top_k) far = mid; else low = mid;
    // between keys of one score there are the classes
    if ((far - 1) >> 32 == low >> 32)
      low = max((unsigned long long)low, (low | 0xffffffffull) - (uint64_t)classes);
    mid = low + (far - low) / 2;
  }
  return mid;
}
// Puts a key where there is room, as there is for all that reach such a bound.
template <typename Key>
__device__ __forceinline__ void PutKey(Key key, Key *keys, int32_t room, int32_t *found) {
  const int32_t at = Count(found);
  if (at < room) keys[at] = key;
}

template <typename K>
__device__ __forceinline__ void WriteTop(const TokenOut &out, int32_t r, int32_t place,
                                         typename K::Key key, float high, float sum,
                                         float log_sum) {
  const int64_t at = (int64_t)r * out.top_k + place;
  out.top_tokens[at] = K::Class(key);
  out.top_log_probs[at] = sum == 0.0f ? -INFINITY : (K::Score(key) - high) - log_sum;
}

// The values that a row has one of.
__device__ __forceinline__ void Finish(const TokenOut &out, int32_t r, int32_t classes,
                                       int64_t token, float score, float high, float sum,
                                       float slope) {
  const float log_sum = logf(sum);
  const float h = sum == 0.0f ? 0.0f : log_sum - slope * kLn2 / sum;
  if (out.entropy) out.entropy[r] = h;
  if (out.norm) out.norm[r] = make_float4(high, sum, h, 0.0f);
  if (out.log_probs)
    out.log_probs[r] = token == -1                     ? 0.0f
                       : token < 0 || token >= classes ? NAN
                       : sum == 0.0f                   ? -INFINITY
                                                       : (score - high) - log_sum;
}

// What does not count: log-probs and entropy 0, no classes.
__device__ __forceinline__ void SkipRow(const TokenOut &out, int32_t r) {
  if (out.log_probs) out.log_probs[r] = 0.0f;
  if (out.entropy) out.entropy[r] = 0.0f;
  if (out.norm) out.norm[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}
__device__ __forceinline__ void SkipTop(const TokenOut &out, int32_t r, int32_t tid,
                                        int32_t team) {
  for (int32_t k = tid; k < out.top_k; k += team) {
    out.top_log_probs[(int64_t)r * out.top_k + k] = 0.0f;
    out.top_tokens[(int64_t)r * out.top_k + k] = -1;
  }
}

// f(place, key) for the places of n keys among them, by counting the larger ones: a warp, two keys to
// a lane at a time.
template <typename Key, typename F>
__device__ __forceinline__ void EachPlaceWarp(const Key *keys, int32_t n, int32_t lane, F &&f) {
  for (int32_t k = lane; k < n; k += 64) {
    const Key a = keys[k];
    int32_t place = 0;
    if (n <= 32) {
#pragma unroll 4
      for (int32_t o = 0; o < n; ++o) place += keys[o] > a;
      f(place, a);
      continue;
    }
    const bool two = k + 32 < n;
    const Key b = two ? keys[k + 32] : a;
    int32_t other = 0;
#pragma unroll 4
    for (int32_t o = 0; o < n; ++o) {
      const Key key = keys[o];
      place += key > a;
      other += key > b;
    }
    f(place, a);
    if (two) f(other, b);
  }
}
// ... or a block, several threads to a key where there are many (places: room for n numbers).
template <int kTeam, typename F>
__device__ __forceinline__ void EachPlaceBlock(const uint64_t *keys, int32_t n, int32_t *places,
                                               int32_t tid, F &&f) {
  constexpr int kParts = kTeam / 128;
  if (n <= 32) {
    if (tid < 32) EachPlaceWarp(keys, n, tid, f);
    return;
  }
  for (int32_t k = tid; k < n; k += kTeam) places[k] = 0;
  __syncthreads();
  for (int32_t k = tid & 127; k < n; k += 128) {
    const uint64_t key = keys[k];
    int32_t place = 0;
#pragma unroll 4
    for (int32_t o = tid >> 7; o < n; o += kParts) place += keys[o] > key;
    atomicAdd(&places[k], place);
  }
  __syncthreads();
  for (int32_t k = tid; k < n; k += kTeam) f(places[k], keys[k]);
}

// Short rows: each warp is a team.  It takes 32 rows at a time, a whole grid of warps apart; lane q
// knows where the q-th of them is and its given class, gathers its sums, and computes what a row
// has one of, for all of them at once.  Bound by instructions: of 64 x 1000 rows of 500 bf16 classes,
// a fifth of them beyond their lengths, 46 us for log-probs, entropy and 8 top classes (600
// instructions a row, 340 of them for the top classes; three quarters of the issue slots), 1.2 TB/s.
template <typename T, int kVectors, bool kTop>
__global__ void __launch_bounds__(128, ResidentBlocks(kVectors))
TokenWarps(Rows<T> rows, TokenOut out) {
  extern __shared__ uint4 shared[];
  __shared__ int32_t all_found[4];
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  using K = Keys<T, 32>;
  // (with top classes two rows, since the one at hand is read again)
  constexpr int32_t kStage = 32 * kVectors, kRows = kTop ? 2 : 1;
  uint4 *const ring = shared + warp * kRows * kStage + lane;
  typename K::Key *keys =
      reinterpret_cast<typename K::Key *>(shared + warps * kRows * kStage) + warp * out.room;
  const int32_t apart = (int32_t)gridDim.x * warps;
  const bool slopes = out.entropy != nullptr;
  for (int32_t base = (int32_t)blockIdx.x * warps + warp; base < rows.count; base += 32 * apart) {
    const int32_t mine = base + lane * apart,
                  taken = min(32, (rows.count - base + apart - 1) / apart);
    const T *my_row = nullptr;
    int64_t token = -1;
    float score = 0.0f, my_high = 0.0f, my_sum = 0.0f, my_slope = 0.0f;
    if (lane < taken) {
      const RowPlace at = PlaceOf(rows, mine);
      if (at.counts) {
        my_row = rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride;
        if (out.log_probs) {
          token = IntAt(out.tokens, out.tokens_64, mine);
          if (token >= 0 && token < rows.classes) score = ToFloat(my_row[token]);
        }
      }
    }
    const auto row_of = [&](int32_t q) {
      return reinterpret_cast<const T *>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_row), q & 31));
    };
    const T *next = row_of(0);
    if (next != nullptr) {
      const RowSpan<T> span(next, rows.classes);
      SendFor<32, kVectors>(ring, RowPart<T>(span, 0, span.vectors, lane, 32), rows);
    }
    for (int32_t q = 0; q < taken; ++q) {
      const T *row = next;
      const RowSpan<T> span(row, rows.classes);
      const RowPart<T> part(span, 0, span.vectors, lane, 32);
      uint4 *const slot = ring + (kRows > 1 ? q & 1 : 0) * kStage,
                   *const other = ring + (kRows > 1 ? ~q & 1 : 0) * kStage;
      uint4 v[kVectors];
      if (row != nullptr) {
        WaitForAll();
        CutEnds<32>(slot, part);
        Take<32, kVectors>(v, slot, part);
      }
      next = row_of(q + 1);
      if (q + 1 < taken && next != nullptr) {
        const RowSpan<T> coming(next, rows.classes);
        SendFor<32, kVectors>(other, RowPart<T>(coming, 0, coming.vectors, lane, 32), rows);
      }
      if (row == nullptr) {
        if (kTop) SkipTop(out, base + q * apart, lane, 32);
        continue;
      }
      const float2 half = Highest(v, row);
      const float high = WarpMaxF(fmaxf(half.x, half.y)), from = high == -INFINITY ? 0.0f : high;
      float2 both;
      if (slopes) {
        const float2 s = SumUp<true>(v, row, from, kLog2e);
        both = WarpSum2F(s.x, s.y);
      } else {
        both = make_float2(WarpSumF(SumUp<false>(v, row, from, kLog2e).x), 0.0f);
      }
      const float sum = both.x;
      if (lane == q) {
        my_high = from;
        my_sum = sum;
        my_slope = both.y;
      }
      if (kTop) {
        float least;
        if (out.top_k <= 16) {
          // the k-th of the lanes' largest: take away the largest k times, whoever has it
          float left = fmaxf(half.x, half.y);
          least = high;
          for (int32_t k = 1; k < out.top_k; ++k) {
            if (left == least) left = -INFINITY;
            least = WarpMaxF(left);
          }
        } else {
          const uint32_t two[2] = {OrderOf(half.x), OrderOf(half.y)};
          least = ScoreOf(BoundOf(two, out.top_k));
        }
        if (lane == 0) all_found[warp] = 0;
        __syncwarp();  // (and the keys of the row before have been read)
        Collect<32>(v, slot, part, least, keys, out.room, &all_found[warp]);
        __syncwarp();
        int32_t found = all_found[warp];
        if (found > out.room) {
          const uint64_t bound = RaiseBound(
              (uint64_t)OrderOf(least) << 32, out.top_k, out.room, span.classes,
              [&](uint64_t key) {
                int32_t n = 0;
                EachKey<32>(span, 0, span.vectors, lane, key, [&](uint64_t) { ++n; });
                return (int32_t)__reduce_add_sync(0xffffffffu, n);
              });
          __syncwarp();
          if (lane == 0) all_found[warp] = 0;
          __syncwarp();
          EachKey<32>(span, 0, span.vectors, lane, bound,
                      [&](uint64_t key) {
                        PutKey(K::From(key), keys, out.room, &all_found[warp]);
                      });
          __syncwarp();
          found = min(all_found[warp], out.room);
        }
        const float log_sum = logf(sum);
        EachPlaceWarp(keys, found, lane, [&](int32_t place, typename K::Key key) {
          if (place < out.top_k)
            WriteTop<K>(out, base + q * apart, place, key, from, sum, log_sum);
        });
      }
    }
    if (lane < taken) {
      if (my_row != nullptr)
        Finish(out, mine, rows.classes, token, score, my_high, my_sum, my_slope);
      else
        SkipRow(out, mine);
    }
  }
}

template <int kTeam>
struct TokenShared {
  float high[2][kTeam / 32];
  float2 sums[2][kTeam / 32];
  int32_t counted[kTeam / 32];
  int32_t found;
  uint32_t bound;
  float all_high;  // of a block, for its cluster
  float2 all_sums;
  float group[kTeam == 32 ? 1 : kTeam];
  int32_t places[kTeam == 32 ? 1 : 288];  // RoomFor(K2B200_MAX_TOP)
};

// The keys that the blocks of a cluster show each other.
struct TokenTogether {
  int32_t top;                    // keys in `list`
  uint64_t list[K2B200_MAX_TOP];  // this block's, largest first
  uint64_t lists[8][K2B200_MAX_TOP];
  int32_t tops[8];
};

// The places of a row's keys where the blocks of a cluster have been through a slice each: every
// block finds those of its own, a thread for each of them and each list.
__device__ __forceinline__ void PlaceTogether(const TokenOut &out, TokenTogether &together,
                                              int32_t *places, int32_t top_k, int32_t r,
                                              uint32_t cluster, int32_t tid, int32_t team,
                                              float high, float sum) {
  using K = Keys<float, 512>;
  const float log_sum = logf(sum);
  if (tid < (int32_t)cluster) together.tops[tid] = ReadFrom(&together.top, tid);
  for (int32_t k = tid; k < top_k; k += team) places[k] = 0;
  __syncthreads();
  for (int32_t k = tid; k < (int32_t)cluster * K2B200_MAX_TOP; k += team) {
    const int32_t b = k / K2B200_MAX_TOP, at = k % K2B200_MAX_TOP;
    if (at < together.tops[b]) together.lists[b][at] = ReadFrom(&together.list[at], b);
  }
  __syncthreads();
  for (int32_t k = tid; k < (int32_t)cluster * K2B200_MAX_TOP; k += team) {
    const int32_t b = k / K2B200_MAX_TOP, at = k % K2B200_MAX_TOP;
    if (at >= top_k) continue;
    const uint64_t key = together.list[at];
    // how many of a list that falls are larger
    int32_t low = 0, far = together.tops[b];
    while (low < far) {
      const int32_t mid = (low + far) / 2;
      if (together.lists[b][mid] > key) low = mid + 1; else far = mid;
    }
    if (low > 0) atomicAdd(&places[at], low);
  }
  __syncthreads();
  for (int32_t k = tid; k < top_k; k += team)
    if (places[k] < out.top_k)
      WriteTop<K>(out, r, places[k], together.list[k], high, sum, log_sum);
}

// Longer rows without top classes: a block is a team, or a cluster of blocks (kTeam 512); one pass over
// the memory, without a copy of the row.  4096 x 32001 bf16 with entropy: 63 us, 4.2 TB/s, with 65% of
// the issue slots and 58% of what 2^d can do (10 instructions and one 2^d per score); without entropy
// 6666 x 12000 take 32 us, 5.1 TB/s.
template <typename T, int kTeam>
__global__ void __launch_bounds__(kTeam, kTeam == 512 ? 2 : 1280 / kTeam)
TokenStream(Rows<T> rows, TokenOut out) {
  __shared__ TokenShared<kTeam> sh;
  const int32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t cluster = kTeam == 512 ? ClusterSize() : 1,
                 rank = kTeam == 512 ? ClusterRank() : 0;
  const int32_t r = (int32_t)(blockIdx.x / cluster);
  const RowPlace at = PlaceOf(rows, r);
  if (!at.counts) {
    if (rank == 0 && tid == 0) SkipRow(out, r);
    return;  // (all blocks of the cluster)
  }
  const RowSpan<T> span(rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride,
                        rows.classes);
  const int32_t slice = (span.vectors + (int32_t)cluster - 1) / (int32_t)cluster;
  const int32_t first = min(span.vectors, (int32_t)rank * slice);
  const RowStream<T> stream(span, first, min(span.vectors, first + slice));
  int64_t token = -1;
  float score = 0.0f;
  if (out.log_probs && rank == 0 && tid == 0) {
    token = IntAt(out.tokens, out.tokens_64, r);
    if (token >= 0 && token < rows.classes) score = ToFloat(span.row[token]);
  }
  float high;
  float2 both =
      out.entropy
          ? WarpSums<true>(SumStream<true, kTeam>(stream, tid, kLog2e), kLog2e, &high)
          : WarpSums<false>(SumStream<false, kTeam>(stream, tid, kLog2e), kLog2e, &high);
  if (lane == 0) {
    sh.high[0][warp] = high;
    sh.sums[0][warp] = both;
  }
  __syncthreads();
  if (warp > 0 && cluster == 1) return;
  const bool one = lane < kTeam / 32;
  both = JoinWarp(one ? sh.high[0][lane] : -INFINITY,
                  one ? sh.sums[0][lane] : make_float2(0.0f, 0.0f), &high);
  if (cluster > 1) {
    if (tid == 0) {
      sh.all_high = high;
      sh.all_sums = both;
    }
    ClusterSync();
    const bool other = lane < (int32_t)cluster;
    if (rank == 0 && warp == 0) {
      const float h = other ? ReadFrom(&sh.all_high, lane) : -INFINITY;
      const float2 part = other ? ReadFrom(&sh.all_sums, lane) : make_float2(0.0f, 0.0f);
      both = JoinWarp(h, part, &high);
    }
    ClusterSync();  // nobody leaves while others read its memory
  }
  if (rank == 0 && tid == 0)
    Finish(out, r, rows.classes, token, score, high == -INFINITY ? 0.0f : high, both.x, both.y);
}

// Longer rows: a warp (kTeam 32, several to a block) or a block is a team, or a cluster of blocks
// (kTeam 512), to which a row's vectors are dealt out in slices.  Rows come 32 at a time, as in
// TokenWarps; the first warp of a row's first block computes what the rows have one of.  tiles > 1: a
// slice does not fit, and is read again, part by part, for each pass.  16000 x 5000 fp16 with 32 top
// classes: 64 us, 2.6 TB/s, two thirds of the issue slots with the 20 warps that the rows' 10 KB leave
// room for (36 us without top classes).  3 x 131072 fp32 with 64 on clusters of 8: 11 us, a chain of
// reads, barriers and searches.
template <typename T, int kTeam, bool kTop>
__global__ void
__launch_bounds__(kTeam == 32 ? 128 : kTeam, kTeam <= 128 ? 6 : kTeam == 256 ? 3 : 2)
TokenRing(Rows<T> rows, TokenOut out, int32_t vectors, int32_t tiles) {
  extern __shared__ uint4 shared[];
  __shared__ TokenShared<kTeam> all_shared[kTeam == 32 ? 4 : 1];
  static_assert(kTop || kTeam == 32, "TokenStream");
  __shared__ typename std::conditional<kTeam == 512, TokenTogether, int32_t>::type together;
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31,
                teams = kTeam == 32 ? (int32_t)blockDim.x / 32 : 1,
                team = kTeam == 32 ? warp : 0,
                tid = kTeam == 32 ? lane : (int32_t)threadIdx.x;
  const uint32_t cluster = kTeam == 512 ? ClusterSize() : 1,
                 rank = kTeam == 512 ? ClusterRank() : 0;
  TokenShared<kTeam> &sh = all_shared[team];
  const int32_t stage = kTeam * vectors;
  uint4 *slot = shared + team * stage + tid;
  using K = Keys<T, kTeam>;
  typename K::Key *keys =
      reinterpret_cast<typename K::Key *>(shared + teams * stage) + team * out.room;
  const int32_t apart = (int32_t)(gridDim.x / cluster) * teams;
  const bool slopes = out.entropy != nullptr,
             speaks = rank == 0 && (kTeam == 32 || warp == 0);
  int32_t parity = 0;
  for (int32_t base = (int32_t)(blockIdx.x / cluster) * teams + team; base < rows.count;
       base += 32 * apart) {
    const int32_t mine = base + lane * apart,
                  taken = min(32, (rows.count - base + apart - 1) / apart);
    const T *my_row = nullptr;
    int64_t token = -1;
    float score = 0.0f, my_high = 0.0f, my_sum = 0.0f, my_slope = 0.0f;
    if (lane < taken) {
      const RowPlace at = PlaceOf(rows, mine);
      if (at.counts) {
        my_row = rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride;
        if (out.log_probs && speaks) {
          token = IntAt(out.tokens, out.tokens_64, mine);
          if (token >= 0 && token < rows.classes) score = ToFloat(my_row[token]);
        }
      }
    }
    const auto row_of = [&](int32_t q) {
      return reinterpret_cast<const T *>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_row), q & 31));
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
    for (int32_t q = 0; q < taken; ++q) {
      const int32_t r = base + q * apart;
      const T *row = next;
      next = q + 1 < taken ? row_of(q + 1) : nullptr;
      const RowPart<T> whole = part_of(row), coming = part_of(next);
      const RowPart<T> *const then = tiles == 1 && next != nullptr ? &coming : nullptr;
      if (row == nullptr) {
        if (kTop && rank == 0) SkipTop(out, r, tid, kTeam);
        if (then) SendFor<kTeam, 0>(slot, coming, rows);
        continue;  // (all blocks of the cluster)
      }
      WaitForAll();
      const Refill<kTeam, T> refill(then, rows);
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
          f(part);
        }
      };
      // the largest score, of the warp and of four groups of each thread's; the warp's sums
      Sums sums = NoSums();
      each([&](const RowPart<T> &part) {
        CutEnds<kTeam>(slot, part);
        if constexpr (kTop) {
          if (slopes)
            AddRow<true, kTeam>(sums, slot, part.most, row, kLog2e, NoRefill());
          else
            AddRow<false, kTeam>(sums, slot, part.most, row, kLog2e, NoRefill());
        } else {
          if (slopes)
            AddRow<true, kTeam>(sums, slot, part.most, row, kLog2e, refill);
          else
            AddRow<false, kTeam>(sums, slot, part.most, row, kLog2e, refill);
        }
      });
      if (!kTop) refill.Rest(slot, whole.most, then, rows);
      float high;
      float2 both = slopes ? WarpSums<true>(sums, kLog2e, &high)
                           : WarpSums<false>(sums, kLog2e, &high);
      if (kTeam > 32) {
        // (a warp is at most one barrier ahead: the values of the row before are still read)
        parity ^= 1;
        if (lane == 0) {
          sh.high[parity][warp] = high;
          sh.sums[parity][warp] = both;
        }
        // (a block's threads are groups enough)
        sh.group[tid] = sums.high;
        __syncthreads();
        const bool one = lane < kTeam / 32;
        const float h = one ? sh.high[parity][lane] : -INFINITY;
        const float2 part = one ? sh.sums[parity][lane] : make_float2(0.0f, 0.0f);
        both = JoinWarp(h, part, &high);
      }
      int32_t found = 0;
      const int32_t top_k = max(0, min(out.top_k, min(span.classes, span.Column(last)) -
                                                     max(0, span.Column(first))));
      if (kTop) {
        // the bound of the top classes
        if (kTeam == 32 || warp == 0) {
          uint32_t bound, four[4];
          if (kTeam == 32) {
#pragma unroll
            for (int g = 0; g < 4; ++g) four[g] = OrderOf(sums.group[g]);
          } else {
            // (16, 8 or 4 groups per lane become four; of 16 or 8 there are 8 for many classes)
#pragma unroll
            for (int g = 0; g < 4; ++g) four[g] = 0;
#pragma unroll
            for (int g = 0; g < kTeam / 32; ++g)
              four[g & 3] = max(four[g & 3], OrderOf(sh.group[32 * g + lane]));
          }
          if (top_k <= 16) {
            const uint32_t one[1] = {max(max(four[0], four[1]), max(four[2], four[3]))};
            bound = BoundOf(one, top_k);
          } else if (kTeam <= 128 || top_k <= 64) {
            bound = BoundOf(four, top_k);
          } else if constexpr (kTeam > 128) {
            uint32_t eight[8] = {};
#pragma unroll
            for (int g = 0; g < kTeam / 32; ++g)
              eight[g & 7] = max(eight[g & 7], OrderOf(sh.group[32 * g + lane]));
            bound = BoundOf(eight, top_k);
          }
          if (lane == 0) {
            sh.bound = bound;
            sh.found = 0;
          }
        }
        TeamSync<kTeam>();
        const float least = ScoreOf(sh.bound);
        each([&](const RowPart<T> &part) {
          if (tiles > 1) CutEnds<kTeam>(slot, part);
          CollectRow<kTeam>(slot, part, least, keys, out.room, &sh.found, refill);
        });
        refill.Rest(slot, whole.most, then, rows);
        TeamSync<kTeam>();
        found = sh.found;
        if (found > out.room) {
          const uint64_t bound = RaiseBound(
              (uint64_t)sh.bound << 32, top_k, out.room, span.classes, [&](uint64_t key) {
                int32_t n = 0;
                EachKey<kTeam>(span, first, last, tid, key, [&](uint64_t) { ++n; });
                n = __reduce_add_sync(0xffffffffu, n);
                if (kTeam > 32) {
                  __syncthreads();
                  if (lane == 0) sh.counted[warp] = n;
                  __syncthreads();
                  n = 0;
#pragma unroll
                  for (int w = 0; w < kTeam / 32; ++w) n += sh.counted[w];
                }
                return n;
              });
          TeamSync<kTeam>();
          if (tid == 0) sh.found = 0;
          TeamSync<kTeam>();
          EachKey<kTeam>(span, first, last, tid, bound,
                         [&](uint64_t key) { PutKey(K::From(key), keys, out.room, &sh.found); });
          TeamSync<kTeam>();
          found = min(sh.found, out.room);
        }
      }
      if (kTeam == 512 && cluster > 1) {
        if constexpr (kTeam == 512) {
          EachPlaceBlock<kTeam>(keys, found, sh.places, tid, [&](int32_t at, uint64_t key) {
            if (at < top_k) together.list[at] = key;
          });
          if (tid == 0) together.top = top_k;
        }
        if (tid == 0) {
          sh.all_high = high;
          sh.all_sums = both;
        }
        ClusterSync();
        const bool one = lane < (int32_t)cluster;
        const float h = one ? ReadFrom(&sh.all_high, lane) : -INFINITY;
        const float2 part = one ? ReadFrom(&sh.all_sums, lane) : make_float2(0.0f, 0.0f);
        both = JoinWarp(h, part, &high);
        if constexpr (kTeam == 512)
          PlaceTogether(out, together, sh.places, top_k, r, cluster, tid, kTeam,
                        high == -INFINITY ? 0.0f : high, both.x);
        ClusterSync();  // nobody goes on while others read its memory
      } else if (kTop) {
        const float log_sum = logf(both.x), from = high == -INFINITY ? 0.0f : high;
        const auto write = [&](int32_t at, typename K::Key key) {
          if (at < out.top_k) WriteTop<K>(out, r, at, key, from, both.x, log_sum);
        };
        // (the next row's keys come to the same place, in a block behind two more barriers)
        if constexpr (kTeam == 32) {
          EachPlaceWarp(keys, found, lane, write);
          __syncwarp();
        } else {
          EachPlaceBlock<kTeam>(keys, found, sh.places, tid, write);
        }
      }
      if (lane == q) {
        my_high = high == -INFINITY ? 0.0f : high;
        my_sum = both.x;
        my_slope = both.y;
      }
    }
    if (speaks && lane < taken) {
      if (my_row != nullptr)
        Finish(out, mine, rows.classes, token, score, my_high, my_sum, my_slope);
      else
        SkipRow(out, mine);
    }
  }
}

// ---------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------
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
// row; what a class gets as a given or a top one is added where it is.  As 2^((x - high) log2 e) *
// (constant + by * (x - high)); the clamp leaves 0 and not 0 * -inf where p is 0.
struct Spread {
  float high, constant, by;
  __device__ __forceinline__ float operator()(float x) const {
    const float d = x - high;
    return Exp2(d * kLog2e) * (by == 0.0f ? constant : fmaf(by, fmaxf(d, -200.0f), constant));
  }
  template <typename T>
  __device__ __forceinline__ void operator()(const uint4 &v, const T *type,
                                             float (&f)[kPer<T>]) const {
    const Two minus = MakeTwo(-high, -high), k = MakeTwo(kLog2e, kLog2e),
              c = MakeTwo(constant, constant), b = MakeTwo(by, by);
    EachPair(v, type, [&](float2 x, int pair) {
      const Two d = Add(MakeTwo(x.x, x.y), minus);
      const float2 t = Split(Mul(d, k)), s = Split(d);
      const Two e = MakeTwo(Exp2(t.x), Exp2(t.y));
      const float2 g =
          Split(by == 0.0f
                    ? Mul(e, c)
                    : Mul(e, Fma(b, MakeTwo(fmaxf(s.x, -200.0f), fmaxf(s.y, -200.0f)), c)));
      f[2 * pair] = g.x;
      f[2 * pair + 1] = g.y;
    });
  }
};

// What the upstream and the norm say of a row.
struct TokenRowGrad {
  int32_t token;  // -1 for none
  float token_grad, slope, top_sum;
  float4 norm;
};
__device__ __forceinline__ TokenRowGrad ReadRowGrad(const TokenGrad &g, int32_t classes,
                                                    const RowPlace &at, int32_t r) {
  TokenRowGrad row;
  row.norm = g.norm[r];
  const int64_t token = g.log_probs.grad ? IntAt(g.tokens, g.tokens_64, r) : -1;
  const bool some = token >= 0 && token < classes;
  row.token = some ? (int32_t)token : -1;
  row.token_grad = token == -1 ? 0.0f : some ? GradAt(g.log_probs, at) : NAN;
  row.slope = GradAt(g.entropy, at);
  row.top_sum = 0.0f;
  return row;
}
__device__ __forceinline__ Spread SpreadOf(const TokenRowGrad &row, float top_sum) {
  const float inverse = row.norm.y == 0.0f ? 0.0f : 1.0f / row.norm.y;
  Spread spread;
  spread.high = row.norm.x;
  spread.by = -row.slope * inverse;
  // (a row without a class left: no class has a share)
  spread.constant =
      row.norm.y == 0.0f
          ? 0.0f
          : -inverse * fmaf(row.slope, row.norm.z - logf(row.norm.y), row.token_grad + top_sum);
  return spread;
}
// The given class, unless it is a top one, and the top classes, of those in [begin, end): by one warp
// behind the stores of all others.
template <bool kTop, typename T>
__device__ __forceinline__ void WriteTokens(const TokenGrad &g, const TokenRowGrad &row,
                                            const Spread &spread, const RowPlace &at, int32_t r,
                                            const T *x, T *out, int32_t begin, int32_t end,
                                            int32_t lane) {
  bool is_top = false;
  if (kTop) {
    const int32_t *top = g.top_tokens + (int64_t)r * g.top_k;
    for (int32_t k = lane; k < g.top_k; k += 32) {
      const int32_t c = top[k];
      is_top |= c == row.token;
      if (c < begin || c >= end) continue;
      float value = spread(ToFloat(x[c])) + GradAt(g.top, at, k);
      if (c == row.token) value += row.token_grad;
      out[c] = FromFloat<T>(value);
    }
    is_top = __any_sync(0xffffffffu, is_top);
  }
  if (lane == 0 && !is_top && row.token >= begin && row.token < end)
    out[row.token] = FromFloat<T>(spread(ToFloat(x[row.token])) + row.token_grad);
}

// A block per part of `part` vectors of a row: the norm is known, so every class is on its own.  Four
// vectors per thread are read while the four before them are worked on.  The classes that are a given
// or a top one are written again behind the others.  4096 x 32001 bf16: 77 us, 6.8 TB/s read and
// written, the memory's rate.
template <typename T, bool kTop>
__global__ void __launch_bounds__(256, 4)
TokenBlocksBackward(Rows<T> rows, TokenGrad g, T *grad, int32_t parts, int32_t part) {
  constexpr int kTeam = 256, kTile = 4;
  const int32_t tid = threadIdx.x, lane = tid & 31;
  const int32_t r = (int32_t)(blockIdx.x / (uint32_t)parts);
  const int32_t first = (int32_t)(blockIdx.x % (uint32_t)parts) * part;
  const RowPlace at = PlaceOf(rows, r);
  T *out = grad + at.o * g.outer_stride + at.i * g.inner_stride;
  if (!at.counts) {
    WriteZeros(out, rows.classes, first, first + part, tid, kTeam);
    return;
  }
  const RowSpan<T> span(rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride,
                        rows.classes);
  const bool aligned = (((uintptr_t)out ^ (uintptr_t)span.row) & 15) == 0;
  const RowStream<T> stream(span, min(first, span.vectors), min(span.vectors, first + part));
  uint4 v[kTile];
  const auto load = [&](int32_t tile) {
#pragma unroll
    for (int i = 0; i < kTile; ++i)
      if (tile + i * kTeam < stream.to) v[i] = stream.in[tile + i * kTeam];
  };
  load(stream.from + tid);
  const TokenRowGrad row = ReadRowGrad(g, rows.classes, at, r);
  float top_sum = 0.0f;
  if (kTop) {
    // (each warp for itself)
    for (int32_t k = lane; k < g.top_k; k += 32) top_sum += GradAt(g.top, at, k);
    top_sum = WarpSumF(top_sum);
  }
  const Spread spread = SpreadOf(row, top_sum);
  const auto edge = [&](int32_t j, const uint4 &x) {
    float f[kPer<T>];
    spread(x, span.row, f);
    Store(out, span, false, j, f);
  };
  for (int32_t tile = stream.from + tid; tile < stream.to; tile += kTeam * kTile) {
    uint4 x[kTile];
#pragma unroll
    for (int i = 0; i < kTile; ++i) x[i] = v[i];
    load(tile + kTeam * kTile);
    if (aligned) {
#pragma unroll
      for (int i = 0; i < kTile; ++i)
        if (tile + i * kTeam < stream.to) {
          float f[kPer<T>];
          spread(x[i], span.row, f);
          *reinterpret_cast<uint4 *>(out + span.Column(tile + i * kTeam)) = Pack(f, out);
        }
    } else {
#pragma unroll 1
      for (int32_t j = tile; j < min(stream.to, tile + kTeam * kTile); j += kTeam)
        edge(j, stream.in[j]);
    }
  }
  const int32_t end_at = stream.End(tid);
  if (end_at >= 0) edge(end_at, span.Edge(end_at));
  // behind the stores of the other threads
  __syncthreads();
  const int32_t begin = max(0, span.Column(stream.first)),
                end = min(span.classes, span.Column(stream.last));
  if (tid < 32) WriteTokens<kTop>(g, row, spread, at, r, span.row, out, begin, end, lane);
}

// Short rows: a warp takes 32 of them, a whole grid of warps apart.  Lane q reads what there is to
// know of the q-th, for all rows at once.  24000 rows of 29 fp32 classes with 3 top classes: 12 us (a
// warp per row that reads all of it for itself: 21).  64000 of 500 bf16 classes: 66 us, 78 with 8 top
// classes, 112 with 64, whose upstreams a lane reads one by one; 20 would be the memory's.
template <typename T, bool kTop>
__global__ void __launch_bounds__(128, 6)
TokenWarpsBackward(Rows<T> rows, TokenGrad g, T *grad) {
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int32_t apart = (int32_t)gridDim.x * warps;
  for (int32_t base = (int32_t)blockIdx.x * warps + warp; base < rows.count; base += 32 * apart) {
    const int32_t mine = base + lane * apart,
                  taken = min(32, (rows.count - base + apart - 1) / apart);
    RowPlace my_at = {};
    TokenRowGrad my_row = {};
    T *my_out = nullptr;
    if (lane < taken) {
      my_at = PlaceOf(rows, mine);
      my_out = grad + my_at.o * g.outer_stride + my_at.i * g.inner_stride;
      if (my_at.counts) {
        my_row = ReadRowGrad(g, rows.classes, my_at, mine);
        if (kTop)
          for (int32_t k = 0; k < g.top_k; ++k) my_row.top_sum += GradAt(g.top, my_at, k);
      }
    }
    const Spread my_spread = SpreadOf(my_row, my_row.top_sum);
    const auto from = [&](auto v, int32_t q) { return __shfl_sync(0xffffffffu, v, q); };
    for (int32_t q = 0; q < taken; ++q) {
      T *out = reinterpret_cast<T *>(from(reinterpret_cast<unsigned long long>(my_out), q));
      if (!from((int32_t)my_at.counts, q)) {
        WriteZeros(out, rows.classes, 0, INT32_MAX, lane, 32);
        continue;
      }
      RowPlace at;
      at.o = from(my_at.o, q);
      at.i = from(my_at.i, q);
      TokenRowGrad row;
      row.token = from(my_row.token, q);
      row.token_grad = from(my_row.token_grad, q);
      Spread spread;
      spread.high = from(my_spread.high, q);
      spread.constant = from(my_spread.constant, q);
      spread.by = from(my_spread.by, q);
      const RowSpan<T> span(rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride,
                            rows.classes);
      const bool aligned = (((uintptr_t)out ^ (uintptr_t)span.row) & 15) == 0;
      const RowStream<T> stream(span, 0, span.vectors);
#pragma unroll 2
      for (int32_t j = lane; j < span.vectors; j += 32) {
        const bool whole = j >= stream.from && j < stream.to;
        const uint4 x = whole ? stream.in[j] : span.Edge(j);
        float f[kPer<T>];
        spread(x, span.row, f);
        Store(out, span, aligned, j, f);
      }
      __syncwarp();
      WriteTokens<kTop>(g, row, spread, at, base + q * apart, span.row, out, 0, rows.classes, lane);
    }
  }
}

}  // namespace k2b

using namespace k2b;

namespace {

template <typename T, bool kTop>
int32_t LaunchTokenScores(const k2b200_class_rows *rows, const TokenOut &out, cudaStream_t s) {
  const Rows<T> r = RowsOf<T>(rows);
  const int32_t key_bytes = (int32_t)sizeof(uint64_t) * out.room;
  const RowPlan p = PlanRows(r, key_bytes, key_bytes);
  // (short rows with top classes: two of them, see TokenWarps)
  const size_t smem = (size_t)p.ring * (p.in_registers && kTop ? 2 : 1) +
                      (size_t)key_bytes * (p.block / p.team);
  if (p.in_registers) {
    auto kernel = p.vectors == 1   ? TokenWarps<T, 1, kTop>
                  : p.vectors == 2 ? TokenWarps<T, 2, kTop>
                  : p.vectors == 4 ? TokenWarps<T, 4, kTop>
                                   : TokenWarps<T, 8, kTop>;
    K2B_CUDA_OK(AllowShared(kernel, smem));
    kernel<<<(uint32_t)p.blocks, p.block, smem, s>>>(r, out);
  } else if (!kTop && p.team > 32) {
    K2B_CUDA_OK(LaunchRows(p.team == 128   ? TokenStream<T, 128>
                           : p.team == 256 ? TokenStream<T, 256>
                                           : TokenStream<T, 512>,
                           (int64_t)r.count * p.cluster, p.block, 0, p.cluster, false, s, r, out));
  } else {
    auto kernel = p.team == 32    ? TokenRing<T, 32, kTop>
                  : p.team == 128 ? TokenRing<T, 128, true>
                  : p.team == 256 ? TokenRing<T, 256, true>
                                  : TokenRing<T, 512, true>;
    K2B_CUDA_OK(AllowShared(kernel, smem));
    K2B_CUDA_OK(LaunchRows(kernel, p.blocks, p.block, smem, p.cluster, false, s, r, out, p.vectors,
                           p.tiles));
  }
  NoteLaunch();
  K2B_CUDA_OK(cudaGetLastError());
  return kOk;
}

template <typename T>
int32_t LaunchTokenBackward(const k2b200_class_rows *rows, const TokenGrad &g, void *grad,
                            cudaStream_t s) {
  const Rows<T> r = RowsOf<T>(rows);
  T *out = static_cast<T *>(grad);
  const bool top = g.top_k > 0;
  // vectors of a row, wherever it begins: up to 256 of them are a warp's; more are dealt out to
  // blocks in parts of 4096, 16 per thread, or of 1024 where that is too few blocks (4096 x 32001
  // bf16: 102 us in parts of 1024, 83 of 2048, 77 of 4096, at the memory's rate)
  const int32_t vectors = CeilDiv((int64_t)r.classes + kPer<T> - 1, kPer<T>) + 1;
  if (vectors <= 256) {
    const int32_t warps =
        (int32_t)std::min<int64_t>(4, std::max<int64_t>(1, r.count / NumSms()));
    auto kernel = top ? TokenWarpsBackward<T, true> : TokenWarpsBackward<T, false>;
    const int64_t blocks = std::min<int64_t>((r.count + warps - 1) / warps,
                                             (int64_t)NumSms() * 6 * (4 / warps));
    kernel<<<(uint32_t)blocks, 32 * warps, 0, s>>>(r, g, out);
  } else {
    const int32_t part = CeilDiv(vectors, 4096) * (int64_t)r.count >= 2 * NumSms() ? 4096 : 1024,
                  parts = CeilDiv(vectors, part);
    K2B_REQUIRE((int64_t)parts * r.count < ((int64_t)1 << 31), "too many rows of %d classes",
                r.classes);
    auto kernel = top ? TokenBlocksBackward<T, true> : TokenBlocksBackward<T, false>;
    kernel<<<(uint32_t)((int64_t)parts * r.count), 256, 0, s>>>(r, g, out, parts, part);
  }
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
  K2B_REQUIRE(Aligned(norm, 16), "norm that is not aligned to 16 bytes");
  K2B_REQUIRE(Aligned(tokens, IntSize(tokens_64)) && Aligned(log_probs, 4) &&
                  Aligned(entropy, 4) && Aligned(top_log_probs, 4) && Aligned(top_tokens, 4),
              "tokens or outputs that are not aligned to their type");
  K2B_REQUIRE(top_k >= 0 && top_k <= K2B200_MAX_TOP && top_k <= rows->num_classes,
              "top_k is %d: 0 to %d, and at most the %d classes", top_k, K2B200_MAX_TOP,
              rows->num_classes);
  if (rows->outer * rows->inner == 0) return kOk;
  K2B_REQUIRE((log_probs == nullptr) == (tokens == nullptr),
              "tokens and log_probs are given together");
  K2B_REQUIRE(top_k == 0 || (top_log_probs && top_tokens), "NULL pointer");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const TokenOut out = {tokens,     tokens_64,     top_k,
                        RoomFor(top_k), log_probs, entropy,
                        top_log_probs,  top_tokens, reinterpret_cast<float4 *>(norm)};
  const bool top = top_k > 0;
  auto launch =
      rows->type == K2B200_F32   ? (top ? LaunchTokenScores<float, true>
                                        : LaunchTokenScores<float, false>)
      : rows->type == K2B200_F16 ? (top ? LaunchTokenScores<__half, true>
                                        : LaunchTokenScores<__half, false>)
                                 : (top ? LaunchTokenScores<__nv_bfloat16, true>
                                        : LaunchTokenScores<__nv_bfloat16, false>);
  return launch(rows, out, s);
}

int32_t k2b200_token_scores_backward(const k2b200_class_rows *rows, const void *tokens,
                                     int32_t tokens_64, int32_t top_k, const int32_t *top_tokens,
                                     const float *norm, const k2b200_row_grad *log_probs_grad,
                                     const k2b200_row_grad *entropy_grad,
                                     const k2b200_row_grad *top_log_probs_grad,
                                     void *grad_scores, int64_t grad_outer_stride,
                                     int64_t grad_inner_stride, void *stream) {
  K2B_FORWARD(CheckRows(rows));
  K2B_REQUIRE(Aligned(norm, 16), "norm that is not aligned to 16 bytes");
  K2B_REQUIRE(log_probs_grad && entropy_grad && top_log_probs_grad, "NULL pointer");
  K2B_REQUIRE(Aligned(grad_scores, FloatSize(rows->type)) && Aligned(log_probs_grad->grad, 4) &&
                  Aligned(entropy_grad->grad, 4) && Aligned(top_log_probs_grad->grad, 4),
              "a gradient that is not aligned to its type");
  K2B_REQUIRE(Aligned(tokens, IntSize(tokens_64)) && Aligned(top_tokens, 4),
              "tokens that are not aligned to their type");
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
