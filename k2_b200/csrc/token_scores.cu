// Log-probs of given classes, entropies and top classes of rows of scores, and their gradient.
//
// TokenScores holds a row in registers (class_rows.cuh).  Sums: with d_c = (x_c - high) log2 e and
// e_c = 2^d_c, log p_c = (x_c - high) - ln sum e, and the entropy is ln sum e - ln 2 (sum e d) /
// sum e.  Top classes: the threads' largest scores are themselves scores of the row, so that the
// k-th largest of them bounds the row's k-th largest from below, and few scores lie above it (of
// n threads about n ln(n / (n - k))); those are collected in shared memory, and each one's place
// is the number of larger ones.  Where more lie above it than there is room for - ties, or many
// large scores in one thread - the bound is raised by bisection over (score, class), which no two
// classes share.
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
// are so many; -inf else.  By bisection, until no more than a quarter too many reach it.
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
      if (reach <= k + (k >> 2)) break;
    } else {
      high = mid;
    }
  }
  return low;
}

// Whether scores of a thread's vectors are below `least`: bit 31 - k % 32 of word k / 32 for score k
// of them (NaN is not).  The sign of a difference is shifted in, one instruction a score and half a
// one for the difference.
template <typename T, int kVectors>
struct Below {
  static constexpr int kScores = kVectors * kPer<T>, kWords = (kScores + 31) / 32,
                       kEmpty = kWords * 32 - kScores;
  uint32_t word[kWords];
  __device__ __forceinline__ Below(uint4 (&v)[kVectors], const T *type, float least) {
    const float up = 0.0f - least;  // (+0 for both zeros: neither is below the other)
    const Two minus = MakeTwo(up, up);
#pragma unroll
    for (int w = 0; w < kWords; ++w) word[w] = 0;
#pragma unroll
    for (int i = 0; i < kVectors; ++i)
      EachPair(Packed(v[i]), type, [&](float2 x, int) {
        const float2 d = Split(Add(MakeTwo(x.x, x.y), minus));
        uint32_t &w = word[i * kPer<T> / 32];
        w = __funnelshift_l(__float_as_uint(d.x), w, 1);
        w = __funnelshift_l(__float_as_uint(d.y), w, 1);
      });
    word[kWords - 1] <<= kEmpty;
  }
  // The scores that are not, of word w.
  __device__ __forceinline__ uint32_t Not(int w) const {
    return ~word[w] & (w + 1 == kWords ? ~0u << kEmpty : ~0u);
  }
};

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
  for (;;) {
    const int32_t n = count(mid);
    if (n >= top_k && n <= room) return mid;
    if (n < top_k) far = mid; else low = mid;
    // between keys of one score there are the classes
    if ((far - 1) >> 32 == low >> 32)
      low = max((unsigned long long)low, (low | 0xffffffffull) - (uint64_t)classes);
    mid = low + (far - low) / 2;
  }
}

__device__ __forceinline__ void WriteTop(const TokenOut &out, int32_t r, int32_t place,
                                         uint64_t key, float high, float sum, float log_sum) {
  const int64_t at = (int64_t)r * out.top_k + place;
  out.top_tokens[at] = (int32_t)~(uint32_t)key;
  out.top_log_probs[at] =
      sum == 0.0f ? -INFINITY : (ScoreOf((uint32_t)(key >> 32)) - high) - log_sum;
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

// Rows of up to 4 KB: a warp takes `per_warp` of them one after the other.  Lane q knows where the
// q-th of them is and its given class, gathers its sums, and computes what a row has one of, for
// all rows of the warp at once.
template <typename T, int kVectors, bool kTop>
__global__ void __launch_bounds__(128, kVectors >= 8 ? 6 : 8)
TokenWarps(Rows<T> rows, TokenOut out, int32_t per_warp) {
  extern __shared__ uint64_t all_keys[];
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t *keys = all_keys + warp * out.room;
  const int32_t first = (int32_t)(blockIdx.x * (blockDim.x >> 5) + warp) * per_warp,
                mine = first + lane, taken = min(per_warp, rows.count - first);
  if (taken <= 0) return;
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
  const bool slopes = out.entropy || out.norm;
  for (int32_t q = 0; q < taken; ++q) {
    const T *row = reinterpret_cast<const T *>(
        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(my_row), q));
    if (row == nullptr) {
      if (kTop) SkipTop(out, first + q, lane, 32);
      continue;
    }
    const RowSpan<T> span(row, rows.classes);
    uint4 v[kVectors];
    LoadTile<32, kVectors>(v, span, rows, 0, span.vectors, lane);
    // the largest score, of the warp and of two groups per lane
    float group[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      float &g = group[2 * i / kVectors];
      g = fmaxf(g, VectorMax(Packed(v[i]), span.row));
    }
    const float lane_high = fmaxf(group[0], group[1]), high = WarpMaxF(lane_high),
                from = high == -INFINITY ? 0.0f : high;
    // the sums, of two vectors at a time
    Two sums[2] = {}, slope[2] = {};
    if (slopes) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        After(v[i], sums[i & 1]);
        AddVector<true>(v[i], span.row, from, kLog2e, sums[i & 1], slope[i & 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) {
        After(v[i], sums[i & 1]);
        AddVector<false>(v[i], span.row, from, kLog2e, sums[i & 1], slope[i & 1]);
      }
    }
    const float2 s = Split(Add(sums[0], sums[1])), t = Split(Add(slope[0], slope[1]));
    const float2 both =
        slopes ? WarpSum2F(s.x + s.y, t.x + t.y) : make_float2(WarpSumF(s.x + s.y), 0.0f);
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
        float left = lane_high;
        least = high;
        for (int32_t k = 1; k < out.top_k; ++k) {
          if (left == least) left = -INFINITY;
          least = WarpMaxF(left);
        }
      } else {
        const uint32_t two[2] = {OrderOf(group[0]), OrderOf(group[1])};
        least = ScoreOf(BoundOf(two, out.top_k));
      }
      const Below<T, kVectors> below(v, span.row, least);
      int32_t found = 0;
      __syncwarp();  // (the keys of the row before have been read)
#pragma unroll
      for (int w = 0; w < below.kWords; ++w) {
        uint32_t hits = below.Not(w);
        // each lane's hits one after the other; its scores come from a cache again
        for (uint32_t some; (some = __ballot_sync(0xffffffffu, hits != 0)) != 0;) {
          uint64_t key = 0;
          if (hits) {
            const int32_t bit = __clz(hits), k = 32 * w + bit;
            hits &= ~(0x80000000u >> bit);
            const int32_t c = span.Column(k / kPer<T> * 32 + lane) + k % kPer<T>;
            if (c >= 0 && c < span.classes) key = KeyOf(ToFloat(row[c]), c);
          }
          const uint32_t good = __ballot_sync(0xffffffffu, key != 0);
          const int32_t place = found + __popc(good & ((1u << lane) - 1));
          if (key != 0 && place < out.room) keys[place] = key;
          found += __popc(good);
        }
      }
      __syncwarp();
      if (found > out.room) {
        const uint64_t bound = RaiseBound(
            (uint64_t)OrderOf(least) << 32, out.top_k, out.room, span.classes,
            [&](uint64_t key) {
              int32_t n = 0;
              EachKey<32>(span, 0, span.vectors, lane, key, [&](uint64_t) { ++n; });
              return (int32_t)__reduce_add_sync(0xffffffffu, n);
            });
        // (a key's place among those of the lane's and of lower lanes')
        int32_t n = 0;
        EachKey<32>(span, 0, span.vectors, lane, bound, [&](uint64_t) { ++n; });
        int32_t place = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int32_t o = __shfl_up_sync(0xffffffffu, place, d);
          if (lane >= d) place += o;
        }
        found = __shfl_sync(0xffffffffu, place, 31);
        place -= n;
        EachKey<32>(span, 0, span.vectors, lane, bound,
                    [&](uint64_t key) { keys[place++] = key; });
        __syncwarp();
      }
      const float log_sum = logf(sum);
      for (int32_t k = lane; k < found; k += 32) {
        const uint64_t key = keys[k];
        int32_t place = 0;
        for (int32_t o = 0; o < found; ++o) place += keys[o] > key;
        if (place < out.top_k) WriteTop(out, first + q, place, key, from, sum, log_sum);
      }
    }
  }
  if (lane < taken) {
    if (my_row != nullptr)
      Finish(out, mine, rows.classes, token, score, my_high, my_sum, my_slope);
    else
      SkipRow(out, mine);
  }
}

template <int kTeam>
struct TokenShared {
  float high[kTeam / 32];
  float2 sums[kTeam / 32];
  int32_t counted[kTeam / 32];
  int32_t found;
  uint32_t bound;
  float group[2 * kTeam];
};

// What the blocks of a cluster tell each other.
struct TokenCluster {
  float high, sum, slope;
  int32_t top;                       // keys in `list`
  uint64_t list[K2B200_MAX_TOP];     // this block's, largest first
  uint64_t others[8 * K2B200_MAX_TOP];
};

// A block of kTeam threads per row with kVectors vectors each; kAgain: the row does not fit and is
// read again for each pass.  Rows of a cluster of blocks (kTeam 256) are dealt out in slices.
template <typename T, int kTeam, int kVectors, bool kTop, bool kAgain>
__global__ void __launch_bounds__(kTeam, MinBlocks(kTeam, kVectors))
TokenBlocks(Rows<T> rows, TokenOut out) {
  extern __shared__ uint64_t keys[];
  __shared__ TokenShared<kTeam> sh;
  // (the smallest where blocks share no row)
  __shared__ typename std::conditional<kTeam == 256, TokenCluster, int32_t>::type together;
  const int32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t cluster = kTeam == 256 ? ClusterSize() : 1,
                 rank = kTeam == 256 ? ClusterRank() : 0;
  const int32_t r = (int32_t)(blockIdx.x / cluster);
  const RowPlace at = PlaceOf(rows, r);
  if (!at.counts) {
    if (rank == 0) {
      if (tid == 0) SkipRow(out, r);
      SkipTop(out, r, tid, kTeam);
    }
    return;  // (all blocks of the cluster)
  }
  const RowSpan<T> span(rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride,
                        rows.classes);
  const int32_t slice = (span.vectors + (int32_t)cluster - 1) / (int32_t)cluster;
  const int32_t first = min(span.vectors, (int32_t)rank * slice),
                last = min(span.vectors, first + slice);

  uint4 v[kVectors];
  const auto each = [&](auto &&f) {
    if constexpr (kAgain) {
      for (int32_t tile = first; tile < last; tile += kTeam * kVectors) {
        LoadTile<kTeam, kVectors>(v, span, rows, tile, last, tid);
#pragma unroll
        for (int i = 0; i < kVectors; ++i) f(i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) f(i);
    }
  };
  if (!kAgain) LoadTile<kTeam, kVectors>(v, span, rows, first, last, tid);
  // the given class's score is on its way meanwhile
  int64_t token = -1;
  float token_score = 0.0f;
  if (out.log_probs && tid == 0 && rank == 0) {
    token = IntAt(out.tokens, out.tokens_64, r);
    if (token >= 0 && token < rows.classes) token_score = ToFloat(span.row[token]);
  }

  // the largest score, of the warp and of two groups per thread; the warp's sums
  float group[2] = {-INFINITY, -INFINITY};
  each([&](int i) {
    float &g = group[2 * i / kVectors];
    g = fmaxf(g, VectorMax(Packed(v[i]), span.row));
  });
  const float warp_high = WarpMaxF(fmaxf(group[0], group[1])),
              warp_from = warp_high == -INFINITY ? 0.0f : warp_high;
  Two sums[2] = {}, slopes[2] = {};
  if (out.entropy || out.norm)
    each([&](int i) {
      After(v[i], sums[i & 1]);
      AddVector<true>(v[i], span.row, warp_from, kLog2e, sums[i & 1], slopes[i & 1]);
    });
  else
    each([&](int i) {
      After(v[i], sums[i & 1]);
      AddVector<false>(v[i], span.row, warp_from, kLog2e, sums[i & 1], slopes[i & 1]);
    });
  const float2 s = Split(Add(sums[0], sums[1])), t = Split(Add(slopes[0], slopes[1]));
  const float2 both = WarpSum2F(s.x + s.y, t.x + t.y);
  if (lane == 0) {
    sh.high[warp] = warp_high;
    sh.sums[warp] = both;
  }
  if (kTop) {
    sh.group[tid] = group[0];
    sh.group[kTeam + tid] = group[1];
  }
  __syncthreads();
  float high = sh.high[0];
#pragma unroll
  for (int w = 1; w < kTeam / 32; ++w) high = fmaxf(high, sh.high[w]);
  const float from = high == -INFINITY ? 0.0f : high;
  float sum = 0.0f, slope = 0.0f;
#pragma unroll
  for (int w = 0; w < kTeam / 32; ++w)
    Join(sum, slope, sh.sums[w].x, sh.sums[w].y, sh.high[w] - from);

  int32_t found = 0;
  const int32_t top_k = max(0, min(out.top_k, min(span.classes, span.Column(last)) -
                                                 max(0, span.Column(first))));
  if (kTop) {
    // the bound of the top classes
    if (warp == 0) {
      constexpr int kAll = 2 * kTeam / 32;
      uint32_t order[kAll], bound;
#pragma unroll
      for (int g = 0; g < kAll; ++g) order[g] = OrderOf(sh.group[32 * g + lane]);
      if (top_k <= 32) {
        uint32_t two[2] = {0, 0};
#pragma unroll
        for (int g = 0; g < kAll; ++g) two[g & 1] = max(two[g & 1], order[g]);
        const uint32_t one[1] = {max(two[0], two[1])};
        bound = top_k <= 16 ? BoundOf(one, top_k) : BoundOf(two, top_k);
      } else {
        bound = BoundOf(order, top_k);
      }
      if (lane == 0) {
        sh.bound = bound;
        sh.found = 0;
      }
    }
    __syncthreads();
    const float least = ScoreOf(sh.bound);
    const auto collect = [&](int32_t tile) {
      const Below<T, kVectors> below(v, span.row, least);
#pragma unroll
      for (int w = 0; w < below.kWords; ++w) {
        uint32_t hits = below.Not(w);
        while (hits) {
          const int32_t bit = __clz(hits), k = 32 * w + bit;
          hits &= ~(0x80000000u >> bit);
          const int32_t j = tile + k / kPer<T> * kTeam + tid, c = span.Column(j) + k % kPer<T>;
          if (j >= last || c < 0 || c >= span.classes) continue;
          const int32_t place = atomicAdd(&sh.found, 1);
          if (place < out.room) keys[place] = KeyOf(ToFloat(span.row[c]), c);
        }
      }
    };
    if constexpr (kAgain) {
      for (int32_t tile = first; tile < last; tile += kTeam * kVectors) {
        LoadTile<kTeam, kVectors>(v, span, rows, tile, last, tid);
        collect(tile);
      }
    } else {
      collect(first);
    }
    __syncthreads();
    found = sh.found;
    if (found > out.room) {
      const uint64_t bound = RaiseBound(
          (uint64_t)sh.bound << 32, top_k, out.room, span.classes, [&](uint64_t key) {
            int32_t n = 0;
            EachKey<kTeam>(span, first, last, tid, key, [&](uint64_t) { ++n; });
            n = __reduce_add_sync(0xffffffffu, n);
            __syncthreads();
            if (lane == 0) sh.counted[warp] = n;
            __syncthreads();
            n = 0;
#pragma unroll
            for (int w = 0; w < kTeam / 32; ++w) n += sh.counted[w];
            return n;
          });
      __syncthreads();
      if (tid == 0) sh.found = 0;
      __syncthreads();
      EachKey<kTeam>(span, first, last, tid, bound,
                     [&](uint64_t key) { keys[atomicAdd(&sh.found, 1)] = key; });
      __syncthreads();
      found = sh.found;
    }
  }

  if constexpr (kTeam == 256) {
    if (cluster > 1) {
      // the first block of a cluster has the row's sums; each finds the places of its own keys
      if (kTop)
        for (int32_t k = tid; k < found; k += kTeam) {
          const uint64_t key = keys[k];
          int32_t place = 0;
          for (int32_t o = 0; o < found; ++o) place += keys[o] > key;
          if (place < top_k) together.list[place] = key;
        }
      if (tid == 0) {
        together.high = high;
        together.sum = sum;
        together.slope = slope;
        together.top = kTop ? top_k : 0;
      }
      ClusterSync();
      for (uint32_t b = 0; b < cluster; ++b) high = fmaxf(high, ReadFrom(&together.high, b));
      const float all_from = high == -INFINITY ? 0.0f : high;
      sum = slope = 0.0f;
      for (uint32_t b = 0; b < cluster; ++b)
        Join(sum, slope, ReadFrom(&together.sum, b), ReadFrom(&together.slope, b),
             ReadFrom(&together.high, b) - all_from);
      if (tid == 0 && rank == 0)
        Finish(out, r, rows.classes, token, token_score, all_from, sum, slope);
      if (kTop) {
        const float log_sum = logf(sum);
        int32_t others = 0;
        for (uint32_t b = 0; b < cluster; ++b) {
          if (b == rank) continue;
          const int32_t n = ReadFrom(&together.top, b);
          for (int32_t k = tid; k < n; k += kTeam)
            together.others[others + k] = ReadFrom(&together.list[k], b);
          others += n;
        }
        __syncthreads();
        for (int32_t k = tid; k < top_k; k += kTeam) {
          const uint64_t key = together.list[k];
          int32_t place = k, begin = 0;
          for (uint32_t b = 0; b < cluster; ++b) {
            if (b == rank) continue;
            // how many of a list that falls are larger
            const int32_t n = ReadFrom(&together.top, b);
            int32_t low = 0, far = n;
            while (low < far) {
              const int32_t mid = (low + far) / 2;
              if (together.others[begin + mid] > key) low = mid + 1; else far = mid;
            }
            place += low;
            begin += n;
          }
          if (place < out.top_k) WriteTop(out, r, place, key, all_from, sum, log_sum);
        }
      }
      ClusterSync();  // nobody leaves while others read its memory
      return;
    }
  }
  if (tid == 0) Finish(out, r, rows.classes, token, token_score, from, sum, slope);
  if (kTop) {
    const float log_sum = logf(sum);
    for (int32_t k = tid; k < found; k += kTeam) {
      const uint64_t key = keys[k];
      int32_t place = 0;
      for (int32_t o = 0; o < found; ++o) place += keys[o] > key;
      if (place < out.top_k) WriteTop(out, r, place, key, from, sum, log_sum);
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
// row; what a class gets as a given or a top one is added where it is.
struct Spread {
  float high, inverse, all, slope, offset;
  __device__ __forceinline__ float operator()(float x) const {
    const float d = x - high, p = Exp2(d * kLog2e) * inverse;
    return p == 0.0f ? 0.0f : -p * fmaf(slope, d + offset, all);
  }
};

// A team per row and kTile vectors per thread of it at a time: the norm is known, so every class
// is on its own.  The classes that are a given or a top one are written again behind the others.
template <typename T, int kTeam, bool kTop>
__global__ void __launch_bounds__(256, 4)
TokenScoresBackward(Rows<T> rows, TokenGrad g, T *grad, int32_t parts, int32_t part) {
  constexpr int kTile = 4;
  const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t tid = kTeam == 32 ? lane : (int32_t)threadIdx.x;
  const int32_t r = kTeam == 32 ? (int32_t)(blockIdx.x * (blockDim.x >> 5)) + warp
                                : (int32_t)(blockIdx.x / (uint32_t)parts);
  if (r >= rows.count) return;
  const int32_t slice = kTeam == 32 ? 0 : (int32_t)(blockIdx.x % (uint32_t)parts);
  const RowPlace at = PlaceOf(rows, r);
  T *out = grad + at.o * g.outer_stride + at.i * g.inner_stride;
  if (!at.counts) {
    const RowSpan<T> zeros(out, rows.classes);
    const float f[kPer<T>] = {};
    const int32_t end = kTeam == 32 ? zeros.vectors : min(zeros.vectors, (slice + 1) * part);
    for (int32_t j = slice * part + tid; j < end; j += kTeam) Store(out, zeros, true, j, f);
    return;
  }
  const RowSpan<T> span(rows.scores + at.o * rows.outer_stride + at.i * rows.inner_stride,
                        rows.classes);
  const bool aligned = (((uintptr_t)out ^ (uintptr_t)span.row) & 15) == 0;
  const int32_t first = slice * part,
                last = kTeam == 32 ? span.vectors : min(span.vectors, first + part);
  uint4 v[kTile];
  LoadTile<kTeam, kTile>(v, span, rows, first, last, tid);
  const float4 n = g.norm[r];
  const int64_t token = g.log_probs.grad ? IntAt(g.tokens, g.tokens_64, r) : -1;
  const bool some = token >= 0 && token < rows.classes;
  const float token_grad = token == -1 ? 0.0f : some ? GradAt(g.log_probs, at) : NAN;
  float top_sum = 0.0f;
  if (kTop) {
    // (each warp for itself)
    for (int32_t k = lane; k < g.top_k; k += 32) top_sum += GradAt(g.top, at, k);
    top_sum = WarpSumF(top_sum);
  }
  Spread spread;
  spread.high = n.x;
  spread.inverse = n.y == 0.0f ? 0.0f : 1.0f / n.y;
  spread.all = token_grad + top_sum;
  spread.slope = GradAt(g.entropy, at);
  spread.offset = n.z - logf(n.y);
  for (int32_t tile = first; tile < last; tile += kTeam * kTile) {
    if (tile != first) LoadTile<kTeam, kTile>(v, span, rows, tile, last, tid);
#pragma unroll
    for (int i = 0; i < kTile; ++i) {
      const int32_t j = tile + i * kTeam + tid;
      if (j >= last) continue;
      float f[kPer<T>];
      Unpack(Packed(v[i]), f, span.row);
#pragma unroll
      for (int k = 0; k < kPer<T>; ++k) f[k] = spread(f[k]);
      Store(out, span, aligned, j, f);
    }
  }
  // behind the stores of the other threads: the token, unless a top class, and the top classes
  TeamSync<kTeam>();
  const int32_t begin = max(0, span.Column(first)),
                end = min(span.classes, span.Column(last));
  const auto mine = [&](int64_t c) { return c >= begin && c < end; };
  bool token_is_top = false;
  if (kTop) {
    const int32_t *top = g.top_tokens + (int64_t)r * g.top_k;
    for (int32_t k = tid; k < g.top_k; k += kTeam) {
      const int32_t c = top[k];
      if (!mine(c)) continue;
      float value = spread(ToFloat(span.row[c])) + GradAt(g.top, at, k);
      if (c == token) value += token_grad;
      out[c] = FromFloat<T>(value);
    }
    if (some && tid < 32) {
      for (int32_t k = lane; k < g.top_k; k += 32) token_is_top |= top[k] == token;
      token_is_top = __any_sync(0xffffffffu, token_is_top);
    }
  }
  if (tid == 0 && some && !token_is_top && mine(token))
    out[token] = FromFloat<T>(spread(ToFloat(span.row[token])) + token_grad);
}

}  // namespace k2b

using namespace k2b;

namespace {

template <typename T, bool kTop>
int32_t LaunchTokenScores(const k2b200_class_rows *rows, const TokenOut &out, cudaStream_t s) {
  const Rows<T> r = RowsOf<T>(rows);
  const RowPlan p = PlanRows(r);
  if (p.team == 32) {
    auto kernel = p.vectors == 1   ? TokenWarps<T, 1, kTop>
                  : p.vectors == 2 ? TokenWarps<T, 2, kTop>
                  : p.vectors == 4 ? TokenWarps<T, 4, kTop>
                                   : TokenWarps<T, 8, kTop>;
    kernel<<<CeilDiv(r.count, p.rows_per_block), p.block,
             sizeof(uint64_t) * out.room * (p.block / 32), s>>>(r, out, p.rows_per_warp);
  } else {
    auto kernel = p.team == 128   ? (p.vectors == 4 ? TokenBlocks<T, 128, 4, kTop, false>
                                                    : TokenBlocks<T, 128, 8, kTop, false>)
                  : p.again        ? TokenBlocks<T, 256, 16, kTop, true>
                  : p.vectors == 4 ? TokenBlocks<T, 256, 4, kTop, false>
                  : p.vectors == 8 ? TokenBlocks<T, 256, 8, kTop, false>
                                   : TokenBlocks<T, 256, 16, kTop, false>;
    K2B_CUDA_OK(LaunchRows(kernel, (int64_t)r.count * p.cluster, p.block,
                           sizeof(uint64_t) * out.room, p.cluster, false, s, r, out));
  }
  NoteLaunch();
  K2B_CUDA_OK(cudaGetLastError());
  return kOk;
}

template <typename T>
int32_t LaunchTokenBackward(const k2b200_class_rows *rows, const TokenGrad &g, void *grad,
                            cudaStream_t s) {
  const Rows<T> r = RowsOf<T>(rows);
  const RowPlan p = PlanRows(r);
  T *out = static_cast<T *>(grad);
  const bool top = g.top_k > 0;
  // vectors of a row, wherever it begins, in parts of 1024: a block's four per thread
  const int32_t vectors =
      (int32_t)((rows->num_classes + kPer<T> - 1) / kPer<T>) + (kPer<T> > 1 ? 1 : 0);
  if (p.team == 32) {
    auto kernel = top ? TokenScoresBackward<T, 32, true> : TokenScoresBackward<T, 32, false>;
    kernel<<<CeilDiv(r.count, p.block / 32), p.block, 0, s>>>(r, g, out, 1, 0);
  } else {
    const int32_t part = 1024, parts = CeilDiv(vectors, part);
    K2B_REQUIRE((int64_t)parts * r.count < ((int64_t)1 << 31), "too many rows of %d classes",
                rows->num_classes);
    auto kernel = top ? TokenScoresBackward<T, 256, true> : TokenScoresBackward<T, 256, false>;
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
