// Log probabilities of given tokens, entropy and the likeliest alternatives of
// rows of logits, and the gradient of the first two.
//
//   m = max x,  z_j = s (x_j - m),  S0 = sum e^z,  S1 = sum z e^z,  logsum = ln S0
//   logprob = z_t - logsum,   entropy = logsum - S1 / S0
//   dx_j = s (g (1[j = t] - p_j) - h p_j (ln p_j + entropy)),   p_j = e^(z_j - logsum)
//
// The forward pass reads the logits once.  A wave keeps one reference for its
// exponentials, the largest logit seen when it was last set, and sets it anew
// only when a logit exceeds it by 2^64 in the exponential (far from zero, whenever one
// exceeds it): sums in fp32 have the room, and a tile of up to 32 logits per lane costs
// one comparison instead of a rescaling.  Lanes, waves and parts of a row are joined
// relative to the true maximum.  Memory bounds it, with the vector units close behind (nine issue
// slots per 16-bit logit, four of them the exponential's): 4096 rows of 131072
// bf16 160 us without alternatives (6.7 TB/s), 173 with eight; of 65536 fp32 155
// and 165.  Eight rows of 131072 with twenty alternatives take 10.7 us, one row
// 9.8: there it is the chain of steps that counts.
//
// Alternatives cost next to nothing while the row streams by: a lane notes the
// maximum of each of its tiles (a "segment") in LDS.  The k-th best of the
// lanes' maxima bounds the k-th best logit from below, and only segments that
// reach the bound are looked at again: k of them and a few more.  Logits are
// compared as (value, place) with the lowest place first, an order without
// ties.  Where equal logits are so many that the bound leaves a long list
// (constant rows, rows with fewer than k logits that are not -infinity), the
// lanes' and then the segments' maxima are ordered by place as well, which
// bounds every list whatever the data: k lanes per wave, 16 segments per lane,
// then k segments of 32 logits.  The answer is the same on every run.
#include "typed.h"

#include <algorithm>
#include <cmath>

using namespace polar_hip_detail;

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kPacks = 4;        // 16-byte packs a lane takes per tile
constexpr int kMaxTiles = 16;    // tiles of a part, so segments per lane
constexpr int kMaxTop = 32;
constexpr int kMaxListed = kWaves * kMaxTop * kMaxTiles;  // segments that can reach the exact bound
constexpr uint32_t kShortList = 64;                       // segments whose logits are looked at without ordering them first
constexpr uint32_t kStagedAt = 12288;                     // bytes in front of the staged packs of a part of one tile
constexpr uint64_t kMaxCols = 1ull << 24;                 // places are exact as fp32 tokens
constexpr uint64_t kMostGroups = 1ull << 23;              // of a launch, whose lanes are counted in 32 bits
constexpr float kLeastScale = 0x1p-64f, kMostScale = 0x1p64f; // far from where scale * log2 e overflows or vanishes
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

template <typename T> constexpr uint32_t tileCols() { return kBlock * kPacks * T::kVec; }

// Sums relative to a maximum, exponents in base 2: s0 = sum 2^y, s1 = sum y 2^y
// with y = (x - m) c.
struct RowSums {
  float m, s0, s1;
};

// What a sum relative to `from` is multiplied by to be relative to `to` >= from,
// as an exponent; an empty sum's `from` is -infinity, and both may be.  No less than
// -300: sums are below 2^80, so that nothing of them is left there, and a sum times the
// exponent (which s1 needs) stays far from fp32's limit.
__device__ __forceinline__ float rebase(float from, float to, float c) { return fmaxf((from - to) * c, -300.0f); }

__device__ __forceinline__ RowSums join(RowSums a, RowSums b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float da = rebase(a.m, m, c), db = rebase(b.m, m, c);
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  return RowSums{m, a.s0 * fa + b.s0 * fb, (a.s1 + a.s0 * da) * fa + (b.s1 + b.s0 * db) * fb};
}

// Whole numbers in the order of the logits; 0 for none.  +0 and -0 are equal,
// NaN is no alternative.
__device__ __forceinline__ uint32_t orderOf(float x) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, x + 0.0f); // -0 + 0 = +0
  return x != x ? 0u : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float valueOf(uint32_t order) {
  return __builtin_bit_cast(float, (order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t keyOf(float x, uint32_t place) {
  return (uint64_t(orderOf(x)) << 32) | (0xffffffffu - place);
}
__device__ __forceinline__ uint32_t placeOf(uint64_t key) { return 0xffffffffu - static_cast<uint32_t>(key); }

__device__ __forceinline__ int64_t tokenAt(const void* tokens, int type, uint64_t row) {
  if (type == POLAR_HIP_INDEX_I64) return static_cast<const int64_t*>(tokens)[row];
  if (type == POLAR_HIP_INDEX_I32) return static_cast<const int32_t*>(tokens)[row];
  const float f = static_cast<const float*>(tokens)[row];
  // anything that is not a whole number in range is out of range; -1 is not counted
  return f < 0.0f ? -1 : f < 16777216.0f && f == truncf(f) ? static_cast<int64_t>(f) : int64_t(1) << 40;
}

// The `wanted` largest of `count` distinct keys in LDS, in order: each key's
// place is the number of larger ones.  emit(place, key, index).
template <typename F>
__device__ __forceinline__ void rankKeys(const uint64_t* keys, uint32_t count, uint32_t wanted, F emit) {
  for (uint32_t e = threadIdx.x; e < count; e += kBlock) {
    const uint64_t mine = keys[e];
    uint32_t above = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < count; ++i) above += keys[i] > mine;
    if (above < wanted) emit(above, mine, e);
  }
}

// A lower bound, as an order number, of the `wanted`-th best of the work-group's
// values: the wanted-th best of 64 groups of them (a lane of each wave; `order` is
// the best a lane has, 0 if it has none), with the bits behind the first kBits
// cleared.  The first wave finds it bit by bit, counting with a ballot the groups
// that reach a candidate.  The group maxima of random data let 24 values pass for
// 20 wanted, 44 for 32; telling all 256 lanes apart would let fewer pass but takes
// three times the instructions, and a wave that works alone issues one in ten
// cycles.
struct BoundScratch {
  uint32_t lanes[kBlock];
  uint32_t bound;
};
template <int kBits> __device__ __forceinline__ uint32_t laneBound(uint32_t order, uint32_t wanted, BoundScratch& lds) {
  lds.lanes[threadIdx.x] = order;
  __syncthreads();
  if (threadIdx.x < 64) {
    uint32_t mine = order;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mine = max(mine, lds.lanes[w * 64 + threadIdx.x]);
    uint32_t bound = 0;
#pragma unroll 1 // code that runs once per work-group is mostly waited for: short is fast
    for (uint32_t bit = 0x80000000u; bit != (1u << (31 - kBits)); bit >>= 1)
      bound = static_cast<uint32_t>(__popcll(__ballot(mine >= (bound | bit)))) >= wanted ? bound | bit : bound;
    if (threadIdx.x == 0) lds.bound = bound;
  }
  __syncthreads();
  return lds.bound;
}

struct ForwardArgs {
  const void* logits;
  uint64_t stride;
  const void* tokens;
  int tokenType;
  float scale;
  float *logprob, *stats, *entropy;
  int32_t* topIndex;
  float* topLogprob;
  uint32_t top, cols, parts, tilesPerPart;
  uint64_t firstRow;
  // parts > 1: a slot per part, and per row how many of its work-groups have
  // written theirs (all zero when the kernel starts)
  unsigned char* slots;
  uint32_t slotBytes;
  uint32_t* arrived;
};

// A row's given token and its logit, loaded by one lane before the row streams by.
struct Given {
  int64_t token;
  float logit;
};
template <typename T> __device__ __forceinline__ Given givenOf(const ForwardArgs& a, uint64_t row) {
  Given g{-1, 0.0f};
  if (threadIdx.x == 0 && a.logprob != nullptr) {
    g.token = tokenAt(a.tokens, a.tokenType, row);
    if (g.token >= 0 && g.token < int64_t(a.cols))
      g.logit = T::widen((static_cast<const typename T::Stored*>(a.logits) + row * a.stride)[g.token]);
  }
  return g;
}

// The row's answers, from its joined sums and its best keys in LDS.
__device__ __forceinline__ void finishRow(const ForwardArgs& a, uint64_t row, Given given, RowSums r, const uint64_t* best) {
  const float logsum = logf(r.s0); // -infinity where every logit is
  const bool none = r.s0 == 0.0f;
  if (threadIdx.x == 0) {
    if (a.stats != nullptr) {
      a.stats[2 * row] = r.m;
      a.stats[2 * row + 1] = logsum;
    }
    if (a.entropy != nullptr) a.entropy[row] = none ? 0.0f : kLn2 * (log2f(r.s0) - r.s1 / r.s0);
    if (a.logprob != nullptr) {
      float lp = 0.0f;
      if (given.token >= int64_t(a.cols))
        lp = __builtin_nanf("");
      else if (given.token >= 0)
        lp = none ? -__builtin_inff() : (given.logit - r.m) * a.scale - logsum;
      a.logprob[row] = lp;
    }
  }
  if (threadIdx.x < a.top) {
    const uint64_t key = best[threadIdx.x];
    const bool valid = key != 0 && r.s0 == r.s0; // a NaN among the sums: no order
    const float v = valueOf(static_cast<uint32_t>(key >> 32));
    a.topIndex[row * a.top + threadIdx.x] = valid ? static_cast<int32_t>(placeOf(key)) : -1;
    a.topLogprob[row * a.top + threadIdx.x] =
        !valid ? __builtin_nanf("") : none ? -__builtin_inff() : (v - r.m) * a.scale - logsum;
  }
}

// ---- parts of a row --------------------------------------------------------------
// The work-group that finishes its part last joins the row: no second launch.  A
// part's answer goes into a slot of whole 128-byte lines of its own (sums, then its
// best keys) with stores that are visible to the whole device (written through the
// XCD's L2), is acknowledged, and only then counted.  No fence: writing back and
// invalidating an L2 per work-group costs far more than all of this (64 rows of
// 131072 in sixteen parts, when it was taken: 33 us with fences, 18 so).  A second
// kernel for the join was faster there (15) and slower for eight rows (15, against
// 13.5 so), which is the call that waits on every token; the one launch was kept
// for those.  Since then 64 rows take eight parts, 14.0 us, and would take 16.4 in
// sixteen; a second kernel was not measured again.
constexpr uint32_t kSumsBytes = 16;
template <typename V> __device__ __forceinline__ void putPart(unsigned char* at, V value) {
  __hip_atomic_store(reinterpret_cast<V*>(at), value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V> __device__ __forceinline__ V takePart(const unsigned char* at) {
  return __hip_atomic_load(reinterpret_cast<const V*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ uint64_t partKey(const unsigned char* slots, uint32_t slotBytes, uint32_t top, uint32_t e) {
  return takePart<uint64_t>(slots + uint64_t(e / top) * slotBytes + kSumsBytes + e % top * sizeof(uint64_t));
}

// The row's parts joined, in every wave by itself: a lane per part.
__device__ __forceinline__ RowSums joinSums(const unsigned char* slots, uint32_t slotBytes, uint32_t parts, float c) {
  RowSums r{-__builtin_inff(), 0.0f, 0.0f};
  for (uint32_t p = threadIdx.x % 64; p < parts; p += 64) {
    const unsigned char* at = slots + uint64_t(p) * slotBytes;
    const RowSums part{takePart<float>(at), takePart<float>(at + 4), takePart<float>(at + 8)};
    r = p < 64 ? part : join(r, part, c);
  }
  const float m = waveMax(r.m);
  const float d = rebase(r.m, m, c), f = __builtin_amdgcn_exp2f(d);
  return RowSums{m, waveSum(r.s0 * f), waveSum((r.s1 + r.s0 * d) * f)};
}

// The `top` best of the parts' keys (0 for none) into `best`: those that reach the
// bound that the lanes' best ones give, ranked.  Where these are too many (logits
// that are equal all over the row) stretches of the keys are ranked together with the
// best so far.  `first`: the key of the lane's own number; `keys` has room for kJoinKeys.
constexpr uint32_t kJoinKeys = kMaxListed;
template <typename T>
__device__ __forceinline__ void joinKeys(const unsigned char* slots, uint32_t slotBytes, uint32_t parts, uint32_t top,
                                         uint64_t first, uint64_t* keys, uint64_t* best, BoundScratch& scratch,
                                         uint32_t* listed) {
  const uint32_t all = parts * top;
  auto keyAt = [&](uint32_t e) { return partKey(slots, slotBytes, top, e); };
  uint64_t mine = first;
  for (uint32_t e = threadIdx.x + kBlock; e < all; e += kBlock) mine = keyAt(e) > mine ? keyAt(e) : mine;
  if (threadIdx.x == 0) *listed = 0;
  const uint32_t least = laneBound<T::kOrderBits>(static_cast<uint32_t>(mine >> 32), top, scratch);
  for (uint32_t e = threadIdx.x; e < all; e += kBlock) {
    const uint64_t key = e < kBlock ? first : keyAt(e);
    if (key != 0 && static_cast<uint32_t>(key >> 32) >= least) {
      const uint32_t at = atomicAdd(listed, 1u);
      if (at < kJoinKeys) keys[at] = key;
    }
  }
  if (threadIdx.x < kMaxTop) best[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t count = *listed;
  if (count <= kJoinKeys) { // uniform
    rankKeys(keys, count, top, [&](uint32_t rank, uint64_t key, uint32_t) { best[rank] = key; });
  } else {
    for (uint32_t at = 0; at < all; at += kJoinKeys - kMaxTop) {
      const uint32_t n = all - at < kJoinKeys - kMaxTop ? all - at : kJoinKeys - kMaxTop;
      __syncthreads();
      for (uint32_t e = threadIdx.x; e < n; e += kBlock) keys[e] = keyAt(at + e);
      if (threadIdx.x < top) keys[n + threadIdx.x] = best[threadIdx.x];
      __syncthreads();
      if (threadIdx.x < kMaxTop) best[threadIdx.x] = 0;
      __syncthreads();
      // empty places (key 0) are not distinct, but rank below every logit
      rankKeys(keys, n + top, top, [&](uint32_t rank, uint64_t key, uint32_t) {
        if (key != 0) best[rank] = key;
      });
    }
  }
  __syncthreads();
}

template <typename T, bool kEntropy, bool kTop>
__global__ __launch_bounds__(kBlock, 5) void logprobKernel(ForwardArgs a) {
  constexpr int kVec = T::kVec;
  constexpr int kLane = kPacks * kVec; // logits of a lane per tile
  constexpr uint32_t kTile = tileCols<T>();
  using Stored = typename T::Stored;
  __shared__ RowSums waveSums[kWaves];
  __shared__ uint64_t waveBound[kWaves];
  __shared__ BoundScratch scratch;
  __shared__ uint32_t listed, found;
  // segment maxima while the row streams by, then the listed segments' keys, then the logits' keys
  __shared__ __align__(16) unsigned char area[kTop ? kMaxListed * sizeof(uint64_t) : 16];
  __shared__ uint16_t list[kTop ? kMaxListed : 1];
  __shared__ uint16_t kept[kTop ? kMaxTop : 1];
  __shared__ uint64_t best[kTop ? kMaxTop : 1];
  static_assert(kMaxListed * sizeof(uint64_t) >= kMaxTiles * kBlock * sizeof(float), "segment maxima fit");
  static_assert(kMaxListed >= kShortList * kLane && kMaxListed >= kMaxTop * kLane, "the looked-at segments' logits fit");
  static_assert(kStagedAt + kShortList * kPacks * sizeof(Pack) <= kMaxListed * sizeof(uint64_t), "staged packs fit");

  const uint64_t row = a.firstRow + blockIdx.x / a.parts;
  const uint32_t part = blockIdx.x % a.parts;
  const Stored* x = static_cast<const Stored*>(a.logits) + row * a.stride;
  const uint32_t begin = part * a.tilesPerPart * kTile;
  const uint32_t end = a.cols - begin > a.tilesPerPart * kTile ? begin + a.tilesPerPart * kTile : a.cols;
  const uint32_t tiles = (end - begin + kTile - 1) / kTile;
  const float c = a.scale * kLog2e;
  const Stored kNothing = static_cast<Stored>(-__builtin_inff());
  float* segments = reinterpret_cast<float*>(area);
  const Given given = givenOf<T>(a, row); // by every part: any of them may be the last

  auto place = [&](uint32_t tile, int k, uint32_t lane) { return begin + tile * kTile + (k * kBlock + lane) * kVec; };

  // the wave's reference; a lane's sums of 2^(x c + shift), whose exponents lack `rest`:
  // the product's rounding error is the same for all of them and is put in at the end,
  // so that logits far from zero lose nothing against (x - reference) c
  float reference = -__builtin_inff(), limit = -__builtin_inff(), shift = 0.0f, rest = 0.0f;
  bool wide = false, masked = false; // of the whole wave
  float laneBest = -__builtin_inff(), s0 = 0.0f, s1 = 0.0f;
  uint32_t laneTile = 0;
  auto settle = [&](float to) { // sums relative to `to`
    if constexpr (kEntropy) s1 += rest * s0;
    const float d = rebase(reference, to, c), f = __builtin_amdgcn_exp2f(d + rest);
    if constexpr (kEntropy) s1 = (s1 + s0 * d) * f;
    s0 *= f;
  };
  Pack next[kPacks];
#pragma unroll
  for (int k = 0; k < kPacks; ++k) next[k] = loadPack<T>(x, place(0, k, threadIdx.x), end, kNothing);
  for (uint32_t tile = 0; tile < tiles; ++tile) {
    float v[kLane];
#pragma unroll
    for (int k = 0; k < kPacks; ++k) T::unpack(next[k], v + k * kVec);
    if (tile + 1 < tiles) {
#pragma unroll
      for (int k = 0; k < kPacks; ++k) next[k] = loadPack<T>(x, place(tile + 1, k, threadIdx.x), end, kNothing);
    }
    float most = v[0];
#pragma unroll
    for (int i = 1; i < kLane; ++i) most = fmaxf(most, v[i]);
    if constexpr (kTop) {
      // a lane whose segment lies behind the end has none
      segments[tile * kBlock + threadIdx.x] = place(tile, 0, threadIdx.x) < end ? most : __builtin_nanf("");
      if (most > laneBest) laneTile = tile;
    }
    laneBest = fmaxf(laneBest, most);
    if (__any(most > limit)) {
      const float to = waveMax(laneBest);
      settle(to);
      reference = to;
      // far from zero `rest` is no small correction any more, and to * c may overflow (a row masked
      // with the type's lowest value): the difference is taken first, one instruction more per logit
      wide = fabsf(to) * fmaxf(c, 1.0f) > 0x1p20f;
      // there the next float above `to` may lie as far as 2^64 is: `to + 64 / c` would be rounded up
      // to it, and terms of up to 2^128 pass
      limit = wide ? to : to + 64.0f / c;
      shift = wide ? 0.0f : -to * c;
      rest = wide ? 0.0f : __builtin_fmaf(-to, c, -shift);
    }
    // (the empty asm statements keep the three loops apart: with what they have in common
    // merged in front of or behind the branches, all of a tile's exponentials would sit in
    // registers at once: 156 registers and three waves per SIMD instead of 80 and six)
    float t0 = 0.0f, t1 = 0.0f;
    if (wide) {
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        const float y = (v[i] - reference) * c, e = __builtin_amdgcn_exp2f(y);
        t0 += e;
        if constexpr (kEntropy) t1 = __builtin_fmaf(e, fmaxf(y, -160.0f), t1);
      }
      asm volatile("" : "+v"(t0), "+v"(t1));
    } else if (kEntropy && masked) {
      float factor = c;
      asm volatile("" : "+v"(factor));
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        const float y = __builtin_fmaf(v[i], factor, shift), e = __builtin_amdgcn_exp2f(y);
        t0 += e;
        t1 = __builtin_fmaf(e, fmaxf(y, -160.0f), t1);
      }
      asm volatile("" : "+v"(t0), "+v"(t1));
    } else {
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        const float y = __builtin_fmaf(v[i], c, shift), e = __builtin_amdgcn_exp2f(y); // 0 below 2^-149, NaN for NaN
        t0 += e;
        if constexpr (kEntropy) t1 = __builtin_fmaf(e, y, t1);
      }
      asm volatile("" : "+v"(t0), "+v"(t1));
      if constexpr (kEntropy) {
        // 0 * -infinity is no term: from the first one on the wave clamps its exponents
        masked = __any(t1 != t1);
        if (masked) {
          t1 = 0.0f;
          float again = c; // opaque: this loop happens once per wave and is not to be merged into the one above
          asm volatile("" : "+v"(again));
#pragma unroll
          for (int i = 0; i < kLane; ++i) {
            const float y = __builtin_fmaf(v[i], again, shift);
            t1 = __builtin_fmaf(__builtin_amdgcn_exp2f(y), fmaxf(y, -160.0f), t1);
          }
        }
      }
    }
    s0 += t0;
    if constexpr (kEntropy) s1 += t1;
  }

  // lanes, then waves
  {
    const float m = waveMax(laneBest);
    settle(m);
    const float sum1 = kEntropy ? waveSum(s1) : 0.0f, sum0 = waveSum(s0);
    if (threadIdx.x % 64 == 0) waveSums[threadIdx.x / 64] = RowSums{m, sum0, sum1};
  }

  if constexpr (kTop) {
    uint64_t* keys = reinterpret_cast<uint64_t*>(area);
    const bool some = place(0, 0, threadIdx.x) < end;
    if (threadIdx.x == 0) listed = found = 0;
    const uint32_t least = laneBound<T::kOrderBits>(some ? orderOf(laneBest) : 0u, a.top, scratch);
    auto listSegments = [&](uint32_t from) { // those whose maximum's order is not below `from`
#pragma unroll 4
      for (uint32_t tile = 0; tile < tiles; ++tile) {
        const uint32_t order = orderOf(segments[tile * kBlock + threadIdx.x]);
        if (order >= from && order != 0) {
          const uint32_t at = atomicAdd(&listed, 1u);
          if (at < kMaxListed) list[at] = static_cast<uint16_t>(tile * kBlock + threadIdx.x);
        }
      }
    };
    // Few segments: their packs are looked at, one by each lane.  A part of one tile has them in registers
    // still and puts them into LDS (behind the keys) instead of loading them again.
    Pack* staged = reinterpret_cast<Pack*>(area + kStagedAt);
    if (orderOf(laneBest) >= least) {
      if (tiles > 1) {
        listSegments(least);
      } else if (some) {
        const uint32_t at = atomicAdd(&listed, 1u);
        if (at < kShortList) {
          list[at] = static_cast<uint16_t>(threadIdx.x);
#pragma unroll
          for (int k = 0; k < kPacks; ++k) staged[at * kPacks + k] = next[k];
        }
      }
    }
    __syncthreads();
    bool exact = listed > kShortList; // uniform: too many reach the bound
    if (!exact) {
      const uint32_t lowest = orderOf(-__builtin_inff());
      const float low = least <= lowest ? -__builtin_inff() : valueOf(least); // orders below -infinity's are no numbers
      const uint32_t room = tiles > 1 ? kMaxListed : kStagedAt / sizeof(uint64_t), segmentsListed = listed;
      if (tiles == 1) { // an element per lane: short code
        const Stored* elements = reinterpret_cast<const Stored*>(staged);
#pragma unroll 1
        for (uint32_t e = threadIdx.x; e < segmentsListed * kLane; e += kBlock) {
          const float w = T::widen(elements[e]);
          const uint32_t at = place(0, e % kLane / kVec, list[e / kLane]) + e % kVec;
          if (w >= low && at < end) {
            const uint32_t slot = atomicAdd(&found, 1u);
            if (slot < room) keys[slot] = keyOf(w, at);
          }
        }
      } else { // a pack per lane: one load
        for (uint32_t e = threadIdx.x; e < segmentsListed * kPacks; e += kBlock) {
          const uint32_t segment = list[e / kPacks];
          const uint32_t from = place(segment / kBlock, e % kPacks, segment % kBlock);
          float w[kVec];
          T::unpack(loadPack<T, false>(x, from, end, kNothing), w);
          uint32_t n = 0;
#pragma unroll
          for (int i = 0; i < kVec; ++i) n += w[i] >= low && from + i < end;
          if (n == 0) continue;
          uint32_t at = atomicAdd(&found, n);
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (w[i] >= low && from + i < end) keys[at++] = keyOf(w[i], from + i);
        }
      }
      __syncthreads();
      exact = found > room;
      if (exact) { // of one tile; the keys lie where the maxima were
        __syncthreads();
        segments[threadIdx.x] = some ? laneBest : __builtin_nanf("");
      }
    }
    if (exact) {
      const uint16_t* looked = list;
      // first place of a segment's maximum
      auto segmentKey = [&](uint32_t tile, uint32_t lane, float most) {
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int k = kPacks - 1; k >= 0; --k) {
          float w[kVec];
          T::unpack(loadPack<T, false>(x, place(tile, k, lane), end, kNothing), w);
#pragma unroll
          for (int i = kVec - 1; i >= 0; --i) {
            const uint32_t p = place(tile, k, lane) + i;
            if (p < end && w[i] == most) at = p;
          }
        }
        return at == 0xffffffffu ? 0ull : keyOf(most, at);
      };
      // the wave's k-th best lane: a bitonic network over the 64 lanes' best keys
      const uint32_t lane = threadIdx.x % 64;
      const uint64_t laneKey = segmentKey(laneTile, threadIdx.x, laneBest);
      uint64_t sorted = laneKey;
#pragma unroll
      for (uint32_t size = 2; size <= 64; size *= 2) {
#pragma unroll
        for (uint32_t gap = size / 2; gap > 0; gap /= 2) {
          const uint64_t other = __shfl_xor(sorted, gap, 64);
          const bool larger = ((lane & size) == 0) == ((lane & gap) == 0); // descending over the whole wave
          sorted = (other > sorted) == larger ? other : sorted;
        }
      }
      const uint64_t bound1 = __shfl(sorted, a.top - 1, 64);
      if (lane == 0) waveBound[threadIdx.x / 64] = bound1;
      __syncthreads(); // everyone has read the first list's length
      if (threadIdx.x == 0) listed = found = 0;
      __syncthreads();
      uint64_t bound = waveBound[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) bound = bound > waveBound[w] ? bound : waveBound[w];
      // of at most k lanes per wave the segments that may reach the bound: at most kMaxListed
      if (laneKey != 0 && laneKey >= bound) listSegments(static_cast<uint32_t>(bound >> 32));
      __syncthreads(); // the list is whole, and the maxima are not needed any more
      uint32_t count = listed;
      if (count > a.top) {
        for (uint32_t e = threadIdx.x; e < count; e += kBlock) {
          const uint32_t tile = list[e] / kBlock, owner = list[e] % kBlock;
          float most = -__builtin_inff();
#pragma unroll
          for (int k = 0; k < kPacks; ++k) {
            float w[kVec];
            T::unpack(loadPack<T, false>(x, place(tile, k, owner), end, kNothing), w);
#pragma unroll
            for (int i = 0; i < kVec; ++i) most = fmaxf(most, w[i]);
          }
          // without a logit: a key below all others, and no two alike
          const uint64_t key = segmentKey(tile, owner, most);
          keys[e] = key != 0 ? key : e;
        }
        __syncthreads();
        rankKeys(keys, count, a.top, [&](uint32_t rank, uint64_t key, uint32_t e) {
          kept[rank] = list[e];
          best[rank] = key;
        });
        __syncthreads(); // also: the segments' keys are read
        bound = bound > best[a.top - 1] ? bound : best[a.top - 1];
        count = a.top;
        looked = kept;
      }
      for (uint32_t e = threadIdx.x; e < count * kPacks; e += kBlock) {
        const uint32_t segment = looked[e / kPacks];
        const uint32_t from = place(segment / kBlock, e % kPacks, segment % kBlock);
        float w[kVec];
        T::unpack(loadPack<T, false>(x, from, end, kNothing), w);
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          if (from + i < end && w[i] == w[i] && keyOf(w[i], from + i) >= bound)
            keys[atomicAdd(&found, 1u)] = keyOf(w[i], from + i);
      }
    }
    __syncthreads();
    if (threadIdx.x < kMaxTop) best[threadIdx.x] = 0;
    __syncthreads();
    rankKeys(keys, found, a.top, [&](uint32_t rank, uint64_t key, uint32_t) { best[rank] = key; });
  }
  __syncthreads();
  RowSums total = waveSums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) total = join(total, waveSums[w], c);
  if (a.parts > 1) {
    const uint32_t rowInLaunch = blockIdx.x / a.parts;
    if (threadIdx.x < 64) { // all that is written is this wave's, and it waits for it
      unsigned char* slot = a.slots + uint64_t(blockIdx.x) * a.slotBytes;
      if (threadIdx.x == 0) putPart(slot, total.m), putPart(slot + 4, total.s0), putPart(slot + 8, total.s1);
      if (kTop && threadIdx.x < a.top) putPart(slot + kSumsBytes + threadIdx.x * sizeof(uint64_t), best[threadIdx.x]);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (threadIdx.x == 0)
        listed = __hip_atomic_fetch_add(&a.arrived[rowInLaunch], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == a.parts;
    }
    __syncthreads();
    if (listed == 0) return; // the whole work-group
    if (threadIdx.x == 0) __hip_atomic_store(&a.arrived[rowInLaunch], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const unsigned char* slots = a.slots + uint64_t(rowInLaunch) * a.parts * a.slotBytes;
    uint64_t first = 0; // on its way while the sums are joined
    if (kTop && threadIdx.x < a.parts * a.top) first = partKey(slots, a.slotBytes, a.top, threadIdx.x);
    total = joinSums(slots, a.slotBytes, a.parts, c);
    if constexpr (kTop)
      joinKeys<T>(slots, a.slotBytes, a.parts, a.top, first, reinterpret_cast<uint64_t*>(area), best, scratch, &found);
  }
  finishRow(a, row, given, total, best);
}

// ---- gradient ----------------------------------------------------------------------

struct GradArgs {
  const void* logits;
  uint64_t stride;
  const void* tokens;
  int tokenType;
  float scale;
  const float *stats, *dlogprob, *entropy, *dentropy;
  void* dlogits;
  uint64_t dlogitsStride, rows;
  uint32_t cols, chunks;
};

// 128 lanes of two packs: 8192 x 32768 bf16 166 us (6.45 TB/s; a copy of the same bytes 157), with 256
// lanes 169, with one pack 171 to 177, with four 179
constexpr int kGradBlock = 128;
constexpr int kGradPacks = 2;
template <typename T, bool kEntropy>
__global__ __launch_bounds__(kGradBlock) void logprobGradKernel(GradArgs a) {
  constexpr int kVec = T::kVec;
  const uint64_t row = blockIdx.x / a.chunks;
  const uint32_t first = (blockIdx.x % a.chunks) * (kGradBlock * kGradPacks * kVec);
  const typename T::Stored* x = static_cast<const typename T::Stored*>(a.logits) + row * a.stride;
  typename T::Stored* dx = static_cast<typename T::Stored*>(a.dlogits) + row * a.dlogitsStride;
  Pack in[kGradPacks];
#pragma unroll
  for (int k = 0; k < kGradPacks; ++k)
    in[k] = loadPack<T>(x, first + (k * kGradBlock + threadIdx.x) * kVec, a.cols, typename T::Stored(0.0f));
  const float m = a.stats[2 * row], logsum = a.stats[2 * row + 1];
  const bool none = logsum == -__builtin_inff();
  const int64_t token = a.dlogprob != nullptr ? tokenAt(a.tokens, a.tokenType, row) : -1;
  float g = token >= 0 && !none ? a.dlogprob[row] * a.scale : 0.0f;
  if (token >= int64_t(a.cols)) g = __builtin_nanf("");
  float h = 0.0f, entropy = 0.0f;
  if constexpr (kEntropy) h = none ? 0.0f : a.dentropy[row] * a.scale, entropy = a.entropy[row];
  const float c = a.scale * kLog2e, logsum2 = logsum * kLog2e;
#pragma unroll
  for (int k = 0; k < kGradPacks; ++k) {
    const uint32_t at = first + (k * kGradBlock + threadIdx.x) * kVec;
    if (at >= a.cols) continue;
    float v[kVec];
    T::unpack(in[k], v);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float y = __builtin_fmaf(v[i] - m, c, -logsum2); // log2 p
      const float p = none ? 0.0f : __builtin_amdgcn_exp2f(y);
      float d = -p * g;
      // a masked logit has no share in the entropy: 0 * -infinity is no term
      if constexpr (kEntropy) d -= p * __builtin_fmaf(fmaxf(y, -160.0f), kLn2, entropy) * h;
      v[i] = d;
    }
    const int64_t here = token - int64_t(at);
    if (here >= 0 && here < kVec) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] += here == i ? g : 0.0f;
    }
    storePack<T>(dx, at, a.cols, v);
  }
}

// `reserved`: bytes at the workspace's beginning that are the caller's (who holds the lock); where there
// are any, stats go to them.
template <typename T> int forward(polar_hip_device* dev, ForwardArgs a, uint64_t rows, uint64_t reserved = 0) {
  const uint32_t tiles = (a.cols + tileCols<T>() - 1) / tileCols<T>();
  // parts: at most kMaxTiles tiles each, and enough of them for two work-groups per CU (64 rows of 131072
  // bf16 with 20 alternatives: 14.0 us, with four per CU 16.4; 512 rows 28.5, 32 and with eight 40; eight rows
  // have a part per tile, 11, whichever it is)
  const uint64_t groups = 2ull * dev->info.compute_units;
  const uint64_t wanted = std::max<uint64_t>((tiles + kMaxTiles - 1) / kMaxTiles, groups / std::max<uint64_t>(rows, 1));
  a.tilesPerPart = static_cast<uint32_t>((tiles + std::min<uint64_t>(wanted, tiles) - 1) / std::min<uint64_t>(wanted, tiles));
  a.parts = (tiles + a.tilesPerPart - 1) / a.tilesPerPart;
  const bool entropy = a.entropy != nullptr, top = a.top != 0;
  auto kernel = entropy ? (top ? logprobKernel<T, true, true> : logprobKernel<T, true, false>)
                        : (top ? logprobKernel<T, false, true> : logprobKernel<T, false, false>);
  // rows per launch: lanes in 32 bits, parts' slots in 64 MiB of workspace, a counter per row
  a.slotBytes = static_cast<uint32_t>((kSumsBytes + a.top * sizeof(uint64_t) + 127) / 128 * 128);
  uint64_t batch = kMostGroups / a.parts;
  if (a.parts > 1)
    batch = std::min({batch, uint64_t(kTileCounters), std::max<uint64_t>(1, (64ull << 20) / (uint64_t(a.parts) * a.slotBytes))});
  void* area = nullptr;
  if (reserved != 0 || a.parts > 1) {
    const int st = workspaceFor(dev, reserved + (a.parts > 1 ? std::min(batch, rows) * a.parts * a.slotBytes : 0), &area);
    if (st != POLAR_HIP_OK) return st;
    a.slots = static_cast<unsigned char*>(area) + reserved;
    a.arrived = dev->tileCounters;
    if (reserved != 0) a.stats = static_cast<float*>(area);
  }
  for (uint64_t r = 0; r < rows; r += batch) {
    const uint64_t n = std::min(batch, rows - r);
    a.firstRow = r;
    POLAR_HIP_TRY(launchKernel(dev, kernel, dim3(static_cast<unsigned>(n * a.parts)), dim3(kBlock), a));
  }
  return POLAR_HIP_OK;
}

template <typename T> int backward(polar_hip_device* dev, GradArgs a) {
  constexpr uint32_t kChunk = kGradBlock * kGradPacks * T::kVec;
  a.chunks = (a.cols + kChunk - 1) / kChunk;
  auto kernel = a.dentropy != nullptr ? logprobGradKernel<T, true> : logprobGradKernel<T, false>;
  std::unique_lock<std::mutex> lock(dev->workspaceMu, std::defer_lock);
  if (a.stats == nullptr) { // a forward pass for the stats alone
    ForwardArgs f{};
    f.logits = a.logits, f.stride = a.stride, f.scale = a.scale, f.cols = a.cols;
    lock.lock(); // until the kernels that use the workspace are enqueued
    const int st = forward<T>(dev, f, a.rows, (a.rows * 2 * sizeof(float) + 255) / 256 * 256);
    if (st != POLAR_HIP_OK) return st;
    a.stats = static_cast<const float*>(dev->workspace);
  }
  const uint64_t batch = kMostGroups / a.chunks, rows = a.rows;
  GradArgs part = a;
  for (uint64_t r = 0; r < rows; r += batch) {
    const uint64_t n = std::min(batch, rows - r);
    POLAR_HIP_TRY(launchKernel(dev, kernel, dim3(static_cast<unsigned>(n * a.chunks)), dim3(kGradBlock), part));
    if (r + n == rows) break;
    const uint64_t tokenBytes = a.tokenType == POLAR_HIP_INDEX_I64 ? 8 : 4;
    part.logits = static_cast<const typename T::Stored*>(part.logits) + n * a.stride;
    part.dlogits = static_cast<typename T::Stored*>(part.dlogits) + n * a.dlogitsStride;
    part.stats += 2 * n;
    if (part.tokens) part.tokens = static_cast<const char*>(part.tokens) + n * tokenBytes;
    if (part.dlogprob) part.dlogprob += n;
    if (part.entropy) part.entropy += n;
    if (part.dentropy) part.dentropy += n;
  }
  return POLAR_HIP_OK;
}

bool knownIndex(int type) {
  return type == POLAR_HIP_INDEX_I32 || type == POLAR_HIP_INDEX_I64 || type == POLAR_HIP_INDEX_F32;
}

} // namespace

extern "C" {

int polar_hip_flogprob(polar_hip_device* dev, int type, const void* logits, uint64_t stride, int tokenType,
                       const void* tokens, float scale, float* logprob, float* stats, float* entropy, uint32_t top,
                       int32_t* topIndex, float* topLogprob, uint64_t rows, uint64_t cols) {
  POLAR_HIP_REQUIRE(dev != nullptr, "dev is null");
  POLAR_HIP_REQUIRE(knownType(type), "unknown element type");
  POLAR_HIP_REQUIRE(knownIndex(tokenType), "unknown token type");
  POLAR_HIP_REQUIRE(cols >= 1 && cols <= kMaxCols, "rows of 1 to 2^24 logits");
  POLAR_HIP_REQUIRE(scale >= kLeastScale && scale <= kMostScale, "scale must lie between 2^-64 and 2^64");
  POLAR_HIP_REQUIRE(top <= POLAR_HIP_LOGPROB_MAX_TOP && top <= cols, "too many alternatives");
  if (rows == 0) return POLAR_HIP_OK;
  POLAR_HIP_REQUIRE(logits != nullptr, "null tensor");
  POLAR_HIP_REQUIRE(logprob == nullptr || tokens != nullptr, "log probabilities need tokens");
  POLAR_HIP_REQUIRE(top == 0 || (topIndex && topLogprob), "null tensor for the alternatives");
  POLAR_HIP_REQUIRE(stride >= cols, "a row's stride is shorter than the row");
  POLAR_HIP_REQUIRE(addressable(rows, stride, sizeOf(type)), "tensor too large");
  POLAR_HIP_REQUIRE(alignedTo(logits, sizeOf(type)) && alignedTo(tokens, tokenType == POLAR_HIP_INDEX_I64 ? 8 : 4) &&
                        alignedTo(logprob, 4) && alignedTo(stats, 4) && alignedTo(entropy, 4) &&
                        alignedTo(topIndex, 4) && alignedTo(topLogprob, 4),
                    "misaligned pointer");
  if (logprob == nullptr && stats == nullptr && entropy == nullptr && top == 0) return POLAR_HIP_OK;
  POLAR_HIP_TRY(hipSetDevice(dev->ordinal));
  ForwardArgs a{};
  a.logits = logits, a.stride = stride, a.tokens = tokens, a.tokenType = tokenType, a.scale = scale;
  a.logprob = logprob, a.stats = stats, a.entropy = entropy, a.topIndex = topIndex, a.topLogprob = topLogprob;
  a.top = top, a.cols = static_cast<uint32_t>(cols);
  std::lock_guard<std::mutex> lock(dev->workspaceMu);
  return type == POLAR_HIP_F32   ? forward<TypeF32>(dev, a, rows)
         : type == POLAR_HIP_F16 ? forward<TypeF16>(dev, a, rows)
                                 : forward<TypeBF16>(dev, a, rows);
}

int polar_hip_flogprob_grad(polar_hip_device* dev, int type, const void* logits, uint64_t stride, int tokenType,
                            const void* tokens, float scale, const float* stats, const float* dlogprob,
                            const float* entropy, const float* dentropy, void* dlogits, uint64_t dlogitsStride,
                            uint64_t rows, uint64_t cols) {
  POLAR_HIP_REQUIRE(dev != nullptr, "dev is null");
  POLAR_HIP_REQUIRE(knownType(type), "unknown element type");
  POLAR_HIP_REQUIRE(knownIndex(tokenType), "unknown token type");
  POLAR_HIP_REQUIRE(cols >= 1 && cols <= kMaxCols, "rows of 1 to 2^24 logits");
  POLAR_HIP_REQUIRE(scale >= kLeastScale && scale <= kMostScale, "scale must lie between 2^-64 and 2^64");
  if (rows == 0) return POLAR_HIP_OK;
  POLAR_HIP_REQUIRE(logits && dlogits, "null tensor");
  POLAR_HIP_REQUIRE(dlogprob == nullptr || tokens != nullptr, "log probabilities need tokens");
  POLAR_HIP_REQUIRE(dentropy == nullptr || entropy != nullptr, "the entropy's gradient needs the entropy");
  POLAR_HIP_REQUIRE(stride >= cols && dlogitsStride >= cols, "a row's stride is shorter than the row");
  POLAR_HIP_REQUIRE(addressable(rows, std::max(stride, dlogitsStride), sizeOf(type)), "tensor too large");
  POLAR_HIP_REQUIRE(alignedTo(logits, sizeOf(type)) && alignedTo(dlogits, sizeOf(type)) &&
                        alignedTo(tokens, tokenType == POLAR_HIP_INDEX_I64 ? 8 : 4) && alignedTo(stats, 4) &&
                        alignedTo(dlogprob, 4) && alignedTo(entropy, 4) && alignedTo(dentropy, 4),
                    "misaligned pointer");
  POLAR_HIP_REQUIRE(logits != dlogits || stride == dlogitsStride, "in place needs equal strides");
  POLAR_HIP_TRY(hipSetDevice(dev->ordinal));
  GradArgs a{};
  a.logits = logits, a.stride = stride, a.tokens = tokens, a.tokenType = tokenType, a.scale = scale;
  a.stats = stats, a.dlogprob = dlogprob, a.entropy = entropy, a.dentropy = dentropy;
  a.dlogits = dlogits, a.dlogitsStride = dlogitsStride, a.rows = rows, a.cols = static_cast<uint32_t>(cols);
  return type == POLAR_HIP_F32   ? backward<TypeF32>(dev, a)
         : type == POLAR_HIP_F16 ? backward<TypeF16>(dev, a)
                                 : backward<TypeBF16>(dev, a);
}

} // extern "C"
