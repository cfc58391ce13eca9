// Log probabilities of given tokens, entropy and the likeliest alternatives of
// rows of logits, and the gradient of the first two.
//
//   m = max x,  z_j = s (x_j - m),  S0 = sum e^z,  S1 = sum z e^z,  logsum = ln S0
//   logprob = z_t - logsum,   entropy = logsum - S1 / S0
//   dx_j = s (g (1[j = t] - p_j) - h p_j (ln p_j + entropy)),   p_j = e^(z_j - logsum)
//
// The forward pass reads the logits once.  Each lane keeps a running maximum
// and both sums relative to it, in base 2, and rescales the sums once per tile
// of up to 32 logits; lanes, waves and parts of a row are joined the same way.
// Alternatives cost next to nothing while the row streams by: a lane notes the
// maximum of each of its tiles (a "segment") in LDS.  The k-th best of the
// lanes' maxima bounds the k-th best logit from below; only segments that reach
// the bound are looked at again, the k best of them are kept, and the k best
// logits lie in those.  Logits are compared as (value, place) with the lowest
// place first, an order without ties, so each list has a fixed bound whatever
// the data (a wave contributes at most k lanes, a lane 16 segments, a segment
// 32 logits) and the answer is the same on every run.
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
constexpr int kMaxListed = kWaves * kMaxTop * kMaxTiles;  // segments that can reach the bound
constexpr uint64_t kMaxCols = 1ull << 24;                 // places are exact as fp32 tokens
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

template <typename T> constexpr uint32_t tileCols() { return kBlock * kPacks * T::kVec; }

// Sums relative to a maximum, exponents in base 2: s0 = sum 2^y, s1 = sum y 2^y
// with y = (x - m) c.
struct RowSums {
  float m, s0, s1;
};

// What a sum relative to `from` is multiplied by to be relative to `to` >= from,
// as an exponent; an empty sum's `from` is -infinity, and both may be.
__device__ __forceinline__ float rebase(float from, float to, float c) { return fmaxf((from - to) * c, -1e30f); }

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
    for (uint32_t i = 0; i < count; ++i) above += keys[i] > mine;
    if (above < wanted) emit(above, mine, e);
  }
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
  // parts > 1: [row][part] sums and [row][part][top] keys
  RowSums* partSums;
  uint64_t* partKeys;
};

// The row's answers, from its joined sums and its best keys in LDS.
template <typename T>
__device__ __forceinline__ void finishRow(const ForwardArgs& a, uint64_t row, RowSums r, const uint64_t* best) {
  const typename T::Stored* x = static_cast<const typename T::Stored*>(a.logits) + row * a.stride;
  const float logsum = logf(r.s0); // -infinity where every logit is
  const bool none = r.s0 == 0.0f;
  if (threadIdx.x == 0) {
    if (a.stats != nullptr) {
      a.stats[2 * row] = r.m;
      a.stats[2 * row + 1] = logsum;
    }
    if (a.entropy != nullptr) a.entropy[row] = none ? 0.0f : kLn2 * (log2f(r.s0) - r.s1 / r.s0);
    if (a.logprob != nullptr) {
      const int64_t t = tokenAt(a.tokens, a.tokenType, row);
      float lp = 0.0f;
      if (t >= int64_t(a.cols))
        lp = __builtin_nanf("");
      else if (t >= 0)
        lp = none ? -__builtin_inff() : (T::widen(x[t]) - r.m) * a.scale - logsum;
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

template <typename T, bool kEntropy, bool kTop>
__global__ __launch_bounds__(kBlock) void logprobKernel(ForwardArgs a) {
  constexpr int kVec = T::kVec;
  constexpr uint32_t kTile = tileCols<T>();
  using Stored = typename T::Stored;
  __shared__ RowSums waveSums[kWaves];
  __shared__ uint64_t waveBound[kWaves];
  __shared__ uint32_t listed, found;
  // segment maxima while the row streams by, then the listed segments' keys, then the logits' keys
  __shared__ __align__(16) unsigned char area[kTop ? kMaxListed * sizeof(uint64_t) : 16];
  __shared__ uint16_t list[kTop ? kMaxListed : 1];
  __shared__ uint16_t kept[kTop ? kMaxTop : 1];
  __shared__ uint64_t best[kTop ? kMaxTop : 1];
  static_assert(kMaxListed * sizeof(uint64_t) >= kMaxTiles * kBlock * sizeof(float), "segment maxima fit");
  static_assert(kMaxListed >= kMaxTop * kPacks * 8, "the kept segments' logits fit");

  const uint64_t row = a.firstRow + blockIdx.x / a.parts;
  const uint32_t part = blockIdx.x % a.parts;
  const Stored* x = static_cast<const Stored*>(a.logits) + row * a.stride;
  const uint32_t begin = part * a.tilesPerPart * kTile;
  const uint32_t end = a.cols - begin > a.tilesPerPart * kTile ? begin + a.tilesPerPart * kTile : a.cols;
  const uint32_t tiles = (end - begin + kTile - 1) / kTile;
  const float c = a.scale * kLog2e;
  const Stored kNothing = static_cast<Stored>(-__builtin_inff());
  float* segments = reinterpret_cast<float*>(area);

  auto place = [&](uint32_t tile, int k, uint32_t lane) { return begin + tile * kTile + (k * kBlock + lane) * kVec; };

  RowSums r{-__builtin_inff(), 0.0f, 0.0f};
  float laneBest = -__builtin_inff();
  uint32_t laneTile = 0;
  Pack next[kPacks];
#pragma unroll
  for (int k = 0; k < kPacks; ++k) next[k] = loadPack<T, false>(x, place(0, k, threadIdx.x), end, kNothing);
  for (uint32_t tile = 0; tile < tiles; ++tile) {
    float v[kPacks * kVec];
#pragma unroll
    for (int k = 0; k < kPacks; ++k) T::unpack(next[k], v + k * kVec);
    if (tile + 1 < tiles) {
#pragma unroll
      for (int k = 0; k < kPacks; ++k) next[k] = loadPack<T, false>(x, place(tile + 1, k, threadIdx.x), end, kNothing);
    }
    float most = v[0];
#pragma unroll
    for (int i = 1; i < kPacks * kVec; ++i) most = fmaxf(most, v[i]);
    if constexpr (kTop) {
      segments[tile * kBlock + threadIdx.x] = most;
      if (most > laneBest) laneBest = most, laneTile = tile;
    }
    const float m = fmaxf(r.m, most);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    // y = x c - base c as one fused multiply-add; the rounding error of base c is
    // the same for the whole tile and is taken out of its sums afterwards, so
    // that logits far from zero lose nothing against (x - base) c
    const float shift = -base * c;
    const float rest = __builtin_fmaf(-base, c, -shift);
    float t0 = 0.0f, t1 = 0.0f, off = rest;
    if (__any(fabsf(base) > 1e30f)) { // base c might overflow (a row masked with the type's lowest value)
#pragma unroll
      for (int i = 0; i < kPacks * kVec; ++i) {
        const float y = (v[i] - base) * c;
        const float e = __builtin_amdgcn_exp2f(y);
        t0 += e;
        if constexpr (kEntropy) t1 = __builtin_fmaf(e, fmaxf(y, -160.0f), t1);
      }
      off = 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < kPacks * kVec; ++i) {
        const float y = __builtin_fmaf(v[i], c, shift);
        const float e = __builtin_amdgcn_exp2f(y); // 0 below 2^-149, NaN for NaN
        t0 += e;
        if constexpr (kEntropy) t1 = __builtin_fmaf(e, fmaxf(y, -160.0f), t1); // 0 * -infinity is no term
      }
    }
    const float d = rebase(r.m, m, c), f = __builtin_amdgcn_exp2f(d), g = __builtin_amdgcn_exp2f(off);
    if constexpr (kEntropy) r.s1 = (r.s1 + r.s0 * d) * f + (t1 + off * t0) * g;
    r.s0 = r.s0 * f + t0 * g;
    r.m = m;
  }

  // lanes, then waves
  {
    const float m = waveMax(r.m);
    const float d = rebase(r.m, m, c), f = __builtin_amdgcn_exp2f(d);
    const float s1 = kEntropy ? waveSum((r.s1 + r.s0 * d) * f) : 0.0f;
    const float s0 = waveSum(r.s0 * f);
    if (threadIdx.x % 64 == 0) waveSums[threadIdx.x / 64] = RowSums{m, s0, s1};
  }

  if constexpr (kTop) {
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
    if (threadIdx.x == 0) listed = found = 0;
    __syncthreads();
    uint64_t bound = waveBound[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) bound = bound > waveBound[w] ? bound : waveBound[w];
    // segments that reach the bound (by their value: the places come next)
    if (laneKey != 0 && laneKey >= bound) {
      const uint32_t least = static_cast<uint32_t>(bound >> 32);
      for (uint32_t tile = 0; tile < tiles; ++tile)
        if (orderOf(segments[tile * kBlock + threadIdx.x]) >= least)
          list[atomicAdd(&listed, 1u)] = static_cast<uint16_t>(tile * kBlock + threadIdx.x);
    }
    __syncthreads(); // the list is whole, and the maxima are not needed any more
    const uint32_t count = listed;
    uint64_t* keys = reinterpret_cast<uint64_t*>(area);
    uint32_t keep = count;
    if (count > a.top) {
      keep = a.top;
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
        // a segment without a valid logit has key 0: distinct below all others is all that rank needs
        const uint64_t key = segmentKey(tile, owner, most);
        keys[e] = key != 0 ? key : e;
      }
      if (threadIdx.x < kMaxTop) best[threadIdx.x] = 0;
      __syncthreads();
      rankKeys(keys, count, a.top, [&](uint32_t rank, uint64_t key, uint32_t e) {
        kept[rank] = list[e];
        best[rank] = key;
      });
      __syncthreads(); // also: the segments' keys are read
      bound = bound > best[a.top - 1] ? bound : best[a.top - 1];
    } else {
      if (threadIdx.x < count) kept[threadIdx.x] = list[threadIdx.x];
      __syncthreads();
    }
    for (uint32_t e = threadIdx.x; e < keep * kPacks; e += kBlock) {
      const uint32_t segment = kept[e / kPacks];
      const uint32_t from = place(segment / kBlock, e % kPacks, segment % kBlock);
      float w[kVec];
      T::unpack(loadPack<T, false>(x, from, end, kNothing), w);
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (from + i < end && w[i] == w[i] && keyOf(w[i], from + i) >= bound)
          keys[atomicAdd(&found, 1u)] = keyOf(w[i], from + i);
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
  if (a.parts == 1) {
    finishRow<T>(a, row, total, best);
  } else {
    const uint64_t slot = uint64_t(blockIdx.x);
    if (threadIdx.x == 0) a.partSums[slot] = total;
    if (kTop && threadIdx.x < a.top) a.partKeys[slot * a.top + threadIdx.x] = best[threadIdx.x];
  }
}

// Joins the parts of a row: one work-group per row, in the order of the parts.
constexpr uint32_t kJoinKeys = 2048;
template <typename T>
__global__ __launch_bounds__(kBlock) void logprobJoinKernel(ForwardArgs a) {
  __shared__ uint64_t keys[kJoinKeys];
  __shared__ uint64_t best[kMaxTop];
  const uint64_t slot = uint64_t(blockIdx.x) * a.parts;
  const float c = a.scale * kLog2e;
  RowSums r = a.partSums[slot];
  for (uint32_t p = 1; p < a.parts; ++p) r = join(r, a.partSums[slot + p], c);
  if (a.top != 0) {
    const uint64_t* from = a.partKeys + slot * a.top;
    const uint32_t all = a.parts * a.top;
    if (threadIdx.x < kMaxTop) best[threadIdx.x] = 0;
    for (uint32_t at = 0; at < all; at += kJoinKeys - kMaxTop) { // and the best so far
      const uint32_t count = all - at < kJoinKeys - kMaxTop ? all - at : kJoinKeys - kMaxTop;
      __syncthreads();
      for (uint32_t e = threadIdx.x; e < count; e += kBlock) keys[e] = from[at + e];
      if (threadIdx.x < a.top) keys[count + threadIdx.x] = best[threadIdx.x];
      __syncthreads();
      if (threadIdx.x < kMaxTop) best[threadIdx.x] = 0;
      __syncthreads();
      // empty places (key 0) are not distinct, but rank below every logit: they emit zeros
      rankKeys(keys, count + a.top, a.top, [&](uint32_t rank, uint64_t key, uint32_t) {
        if (key != 0) best[rank] = key;
      });
    }
    __syncthreads();
  }
  finishRow<T>(a, a.firstRow + blockIdx.x, r, best);
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

constexpr int kGradPacks = 2;
template <typename T, bool kEntropy>
__global__ __launch_bounds__(kBlock) void logprobGradKernel(GradArgs a) {
  constexpr int kVec = T::kVec;
  const uint64_t row = blockIdx.x / a.chunks;
  const uint32_t first = (blockIdx.x % a.chunks) * (kBlock * kGradPacks * kVec);
  const typename T::Stored* x = static_cast<const typename T::Stored*>(a.logits) + row * a.stride;
  typename T::Stored* dx = static_cast<typename T::Stored*>(a.dlogits) + row * a.dlogitsStride;
  Pack in[kGradPacks];
#pragma unroll
  for (int k = 0; k < kGradPacks; ++k)
    in[k] = loadPack<T>(x, first + (k * kBlock + threadIdx.x) * kVec, a.cols, typename T::Stored(0.0f));
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
    const uint32_t at = first + (k * kBlock + threadIdx.x) * kVec;
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

template <typename T> int forward(polar_hip_device* dev, ForwardArgs a, uint64_t rows) {
  const uint32_t tiles = (a.cols + tileCols<T>() - 1) / tileCols<T>();
  // parts: at most kMaxTiles tiles each, and enough of them for four work-groups per CU
  const uint64_t groups = 4ull * dev->info.compute_units;
  const uint64_t wanted = std::max<uint64_t>((tiles + kMaxTiles - 1) / kMaxTiles, groups / std::max<uint64_t>(rows, 1));
  a.tilesPerPart = static_cast<uint32_t>((tiles + std::min<uint64_t>(wanted, tiles) - 1) / std::min<uint64_t>(wanted, tiles));
  a.parts = (tiles + a.tilesPerPart - 1) / a.tilesPerPart;
  const bool entropy = a.entropy != nullptr, top = a.top != 0;
  auto kernel = entropy ? (top ? logprobKernel<T, true, true> : logprobKernel<T, true, false>)
                        : (top ? logprobKernel<T, false, true> : logprobKernel<T, false, false>);
  // rows per launch: block numbers in 31 bits, parts' results in 64 MiB of workspace
  const uint64_t slotBytes = sizeof(RowSums) + uint64_t(a.top) * sizeof(uint64_t);
  uint64_t batch = (1ull << 30) / a.parts;
  if (a.parts > 1) batch = std::min(batch, std::max<uint64_t>(1, (64ull << 20) / (a.parts * slotBytes)));
  std::lock_guard<std::mutex> lock(dev->workspaceMu);
  for (uint64_t r = 0; r < rows; r += batch) {
    const uint64_t n = std::min(batch, rows - r);
    a.firstRow = r;
    if (a.parts > 1) {
      void* area = nullptr;
      const int st = workspaceFor(dev, n * a.parts * slotBytes, &area);
      if (st != POLAR_HIP_OK) return st;
      a.partKeys = static_cast<uint64_t*>(area);
      a.partSums = reinterpret_cast<RowSums*>(a.partKeys + n * a.parts * a.top);
    }
    POLAR_HIP_TRY(launchKernel(dev, kernel, dim3(static_cast<unsigned>(n * a.parts)), dim3(kBlock), a));
    if (a.parts > 1) POLAR_HIP_TRY(launchKernel(dev, logprobJoinKernel<T>, dim3(static_cast<unsigned>(n)), dim3(kBlock), a));
  }
  return POLAR_HIP_OK;
}

template <typename T> int backward(polar_hip_device* dev, GradArgs a) {
  constexpr uint32_t kChunk = kBlock * kGradPacks * T::kVec;
  a.chunks = (a.cols + kChunk - 1) / kChunk;
  auto kernel = a.dentropy != nullptr ? logprobGradKernel<T, true> : logprobGradKernel<T, false>;
  const uint64_t batch = (1ull << 30) / a.chunks, rows = a.rows;
  GradArgs part = a;
  for (uint64_t r = 0; r < rows; r += batch) {
    const uint64_t n = std::min(batch, rows - r);
    POLAR_HIP_TRY(launchKernel(dev, kernel, dim3(static_cast<unsigned>(n * a.chunks)), dim3(kBlock), part));
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
  POLAR_HIP_REQUIRE(scale > 0.0f && std::isfinite(scale), "scale must be positive and finite");
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
  POLAR_HIP_REQUIRE(scale > 0.0f && std::isfinite(scale), "scale must be positive and finite");
  if (rows == 0) return POLAR_HIP_OK;
  POLAR_HIP_REQUIRE(logits && stats && dlogits, "null tensor");
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
