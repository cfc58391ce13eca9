// One AdamW step over a list of tensors, with states in 32 or in 8 bits.
//
//   g = gradScale * grad,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p - lr wd p - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Everything is read once and written once: memory is what bounds it.  100
// million elements in fp32 (28 bytes each) take 456 us, 6.2 TB/s, 90 % of what
// a large copy reaches; 260 million with states in 8 bits, bf16 gradients and
// copies (16 bytes each) 693 us, 6.2 TB/s.  Loads and stores stream past the
// caches (with plain loads or plain stores 510 us).  A launch covers up to
// kTensors tensors, whose table travels in the kernel's arguments: no table in
// device memory to upload and keep, and a model of a few hundred tensors takes
// a few launches.  A work-group takes a chunk of one tensor, a lane four
// consecutive elements of it.
//
// States in 8 bits: 256 consecutive elements of a tensor (one wave's four per
// lane) share a scale, the largest value in the block / 448.  m is held as an
// 8-bit float (sign, four exponent bits, three mantissa bits; 448 is its
// largest), and so is sqrt(v) rather than v: its range of 2^18 spans 2^36 in v.
// Rounding is stochastic: a value between two neighbours goes up with the
// probability of its distance to the lower one.  To nearest, v would stand
// still: a step moves it by (1 - b2) = 0.1 %, far less than half the distance
// of two neighbours (3 to 6 %); stochastically it follows on average.  The 16
// random bits come from a hash of the caller's seed and the element's number.
// The parameter is updated from the unrounded states.
//
// Below the smallest code (4.4e-6 of the block's largest) a root is held as zero
// most of the time, and m, whose random bits are others, now and then as a whole
// code: their quotient was a step of hundreds of lr.  A root that is not zero and
// rounds to zero therefore leaves a trace, code 0x80 (minus zero: it still counts
// as 0 for the next root, so that the average is kept), and the next step divides
// by the smallest code at least: too small a step, as with a larger eps, in place
// of one that is too large (emulated, 1500 steps of elements 10^6 times below the
// largest of their block: root mean square 0.15 lr and at most 1.5 lr, with states
// in 32 bits 0.23 and 1.1, without the trace 8.3 and 399).
#include "typed.h"

#include <algorithm>
#include <cmath>
#include <exception>
#include <utility>
#include <vector>

using namespace polar_hip_detail;

namespace {

// Small work-groups with one group of four elements per lane measured best, as for the
// elementwise kernels: 100 million fp32 elements 457 us, with 256 lanes 500, with two or four
// groups per lane 490
constexpr int kBlock = 128;
constexpr uint32_t kChunk = kBlock * 4;             // elements of a work-group
constexpr uint64_t kScaleBlock = POLAR_HIP_ADAMW_BLOCK; // elements that share a scale
static_assert(kScaleBlock == 64 * 4, "one wave's four elements per lane");
constexpr float kLargest = 448.0f;                  // of the 8-bit floats
constexpr float kTiny = 0x1p-100f;                  // blocks whose scale is not above this are held as zeros

constexpr uint64_t kMostGroups = 1ull << 24; // of a launch, whose lanes are counted in 32 bits
constexpr int kTensors = 46;
struct Entry {
  void *param, *grad, *m, *v;
  float *master, *mScale, *vScale;
  uint64_t count, random;
  float decay; // lr * weight decay
};
struct Table {
  Entry e[kTensors];
  uint32_t firstGroup[kTensors]; // of each tensor; the largest number behind the last one
  float gradScale, beta1, rest1, beta2, rest2, stepSize, byCorrection, eps;
  uint32_t seed;
};
static_assert(sizeof(Table) <= 4000, "kernel arguments");

template <int kBytes> struct Words;
template <> struct Words<16> { typedef uint32_t At __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Words<8> { typedef uint32_t At __attribute__((ext_vector_type(2), aligned(2))); };

// four consecutive elements, the first `n` of them real (0 .. 4)
template <typename T>
__device__ __forceinline__ void load4(const typename T::Stored* at, int n, float* out) {
  using S = typename T::Stored;
  S v[4];
  if (n == 4) {
    const auto w = __builtin_nontemporal_load(reinterpret_cast<const typename Words<4 * sizeof(S)>::At*>(at));
    __builtin_memcpy(v, &w, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? at[i] : S(0.0f);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = T::widen(v[i]);
}
template <typename T>
__device__ __forceinline__ void store4(typename T::Stored* at, int n, const float* x) {
  using S = typename T::Stored;
  S v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = T::narrow(x[i]);
  if (n == 4) {
    using At = typename Words<4 * sizeof(S)>::At;
    At w;
    __builtin_memcpy(&w, v, sizeof(v));
    __builtin_nontemporal_store(w, reinterpret_cast<At*>(at));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) at[i] = v[i];
  }
}

typedef uint32_t WordAt1 __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t loadCodes(const uint8_t* at, int n) {
  if (n == 4) return __builtin_nontemporal_load(reinterpret_cast<const WordAt1*>(at));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= i < n ? uint32_t(at[i]) << (8 * i) : 0u;
  return w;
}
__device__ __forceinline__ void storeCodes(uint8_t* at, int n, uint32_t w) {
  if (n == 4) {
    __builtin_nontemporal_store(w, reinterpret_cast<WordAt1*>(at));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) at[i] = static_cast<uint8_t>(w >> (8 * i));
  }
}
__device__ __forceinline__ void widenCodes(uint32_t w, float* out) {
  const Float2 low = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), high = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  out[0] = low.x, out[1] = low.y, out[2] = high.x, out[3] = high.y;
}
// A value of at most 448 (and a rounding error) in size as an 8-bit float, up where 16
// random bits exceed what is cut off: among the normal ones by adding them below the
// mantissa's last kept bit (the carry may reach the exponent, which is the next float),
// below 2^-6 in steps of 2^-9
__device__ __forceinline__ uint32_t narrowCode(float t, uint32_t random) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, t);
  const float size = fabsf(t);
  const uint32_t normal = (((bits & 0x7fffffffu) + (random << 4)) >> 20) - (120u << 3);
  const uint32_t small = static_cast<uint32_t>(size * 512.0f + static_cast<float>(random) * (1.0f / 65536.0f));
  const uint32_t code = size >= 0x1p-6f ? (normal < 0x7eu ? normal : 0x7eu) : small;
  return code | ((bits >> 24) & 0x80u);
}
constexpr uint32_t kNotANumber = 0x7f; // as an 8-bit float
constexpr uint32_t kTrace = 0x80;      // of a root that is less than the smallest code, but not zero
constexpr float kSmallest = 0x1p-9f;   // code
constexpr uint32_t kInfinity = 0x7f800000u;

// Largest of the wave's sizes, given as the bits of fp32 numbers that are not negative:
// in their order, NaN above infinity
__device__ __forceinline__ uint32_t waveLargest(uint32_t v) {
  auto step = [](uint32_t x, auto move) { return max(x, static_cast<uint32_t>(move(static_cast<int>(x)))); };
  v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(x, x, 0xb1, 0xf, 0xf, false); });
  v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(x, x, 0x4e, 0xf, 0xf, false); });
  v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(x, x, 0x141, 0xf, 0xf, false); });
  v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(x, x, 0x140, 0xf, 0xf, false); });
  v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(x, x, 0x142, 0xa, 0xf, false); });
  v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(x, x, 0x143, 0xc, 0xf, false); });
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

// 32 random bits of an element.  Its number and the seed become one word (the number's
// lower half times 2^32 over the golden ratio, rounded to a prime; the upper half times
// the fraction of the root of two in 32 bits), which goes through a published mix: the
// shifts and the two constants are those of MurmurHash3's 32-bit finaliser (Austin
// Appleby, public domain).
__device__ __forceinline__ uint32_t randomBits(uint32_t seed, uint64_t element) {
  uint32_t h = static_cast<uint32_t>(element) * 0x9e3779b1u + static_cast<uint32_t>(element >> 32) * 0x6a09e667u + seed;
  h = (h ^ (h >> 16)) * 0x85ebca6bu;
  h = (h ^ (h >> 13)) * 0xc2b2ae35u;
  return h ^ (h >> 16);
}

// The square root, rounded to nearest: the hardware's is good to a unit in the last
// place, and Tuckerman's test (published with IBM's elementary functions for the
// System/370, 1986) says which of it and its two neighbours it is: the sign of what
// neighbour * r leaves of v, by a fused multiply-add.  The compiler refines sqrtf by the
// same test, with a scaling of small arguments that is left out here: exact where that
// rest is a normal number (v from 2^-96 on), else as the hardware has it; 0, infinity and
// NaN stay what they are.
__device__ __forceinline__ float rootOf(float v) {
  const float r = __builtin_amdgcn_sqrtf(v);
  const float below = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, r) - 1u);
  const float above = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, r) + 1u);
  float root = __builtin_fmaf(-below, r, v) <= 0.0f ? below : r;
  return __builtin_fmaf(-above, r, v) > 0.0f ? above : root;
}

// Four consecutive elements of a tensor in a lane, `n` of them (0 .. 4) real.  P: the
// parameter's type; one of 16 bits is a copy of the fp32 master.  G: the gradient's.
template <typename P, typename G, bool kSmall> struct Four {
  float p[4], g[4], m[4], v[4], r[4];
  uint32_t traces; // of the roots, at their codes' places
  float leastRoot; // what such a root is at most

  __device__ __forceinline__ void load(const Entry& e, const float* master, uint64_t at, int n) {
    load4<TypeF32>(master + at, n, p);
    load4<G>(static_cast<const typename G::Stored*>(e.grad) + at, n, g);
    if constexpr (kSmall) {
      const uint64_t block = at / kScaleBlock;
      const float ms = e.mScale[block], vs = e.vScale[block];
      widenCodes(loadCodes(static_cast<const uint8_t*>(e.m) + at, n), m);
      const uint32_t roots = loadCodes(static_cast<const uint8_t*>(e.v) + at, n);
      widenCodes(roots, r);
      traces = roots & (kTrace * 0x01010101u);
      leastRoot = kSmallest * vs;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] *= ms;
        r[i] *= vs;
        v[i] = r[i] * r[i];
      }
    } else {
      load4<TypeF32>(static_cast<const float*>(e.m) + at, n, m);
      load4<TypeF32>(static_cast<const float*>(e.v) + at, n, v);
    }
  }

  __device__ __forceinline__ void step(const Table& t, float decay) {
    auto states = [&](int i) {
      g[i] *= t.gradScale;
      m[i] = m[i] * t.beta1 + g[i] * t.rest1;
      v[i] = v[i] * t.beta2 + (g[i] * g[i]) * t.rest2;
    };
    if constexpr (kSmall) {
      float divisor[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        states(i);
        divisor[i] = r[i] = rootOf(v[i]);
      }
      if (traces != 0) { // rare
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (traces & (kTrace << (8 * i))) divisor[i] = r[i] < leastRoot ? leastRoot : r[i];
      }
      // The quotient only moves the parameter, by a thousandth or so of its size: the hardware's
      // reciprocal, good to a unit in the last place, is nothing against the three bits that the
      // states have.  (The divisor is 0, or far above the subnormal numbers: a root's smallest
      // value is 3.7e-23.)  With the exact division and sqrtf their 20 instructions more per
      // element would set the time: 788 us for 260 million elements.
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[i] = (p[i] - p[i] * decay) - m[i] * t.stepSize * __builtin_amdgcn_rcpf(divisor[i] * t.byCorrection + t.eps);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        states(i);
        p[i] = (p[i] - p[i] * decay) - m[i] * t.stepSize / (sqrtf(v[i]) * t.byCorrection + t.eps);
      }
    }
  }

  __device__ __forceinline__ void store(const Table& t, const Entry& e, float* master, uint64_t at, int n) {
    store4<TypeF32>(master + at, n, p);
    if constexpr (sizeof(typename P::Stored) == 2) store4<P>(static_cast<typename P::Stored*>(e.param) + at, n, p);
    if constexpr (kSmall) {
      // elements behind the end are zeros: loads give them as such, and they stay
      uint32_t largestM = 0, largestR = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        largestM = max(largestM, __builtin_bit_cast(uint32_t, fabsf(m[i])));
        largestR = max(largestR, __builtin_bit_cast(uint32_t, fabsf(r[i])));
      }
      largestM = waveLargest(largestM), largestR = waveLargest(largestR);
      const bool odd = largestM >= kInfinity || largestR >= kInfinity; // rare, and the whole wave's
      if (odd) {
        // an element that is not finite is held as NaN and has no say in its block's scale
        largestM = largestR = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t bitsM = __builtin_bit_cast(uint32_t, fabsf(m[i])), bitsR = __builtin_bit_cast(uint32_t, fabsf(r[i]));
          largestM = max(largestM, bitsM < kInfinity ? bitsM : 0u);
          largestR = max(largestR, bitsR < kInfinity ? bitsR : 0u);
        }
        largestM = waveLargest(largestM), largestR = waveLargest(largestR);
      }
      const float ms = __builtin_bit_cast(float, largestM) * (1.0f / kLargest);
      const float vs = __builtin_bit_cast(float, largestR) * (1.0f / kLargest);
      const float byM = ms > kTiny ? 1.0f / ms : 0.0f, byV = vs > kTiny ? 1.0f / vs : 0.0f;
      uint32_t codeM = 0, codeV = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t random = randomBits(t.seed, e.random + at + i);
        codeM |= narrowCode(m[i] * byM, random & 0xffffu) << (8 * i);
        codeV |= narrowCode(r[i] * byV, random >> 16) << (8 * i);
      }
      if (odd) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!(fabsf(m[i]) < __builtin_inff())) codeM = (codeM & ~(0xffu << (8 * i))) | kNotANumber << (8 * i);
          if (!(fabsf(r[i]) < __builtin_inff())) codeV = (codeV & ~(0xffu << (8 * i))) | kNotANumber << (8 * i);
        }
      }
      // codes are below 0x80, so that the sum's upper bit in each byte says whether its code is not 0
      const uint32_t zeros = ~(codeV + 0x7f7f7f7fu) & 0x80808080u;
      if (zeros != 0) { // rare, but for elements that never had a gradient
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r[i] > 0.0f || m[i] != 0.0f) codeV |= zeros & (kTrace << (8 * i));
      }
      storeCodes(static_cast<uint8_t*>(e.m) + at, n, codeM);
      storeCodes(static_cast<uint8_t*>(e.v) + at, n, codeV);
      if (threadIdx.x % 64 == 0) {
        e.mScale[at / kScaleBlock] = ms;
        e.vScale[at / kScaleBlock] = vs;
      }
    } else {
      store4<TypeF32>(static_cast<float*>(e.m) + at, n, m);
      store4<TypeF32>(static_cast<float*>(e.v) + at, n, v);
    }
  }
};

template <typename P, typename G, bool kSmall>
__global__ __launch_bounds__(kBlock) void adamwKernel(Table table) {
  constexpr bool kCopy = sizeof(typename P::Stored) == 2;
  // all the first groups sit side by side in scalar registers: no search through memory
  int which = 0;
#pragma unroll
  for (int i = 1; i < kTensors; ++i) which = blockIdx.x >= table.firstGroup[i] ? i : which;
  which = __builtin_amdgcn_readfirstlane(which);
  const uint32_t first = table.firstGroup[which];
  const Entry e = table.e[which];
  const uint64_t at = uint64_t(blockIdx.x - first) * kChunk + threadIdx.x * 4;
  float* master = kCopy ? e.master : static_cast<float*>(e.param);
  Four<P, G, kSmall> f;
  if (at - threadIdx.x * 4 + kChunk <= e.count) { // a whole chunk: no element is checked
    f.load(e, master, at, 4);
    f.step(table, e.decay);
    f.store(table, e, master, at, 4);
  } else if (at - threadIdx.x % 64 * 4 < e.count) { // not a wave that lies behind the tensor's end as a whole
    const int n = at >= e.count ? 0 : e.count - at < 4 ? static_cast<int>(e.count - at) : 4;
    f.load(e, master, at, n);
    f.step(table, e.decay);
    f.store(table, e, master, at, n);
  }
}

using Kernel = void (*)(Table);
template <typename P, typename G> Kernel pick(bool small) {
  return small ? adamwKernel<P, G, true> : adamwKernel<P, G, false>;
}
template <typename P> Kernel pick(int gradType, bool small) {
  return gradType == POLAR_HIP_F32 ? pick<P, TypeF32>(small)
         : gradType == POLAR_HIP_F16 ? pick<P, TypeF16>(small)
                                     : pick<P, TypeBF16>(small);
}

// What is written must not overlap: a parameter or a state that is listed twice (weights that two
// layers share) would be updated by two work-groups at once.  Most lists go up in memory field by
// field, which one pass shows; else the buffers are sorted.
bool writtenTwice(const polar_hip_adamw_config& config, const polar_hip_adamw_tensor* tensors, uint64_t count) {
  using Span = std::pair<uintptr_t, uintptr_t>;
  const bool small = config.state_bits == 8, copy = config.param_type != POLAR_HIP_F32;
  const uint64_t state = small ? 1 : 4, parameter = sizeOf(config.param_type);
  auto span = [](const void* at, uint64_t bytes) {
    return Span{reinterpret_cast<uintptr_t>(at), reinterpret_cast<uintptr_t>(at) + bytes};
  };
  constexpr int kFields = 6;
  auto buffers = [&](const polar_hip_adamw_tensor& t, Span* out) {
    int n = 0;
    out[n++] = span(t.param, t.count * parameter);
    out[n++] = span(t.m, t.count * state);
    out[n++] = span(t.v, t.count * state);
    if (copy) out[n++] = span(t.master, t.count * 4);
    if (small) {
      const uint64_t blocks = (t.count + kScaleBlock - 1) / kScaleBlock;
      out[n++] = span(t.m_scale, blocks * 4);
      out[n++] = span(t.v_scale, blocks * 4);
    }
    return n;
  };
  auto overlap = [](Span* first, Span* last) {
    std::sort(first, last);
    for (Span* s = first; s + 1 < last; ++s)
      if (s[0].second > s[1].first) return true;
    return false;
  };
  Span area[kFields], mine[kFields]; // of each field
  bool ascending = true;
  int fields = 0;
  for (uint64_t i = 0; i < count && ascending; ++i) {
    if (tensors[i].count == 0) continue;
    const bool first = fields == 0;
    fields = buffers(tensors[i], mine);
    for (int f = 0; f < fields; ++f) {
      if (first) area[f] = mine[f];
      ascending = ascending && (first || mine[f].first >= area[f].second);
      area[f].second = mine[f].second;
    }
  }
  if (ascending && !overlap(area, area + fields)) return false;
  std::vector<Span> all;
  all.reserve(count * kFields);
  for (uint64_t i = 0; i < count; ++i) {
    if (tensors[i].count == 0) continue;
    const int n = buffers(tensors[i], mine);
    all.insert(all.end(), mine, mine + n);
  }
  return overlap(all.data(), all.data() + all.size());
}

} // namespace

extern "C" {

int polar_hip_fadamw(polar_hip_device* dev, const polar_hip_adamw_config* config, const polar_hip_adamw_tensor* tensors,
                     uint64_t count) {
  POLAR_HIP_REQUIRE(dev != nullptr && config != nullptr, "null argument");
  POLAR_HIP_REQUIRE(count == 0 || tensors != nullptr, "null list of tensors");
  POLAR_HIP_REQUIRE(knownType(config->param_type) && knownType(config->grad_type), "unknown element type");
  POLAR_HIP_REQUIRE(config->state_bits == 32 || config->state_bits == 8, "states are held in 32 or 8 bits");
  POLAR_HIP_REQUIRE(config->step >= 1, "steps are counted from 1");
  POLAR_HIP_REQUIRE(config->beta1 >= 0 && config->beta1 < 1 && config->beta2 >= 0 && config->beta2 < 1,
                    "beta1 and beta2 lie in [0, 1)");
  POLAR_HIP_REQUIRE(std::isfinite(config->lr) && config->eps >= 0 && std::isfinite(config->eps) &&
                        std::isfinite(config->grad_scale),
                    "lr, eps and grad_scale must be finite, eps not negative");
  const bool small = config->state_bits == 8, copy = config->param_type != POLAR_HIP_F32;
  // the kernel has them in fp32; an eps that is lost there, or (8-bit states) that the hardware's
  // reciprocal takes for 0, would make 0 / 0 of elements that never had a gradient
  const double stepSize = config->lr / (1.0 - std::pow(config->beta1, static_cast<double>(config->step)));
  auto held = [](double x) { return std::isfinite(static_cast<float>(x)); };
  POLAR_HIP_REQUIRE(held(stepSize) && held(config->grad_scale) && held(config->eps) &&
                        (config->eps == 0 || config->eps >= (small ? 0x1p-126 : 0x1p-149)),
                    "lr, grad_scale or eps is out of fp32's range");
  // everything is checked before the first tensor is touched
  for (uint64_t i = 0; i < count; ++i) {
    const polar_hip_adamw_tensor& t = tensors[i];
    POLAR_HIP_REQUIRE(held(config->lr * t.weight_decay), "lr times a tensor's weight decay is out of fp32's range");
    if (t.count == 0) continue;
    POLAR_HIP_REQUIRE(t.count <= kChunk * kMostGroups, "a tensor is too large");
    POLAR_HIP_REQUIRE(t.param && t.grad && t.m && t.v, "a tensor's pointer is null");
    POLAR_HIP_REQUIRE(!copy || t.master, "16-bit parameters need an fp32 master");
    POLAR_HIP_REQUIRE(!small || (t.m_scale && t.v_scale), "8-bit states need scales");
    POLAR_HIP_REQUIRE(alignedTo(t.param, sizeOf(config->param_type)) && alignedTo(t.grad, sizeOf(config->grad_type)) &&
                          (!copy || alignedTo(t.master, 4)) && (small || (alignedTo(t.m, 4) && alignedTo(t.v, 4))) &&
                          (!small || (alignedTo(t.m_scale, 4) && alignedTo(t.v_scale, 4))),
                      "misaligned pointer");
  }
  try {
    POLAR_HIP_REQUIRE(!writtenTwice(*config, tensors, count), "two of the buffers that are written overlap");
  } catch (const std::exception&) {
    return fail(POLAR_HIP_ERR_OOM, "polar_hip_fadamw: no host memory to check %llu tensors",
                static_cast<unsigned long long>(count));
  }
  POLAR_HIP_TRY(hipSetDevice(dev->ordinal));
  Table table{};
  const double correction2 = 1.0 - std::pow(config->beta2, static_cast<double>(config->step));
  table.gradScale = static_cast<float>(config->grad_scale);
  table.beta1 = static_cast<float>(config->beta1);
  table.rest1 = static_cast<float>(1.0 - config->beta1);
  table.beta2 = static_cast<float>(config->beta2);
  table.rest2 = static_cast<float>(1.0 - config->beta2);
  table.stepSize = static_cast<float>(stepSize);
  table.byCorrection = static_cast<float>(1.0 / std::sqrt(correction2));
  table.eps = static_cast<float>(config->eps);
  table.seed = config->seed;
  const Kernel kernel = config->param_type == POLAR_HIP_F32   ? pick<TypeF32>(config->grad_type, small)
                        : config->param_type == POLAR_HIP_F16 ? pick<TypeF16>(config->grad_type, small)
                                                              : pick<TypeBF16>(config->grad_type, small);
  uint64_t groups = 0;
  int listed = 0;
  auto flush = [&]() -> int {
    if (listed == 0) return POLAR_HIP_OK;
    for (; listed < kTensors; ++listed) table.firstGroup[listed] = 0xffffffffu;
    POLAR_HIP_TRY(launchKernel(dev, kernel, dim3(static_cast<unsigned>(groups)), dim3(kBlock), table));
    listed = 0;
    groups = 0;
    return POLAR_HIP_OK;
  };
  for (uint64_t i = 0; i < count; ++i) {
    const polar_hip_adamw_tensor& t = tensors[i];
    if (t.count == 0) continue;
    const uint64_t mine = (t.count + kChunk - 1) / kChunk;
    if (listed == kTensors || groups + mine > kMostGroups) {
      const int st = flush();
      if (st != POLAR_HIP_OK) return st;
    }
    table.firstGroup[listed] = static_cast<uint32_t>(groups);
    table.e[listed++] = Entry{t.param, const_cast<void*>(t.grad), t.m, t.v, t.master, t.m_scale, t.v_scale, t.count,
                              t.first, static_cast<float>(config->lr * t.weight_decay)};
    groups += mine;
  }
  return flush();
}

} // extern "C"
