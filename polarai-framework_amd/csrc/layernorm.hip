// Layer normalisation of the rows of a matrix, and its gradient.
//
//   y = (x - mean) rstd w + b,   mean = sum(x) / C,   rstd = 1 / sqrt(sum((x - mean)^2) / C + eps)
//   with g = dy w and h = (x - mean) rstd:
//   dx = rstd (g - mean(g) - h mean(g h)),   dw = sum over rows of dy h,   db = sum over rows of dy
//
// A row is held in the registers of 1 to 16 waves (kWaves x 64 lanes x kPacks
// 16-byte packs), so x and dy are read once from memory although the
// statistics need two passes over them: the variance is the sum of squared
// distances from the mean already known, never E[x^2] - mean^2, which loses
// all its digits for rows far from zero.  A team of waves walks over rows
// team, team + teams, ...: weight and bias stay in its registers, the next
// kAhead rows are loaded while the present one is reduced, and in the backward
// pass the columns' sums for dw and db stay in registers until the team's last
// row; a second kernel adds the teams' sums in a fixed order (no atomics: the
// same bits on every run).  Rows that no team's registers hold go through
// memory (cache) once per pass.
//
// Memory bounds it.  16384 x 8192 bf16 takes 89 us (6.0 TB/s; a copy of the
// same bytes 81 us) and 94 to 130 us with more, shorter-lived teams, which load
// weight and bias more often than they gain; without the barriers of the
// reductions it would take as long.  Its gradient, 16384 x 4096, takes 76 us:
// 71 for 403 MB and 5 for the teams' sums, which is why there are few teams
// with many rows in flight (512 teams with one row ahead: 82 us).
#include "typed.h"

#include <algorithm>
#include <cmath>

using namespace polar_hip_detail;

namespace {

constexpr int kTeamBlock = 256; // lanes of a work-group whose teams are one to four waves

// Sums over the team's lanes.  `lds` holds kTeams x kWaves values for each of
// two rounds: a round's values are not overwritten before every wave has read
// them, because the round after next begins behind another barrier.
template <int kWaves>
__device__ __forceinline__ float teamSum(float v, float* lds, int team, int wave) {
  v = waveSum(v);
  if constexpr (kWaves == 1) return v;
  if (threadIdx.x % 64 == 0) lds[team * kWaves + wave] = v;
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += lds[team * kWaves + w];
  return total;
}
template <int kWaves>
__device__ __forceinline__ Float2 teamSum2(Float2 v, Float2* lds, int team, int wave) {
  v.x = waveSum(v.x);
  v.y = waveSum(v.y);
  if constexpr (kWaves == 1) return v;
  if (threadIdx.x % 64 == 0) lds[team * kWaves + wave] = v;
  __syncthreads();
  Float2 total{0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    total.x += lds[team * kWaves + w].x;
    total.y += lds[team * kWaves + w].y;
  }
  return total;
}

template <typename T, int kPacks>
__device__ __forceinline__ void loadRow(const typename T::Stored* row, uint32_t lane, uint32_t lanes, uint64_t cols, Pack* out) {
#pragma unroll
  for (int k = 0; k < kPacks; ++k)
    out[k] = loadPack<T>(row, (uint64_t(k) * lanes + lane) * T::kVec, cols, typename T::Stored(0.0f));
}

template <typename T, typename P, int kWaves, int kPacks, int kAhead>
__global__ __launch_bounds__(kWaves * 64 < kTeamBlock ? kTeamBlock : kWaves * 64) void layerNormKernel(
    const typename T::Stored* x, uint64_t xStride, const typename P::Stored* weight, const typename P::Stored* bias,
    float eps, typename T::Stored* y, uint64_t yStride, float* means, float* rstds, uint64_t rows, uint32_t cols) {
  constexpr int kBlock = kWaves * 64 < kTeamBlock ? kTeamBlock : kWaves * 64;
  constexpr int kTeams = kBlock / (kWaves * 64);
  constexpr int kLanes = kWaves * 64;
  __shared__ float lds[2][kTeams * kWaves];
  const int team = threadIdx.x / kLanes, wave = threadIdx.x / 64 % kWaves;
  const uint32_t lane = threadIdx.x % kLanes;
  const uint64_t step = uint64_t(gridDim.x) * kTeams;
  const float count = static_cast<float>(cols);

  float w[kPacks][T::kVec], b[kPacks][T::kVec];
  uint64_t row = uint64_t(blockIdx.x) * kTeams + team;
  Pack next[kAhead][kPacks]; // the rows that come next, the first one for the round that is due
#pragma unroll
  for (int n = 0; n < kAhead; ++n)
    if (row + n * step < rows) loadRow<T, kPacks>(x + (row + n * step) * xStride, lane, kLanes, cols, next[n]);
#pragma unroll
  for (int k = 0; k < kPacks; ++k) {
    const uint64_t c = (uint64_t(k) * kLanes + lane) * T::kVec;
    loadParams<P, T::kVec>(weight, c, cols, 1.0f, w[k]);
    loadParams<P, T::kVec>(bias, c, cols, 0.0f, b[k]);
  }
  // every team of a work-group makes the same number of rounds (their barriers
  // are the work-group's); a team whose row is behind the last one only keeps step
  for (uint64_t first = uint64_t(blockIdx.x) * kTeams; first < rows;) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n, first += step, row += step) {
      if (n > 0 && first >= rows) break;
      const bool here = row < rows;
      float v[kPacks][T::kVec];
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < kPacks; ++k) {
        T::unpack(next[n][k], v[k]);
#pragma unroll
        for (int i = 0; i < T::kVec; ++i) sum += v[k][i]; // elements behind the row's end are zero
      }
      if (row + kAhead * step < rows) loadRow<T, kPacks>(x + (row + kAhead * step) * xStride, lane, kLanes, cols, next[n]);
      const float mean = teamSum<kWaves>(here ? sum : 0.0f, lds[0], team, wave) / count;
      float squares = 0.0f;
#pragma unroll
      for (int k = 0; k < kPacks; ++k) {
        const uint32_t c = (k * kLanes + lane) * T::kVec;
#pragma unroll
        for (int i = 0; i < T::kVec; ++i) {
          v[k][i] = c + i < cols ? v[k][i] - mean : 0.0f;
          squares += v[k][i] * v[k][i];
        }
      }
      const float rstd = 1.0f / sqrtf(teamSum<kWaves>(squares, lds[1], team, wave) / count + eps);
      if (here) {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
          const uint64_t c = (uint64_t(k) * kLanes + lane) * T::kVec;
          float out[T::kVec];
#pragma unroll
          for (int i = 0; i < T::kVec; ++i) out[i] = v[k][i] * rstd * w[k][i] + b[k][i];
          storePack<T>(y + row * yStride, c, cols, out);
        }
        if (lane == 0) {
          if (means != nullptr) means[row] = mean;
          if (rstds != nullptr) rstds[row] = rstd;
        }
      }
    }
  }
}

// Rows longer than a team's registers: one work-group per row, three passes over it.
constexpr int kLongBlock = 1024;
template <typename T, typename F>
__device__ __forceinline__ void alongRow(const typename T::Stored* row, uint64_t cols, F each) {
  for (uint64_t c = uint64_t(threadIdx.x) * T::kVec; c < cols; c += uint64_t(kLongBlock) * T::kVec) {
    float v[T::kVec];
    T::unpack(loadPack<T, false>(row, c, cols, typename T::Stored(0.0f)), v);
    each(c, v);
  }
}
template <typename T>
__device__ __forceinline__ void longStats(const typename T::Stored* row, uint64_t cols, float eps, float (*lds)[16],
                                          float* mean, float* rstd) {
  float sum = 0.0f, squares = 0.0f;
  alongRow<T>(row, cols, [&](uint64_t, const float* v) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < T::kVec; ++i) s += v[i];
    sum += s;
  });
  const float count = static_cast<float>(cols);
  *mean = teamSum<16>(sum, lds[0], 0, threadIdx.x / 64) / count;
  alongRow<T>(row, cols, [&](uint64_t c, const float* v) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < T::kVec; ++i) {
      const float d = c + i < cols ? v[i] - *mean : 0.0f;
      s += d * d;
    }
    squares += s;
  });
  *rstd = 1.0f / sqrtf(teamSum<16>(squares, lds[1], 0, threadIdx.x / 64) / count + eps);
}

template <typename T, typename P>
__global__ __launch_bounds__(kLongBlock) void layerNormLongKernel(
    const typename T::Stored* x, uint64_t xStride, const typename P::Stored* weight, const typename P::Stored* bias,
    float eps, typename T::Stored* y, uint64_t yStride, float* means, float* rstds, uint64_t rows, uint64_t cols) {
  __shared__ float lds[2][16];
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    float mean, rstd;
    longStats<T>(x + row * xStride, cols, eps, lds, &mean, &rstd);
    alongRow<T>(x + row * xStride, cols, [&](uint64_t c, const float* v) {
      float w[T::kVec], b[T::kVec], out[T::kVec];
      loadParams<P, T::kVec>(weight, c, cols, 1.0f, w);
      loadParams<P, T::kVec>(bias, c, cols, 0.0f, b);
#pragma unroll
      for (int i = 0; i < T::kVec; ++i) out[i] = (v[i] - mean) * rstd * w[i] + b[i];
      storePack<T>(y + row * yStride, c, cols, out);
    });
    if (threadIdx.x == 0) {
      if (means != nullptr) means[row] = mean;
      if (rstds != nullptr) rstds[row] = rstd;
    }
  }
}

// ---- gradient --------------------------------------------------------------------

// A lane's sums for dw and db of its columns, kept over its team's rows: in registers, or,
// for teams of sixteen waves, whose lanes have 128 registers, in LDS (a place of its own for
// each lane and column, the lanes side by side).
constexpr int kMostRegisterWaves = 8;
template <int kWaves, int kPacks, int kVec> struct ColumnSums {
  static constexpr bool kInLds = kWaves > kMostRegisterWaves;
  static constexpr int kLanes = kWaves * 64;
  static constexpr uint32_t kLdsBytes = kInLds ? kLanes * kPacks * kVec * sizeof(Float2) : 0;
  Float2 held[kInLds ? 1 : kPacks * kVec];
  Float2* lds; // the lane's first place

  __device__ __forceinline__ void clear(Float2* area) {
    lds = area + threadIdx.x;
#pragma unroll
    for (int i = 0; i < kPacks * kVec; ++i) at(i) = Float2{0.0f, 0.0f};
  }
  __device__ __forceinline__ Float2& at(int i) {
    if constexpr (kInLds)
      return lds[i * kLanes];
    else
      return held[i];
  }
};

// sums: [2][teams of the whole grid][cols] fp32, dw's before db's; null if neither is wanted
template <typename T, typename P, int kWaves, int kPacks, int kAhead, bool kStats>
__global__ __launch_bounds__(kWaves * 64 < kTeamBlock ? kTeamBlock : kWaves * 64) void layerNormGradKernel(
    const typename T::Stored* dy, uint64_t dyStride, const typename T::Stored* x, uint64_t xStride,
    const typename P::Stored* weight, const float* means, const float* rstds, float eps, typename T::Stored* dx,
    uint64_t dxStride, float* sums, uint64_t rows, uint32_t cols) {
  constexpr int kBlock = kWaves * 64 < kTeamBlock ? kTeamBlock : kWaves * 64;
  constexpr int kTeams = kBlock / (kWaves * 64);
  constexpr int kLanes = kWaves * 64;
  __shared__ float lds[2][kTeams * kWaves];
  __shared__ Float2 lds2[2][kTeams * kWaves];
  const int team = threadIdx.x / kLanes, wave = threadIdx.x / 64 % kWaves;
  const uint32_t lane = threadIdx.x % kLanes;
  const uint64_t step = uint64_t(gridDim.x) * kTeams;
  const float count = static_cast<float>(cols);

  extern __shared__ Float2 columnArea[];
  float w[kPacks][T::kVec];
  ColumnSums<kWaves, kPacks, T::kVec> column;
  column.clear(columnArea);
  uint64_t row = uint64_t(blockIdx.x) * kTeams + team;
  Pack nextX[kAhead][kPacks], nextDy[kAhead][kPacks];
  float nextMean[kAhead], nextRstd[kAhead];
  auto load = [&](int n, uint64_t r) {
    loadRow<T, kPacks>(x + r * xStride, lane, kLanes, cols, nextX[n]);
    loadRow<T, kPacks>(dy + r * dyStride, lane, kLanes, cols, nextDy[n]);
    if constexpr (!kStats) nextMean[n] = means[r], nextRstd[n] = rstds[r];
  };
#pragma unroll
  for (int n = 0; n < kAhead; ++n) {
#pragma unroll
    for (int k = 0; k < kPacks; ++k) nextX[n][k] = nextDy[n][k] = Pack{0, 0, 0, 0};
    nextMean[n] = nextRstd[n] = 0.0f;
    if (row + n * step < rows) load(n, row + n * step);
  }
#pragma unroll
  for (int k = 0; k < kPacks; ++k)
    loadParams<P, T::kVec>(weight, (uint64_t(k) * kLanes + lane) * T::kVec, cols, 1.0f, w[k]);
  int round = 0;
  for (uint64_t first = uint64_t(blockIdx.x) * kTeams; first < rows;) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n, first += step, row += step, round ^= 1) {
      if (n > 0 && first >= rows) break;
      const bool here = row < rows;
      float h[kPacks][T::kVec], g[kPacks][T::kVec];
      float mean = nextMean[n], rstd = nextRstd[n];
#pragma unroll
      for (int k = 0; k < kPacks; ++k) {
        T::unpack(nextX[n][k], h[k]);
        T::unpack(nextDy[n][k], g[k]);
      }
      if (row + kAhead * step < rows) load(n, row + kAhead * step);
      if constexpr (kStats) {
        float sum = 0.0f, squares = 0.0f;
#pragma unroll
        for (int k = 0; k < kPacks; ++k)
#pragma unroll
          for (int i = 0; i < T::kVec; ++i) sum += h[k][i];
        mean = teamSum<kWaves>(sum, lds[0], team, wave) / count;
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
          const uint32_t c = (k * kLanes + lane) * T::kVec;
#pragma unroll
          for (int i = 0; i < T::kVec; ++i) {
            h[k][i] = c + i < cols ? h[k][i] - mean : 0.0f;
            squares += h[k][i] * h[k][i];
          }
        }
        rstd = 1.0f / sqrtf(teamSum<kWaves>(squares, lds[1], team, wave) / count + eps);
      } else if (!(fabsf(mean * rstd) < __builtin_inff())) {
        // Behind the row's end dy is zero, so that whatever finite h is there counts for nothing; where
        // -mean * rstd is not finite (a constant row far from zero), h is made zero there.  Asked once per
        // row: a choice for every element takes 1.3 us of 76 (16384 x 4096).
#pragma unroll
        for (int k = 0; k < kPacks; ++k)
#pragma unroll
          for (int i = 0; i < T::kVec; ++i)
            if ((k * kLanes + lane) * T::kVec + i >= cols) h[k][i] = mean;
      }
      Float2 s{0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < kPacks; ++k)
#pragma unroll
        for (int i = 0; i < T::kVec; ++i) {
          h[k][i] = (kStats ? h[k][i] : h[k][i] - mean) * rstd; // with statistics of its own it is centred already
          if (here) {
            Float2& sum = column.at(k * T::kVec + i);
            sum.x += g[k][i] * h[k][i];
            sum.y += g[k][i];
          }
          g[k][i] *= w[k][i];
          s.x += g[k][i];
          s.y += g[k][i] * h[k][i];
        }
      s = teamSum2<kWaves>(s, lds2[round], team, wave);
      const float alongOnes = s.x / count, alongH = s.y / count;
      if (here && dx != nullptr) {
#pragma unroll
        for (int k = 0; k < kPacks; ++k) {
          float out[T::kVec];
#pragma unroll
          for (int i = 0; i < T::kVec; ++i) out[i] = rstd * (g[k][i] - alongOnes - h[k][i] * alongH);
          storePack<T>(dx + row * dxStride, (uint64_t(k) * kLanes + lane) * T::kVec, cols, out);
        }
      }
    }
  }
  if (sums != nullptr) {
    const uint64_t teams = step, mine = uint64_t(blockIdx.x) * kTeams + team;
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const uint32_t c = (k * kLanes + lane) * T::kVec;
#pragma unroll
      for (int i = 0; i < T::kVec; ++i)
        if (c + i < cols) {
          const Float2 sum = column.at(k * T::kVec + i);
          sums[mine * cols + c + i] = sum.x;
          sums[(teams + mine) * cols + c + i] = sum.y;
        }
    }
  }
}

// dw and db from the teams' sums: a work-group takes 64 columns of one of the
// two, its sixteen waves every sixteenth team; the order is fixed.
template <typename P>
__global__ __launch_bounds__(1024) void layerNormParamKernel(const float* sums, uint64_t teams, uint64_t cols,
                                                             typename P::Stored* dweight, typename P::Stored* dbias) {
  __shared__ float lds[16][64];
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const bool second = blockIdx.y != 0;
  typename P::Stored* out = second ? dbias : dweight;
  if (out == nullptr) return; // the whole work-group
  const uint64_t c = uint64_t(blockIdx.x) * 64 + lane;
  float sum = 0.0f;
  if (c < cols) {
    const float* from = sums + (second ? teams * cols : 0) + c;
#pragma unroll 8
    for (uint64_t t = wave; t < teams; t += 16) sum += from[t * cols];
  }
  lds[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < cols) {
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) total += lds[w][lane];
    out[c] = P::narrow(total);
  }
}

// Long rows, first pass: what a row's gradient needs of the whole row.
struct RowTerms {
  float mean, rstd, alongOnes, alongH;
};
template <typename T, typename P>
__global__ __launch_bounds__(kLongBlock) void layerNormTermsKernel(
    const typename T::Stored* dy, uint64_t dyStride, const typename T::Stored* x, uint64_t xStride,
    const typename P::Stored* weight, const float* means, const float* rstds, float eps, RowTerms* terms,
    uint64_t rows, uint64_t cols) {
  __shared__ float lds[2][16];
  __shared__ Float2 lds2[16];
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    float mean, rstd;
    if (means != nullptr)
      mean = means[row], rstd = rstds[row];
    else
      longStats<T>(x + row * xStride, cols, eps, lds, &mean, &rstd);
    Float2 s{0.0f, 0.0f};
    alongRow<T>(x + row * xStride, cols, [&](uint64_t c, const float* v) {
      float w[T::kVec], g[T::kVec];
      T::unpack(loadPack<T, false>(dy + row * dyStride, c, cols, typename T::Stored(0.0f)), g);
      loadParams<P, T::kVec>(weight, c, cols, 1.0f, w);
      Float2 part{0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < T::kVec; ++i) {
        g[i] *= w[i];
        part.x += g[i];
        part.y += g[i] * (c + i < cols ? (v[i] - mean) * rstd : 0.0f); // -mean * rstd may be infinite
      }
      s.x += part.x;
      s.y += part.y;
    });
    s = teamSum2<16>(s, lds2, 0, threadIdx.x / 64);
    if (threadIdx.x == 0)
      terms[row] = RowTerms{mean, rstd, s.x / static_cast<float>(cols), s.y / static_cast<float>(cols)};
    __syncthreads(); // the next row overwrites lds2
  }
}

// Long rows, second pass: a lane keeps one pack of columns and walks down the
// rows of its slice (blockIdx.y of gridDim.y).
template <typename T, typename P>
__global__ __launch_bounds__(256) void layerNormColumnsKernel(
    const typename T::Stored* dy, uint64_t dyStride, const typename T::Stored* x, uint64_t xStride,
    const typename P::Stored* weight, const RowTerms* terms, typename T::Stored* dx, uint64_t dxStride, float* sums,
    uint64_t rows, uint64_t cols) {
  const uint64_t c = (uint64_t(blockIdx.x) * 256 + threadIdx.x) * T::kVec;
  if (c >= cols) return;
  float w[T::kVec], dw[T::kVec], db[T::kVec];
  loadParams<P, T::kVec>(weight, c, cols, 1.0f, w);
#pragma unroll
  for (int i = 0; i < T::kVec; ++i) dw[i] = db[i] = 0.0f;
  for (uint64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const RowTerms t = terms[row];
    float h[T::kVec], g[T::kVec], out[T::kVec];
    T::unpack(loadPack<T>(x + row * xStride, c, cols, typename T::Stored(0.0f)), h);
    T::unpack(loadPack<T>(dy + row * dyStride, c, cols, typename T::Stored(0.0f)), g);
#pragma unroll
    for (int i = 0; i < T::kVec; ++i) {
      h[i] = (h[i] - t.mean) * t.rstd;
      dw[i] += g[i] * h[i];
      db[i] += g[i];
      out[i] = t.rstd * (g[i] * w[i] - t.alongOnes - h[i] * t.alongH);
    }
    if (dx != nullptr) storePack<T>(dx + row * dxStride, c, cols, out);
  }
  if (sums != nullptr) {
#pragma unroll
    for (int i = 0; i < T::kVec; ++i)
      if (c + i < cols) {
        sums[blockIdx.y * cols + c + i] = dw[i];
        sums[(uint64_t(gridDim.y) + blockIdx.y) * cols + c + i] = db[i];
      }
  }
}

// ---- launches --------------------------------------------------------------------

struct NormArgs {
  const void* x;
  uint64_t xStride;
  const void *weight, *bias;
  float eps;
  void* y;
  uint64_t yStride;
  float *mean, *rstd;
  uint64_t rows, cols;
};
struct NormGradArgs {
  const void* dy;
  uint64_t dyStride;
  const void* x;
  uint64_t xStride;
  const void* weight;
  const float *mean, *rstd;
  float eps;
  void* dx;
  uint64_t dxStride;
  void *dweight, *dbias;
  uint64_t rows, cols;
};

unsigned gridFor(uint64_t rows, uint64_t teamsPerGroup, uint64_t most) {
  return static_cast<unsigned>(std::min((rows + teamsPerGroup - 1) / teamsPerGroup, most));
}

template <typename T, typename P, int kWaves, int kPacks, int kAhead, int kPerCu>
int launchNorm(polar_hip_device* dev, const NormArgs& a) {
  constexpr int kBlock = kWaves * 64 < kTeamBlock ? kTeamBlock : kWaves * 64;
  constexpr int kTeams = kBlock / (kWaves * 64);
  const uint64_t most = uint64_t(dev->info.compute_units) * kPerCu; // work-groups
  POLAR_HIP_TRY(launchKernel(dev, layerNormKernel<T, P, kWaves, kPacks, kAhead>, dim3(gridFor(a.rows, kTeams, most)), dim3(kBlock),
                             static_cast<const typename T::Stored*>(a.x), a.xStride,
                             static_cast<const typename P::Stored*>(a.weight),
                             static_cast<const typename P::Stored*>(a.bias), a.eps,
                             static_cast<typename T::Stored*>(a.y), a.yStride, a.mean, a.rstd, a.rows,
                             static_cast<uint32_t>(a.cols)));
  return POLAR_HIP_OK;
}

template <typename T, typename P> int norm(polar_hip_device* dev, const NormArgs& a) {
  const uint64_t wavePacks = (a.cols + 64 * T::kVec - 1) / (64 * T::kVec); // packs of a wave that a row fills
  // waves per row, packs per lane, rows ahead, work-groups per CU: the fastest of those tried
  // with bf16 rows as long as each line allows (268 MB in and 268 out: 2 waves of 2 packs 48.5
  // us, 4 of 1 53.5; 4 of 2 49.0, 8 of 1 50.6; 8 of 2 with four rows ahead 88.7 for twice
  // that, with one and two groups 90.7, 4 of 4 95)
  if (wavePacks <= 1) return launchNorm<T, P, 1, 1, 1, 6>(dev, a);
  if (wavePacks <= 2) return launchNorm<T, P, 1, 2, 1, 6>(dev, a);
  if (wavePacks <= 4) return launchNorm<T, P, 2, 2, 1, 6>(dev, a);
  if (wavePacks <= 8) return launchNorm<T, P, 4, 2, 1, 4>(dev, a);
  if (wavePacks <= 16) return launchNorm<T, P, 8, 2, 4, 1>(dev, a);
  if (wavePacks <= 32) return launchNorm<T, P, 16, 2, 1, 1>(dev, a);
  if constexpr (T::kVec == 4) {
    if (wavePacks <= 64) return launchNorm<T, P, 16, 4, 1, 1>(dev, a);
  }
  POLAR_HIP_TRY(launchKernel(dev, layerNormLongKernel<T, P>, dim3(gridFor(a.rows, 1, 1u << 20)), dim3(kLongBlock),
                             static_cast<const typename T::Stored*>(a.x), a.xStride,
                             static_cast<const typename P::Stored*>(a.weight),
                             static_cast<const typename P::Stored*>(a.bias), a.eps,
                             static_cast<typename T::Stored*>(a.y), a.yStride, a.mean, a.rstd, a.rows, a.cols));
  return POLAR_HIP_OK;
}

template <typename P>
int launchParams(polar_hip_device* dev, const NormGradArgs& a, const float* sums, uint64_t teams) {
  POLAR_HIP_TRY(launchKernel(dev, layerNormParamKernel<P>, dim3(static_cast<unsigned>((a.cols + 63) / 64), 2), dim3(1024),
                             sums, teams, a.cols, static_cast<typename P::Stored*>(a.dweight),
                             static_cast<typename P::Stored*>(a.dbias)));
  return POLAR_HIP_OK;
}

template <typename T, typename P, int kWaves, int kPacks, int kAhead, int kPerCu>
int launchNormGrad(polar_hip_device* dev, const NormGradArgs& a) {
  constexpr int kBlock = kWaves * 64 < kTeamBlock ? kTeamBlock : kWaves * 64;
  constexpr int kTeams = kBlock / (kWaves * 64);
  const bool params = a.dweight != nullptr || a.dbias != nullptr;
  const unsigned grid = gridFor(a.rows, kTeams, uint64_t(dev->info.compute_units) * kPerCu);
  const uint64_t teams = uint64_t(grid) * kTeams;
  std::lock_guard<std::mutex> lock(dev->workspaceMu);
  void* area = nullptr;
  if (params) {
    const int st = workspaceFor(dev, 2 * teams * a.cols * sizeof(float), &area);
    if (st != POLAR_HIP_OK) return st;
  }
  auto kernel = a.mean == nullptr ? layerNormGradKernel<T, P, kWaves, kPacks, kAhead, true>
                                  : layerNormGradKernel<T, P, kWaves, kPacks, kAhead, false>;
  constexpr uint32_t ldsBytes = ColumnSums<kWaves, kPacks, T::kVec>::kLdsBytes;
  if constexpr (ldsBytes > 48 * 1024) { // has to be asked for, once per kernel and device (asking twice is harmless)
    static std::atomic<uint64_t> raised[2]; // with statistics of its own, and without
    const uint64_t bit = 1ull << (dev->ordinal & 63);
    std::atomic<uint64_t>& done = raised[a.mean == nullptr];
    if (!(done.load(std::memory_order_acquire) & bit)) {
      POLAR_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                        int(ldsBytes)));
      done.fetch_or(bit, std::memory_order_release);
    }
  }
  POLAR_HIP_TRY(launchKernelLds(dev, kernel, dim3(grid), dim3(kBlock), ldsBytes,
                                static_cast<const typename T::Stored*>(a.dy), a.dyStride,
                                static_cast<const typename T::Stored*>(a.x), a.xStride,
                                static_cast<const typename P::Stored*>(a.weight), a.mean, a.rstd, a.eps,
                                static_cast<typename T::Stored*>(a.dx), a.dxStride, static_cast<float*>(area), a.rows,
                                static_cast<uint32_t>(a.cols)));
  return params ? launchParams<P>(dev, a, static_cast<const float*>(area), teams) : POLAR_HIP_OK;
}

template <typename T, typename P> int launchLongGrad(polar_hip_device* dev, const NormGradArgs& a) {
  const bool params = a.dweight != nullptr || a.dbias != nullptr;
  const uint64_t groups = (a.cols + 256 * T::kVec - 1) / (256 * T::kVec);
  // slices of the rows: work for two work-groups per CU, sums of at most 64 MiB
  uint64_t slices = std::max<uint64_t>(1, 2 * dev->info.compute_units / groups);
  slices = std::min(slices, std::max<uint64_t>(1, (64ull << 20) / (2 * a.cols * sizeof(float))));
  slices = std::min(slices, a.rows);
  const uint64_t termBytes = (a.rows * sizeof(RowTerms) + 255) / 256 * 256;
  std::lock_guard<std::mutex> lock(dev->workspaceMu);
  void* area = nullptr;
  const int st = workspaceFor(dev, termBytes + (params ? 2 * slices * a.cols * sizeof(float) : 0), &area);
  if (st != POLAR_HIP_OK) return st;
  RowTerms* terms = static_cast<RowTerms*>(area);
  float* sums = params ? reinterpret_cast<float*>(static_cast<char*>(area) + termBytes) : nullptr;
  const auto* dy = static_cast<const typename T::Stored*>(a.dy);
  const auto* x = static_cast<const typename T::Stored*>(a.x);
  const auto* weight = static_cast<const typename P::Stored*>(a.weight);
  POLAR_HIP_TRY(launchKernel(dev, layerNormTermsKernel<T, P>, dim3(gridFor(a.rows, 1, 1u << 20)), dim3(kLongBlock), dy,
                             a.dyStride, x, a.xStride, weight, a.mean, a.rstd, a.eps, terms, a.rows, a.cols));
  POLAR_HIP_TRY(launchKernel(dev, layerNormColumnsKernel<T, P>,
                             dim3(static_cast<unsigned>(groups), static_cast<unsigned>(slices)), dim3(256), dy,
                             a.dyStride, x, a.xStride, weight, static_cast<const RowTerms*>(terms),
                             static_cast<typename T::Stored*>(a.dx), a.dxStride, sums, a.rows, a.cols));
  return params ? launchParams<P>(dev, a, sums, slices) : POLAR_HIP_OK;
}

template <typename T, typename P> int normGrad(polar_hip_device* dev, const NormGradArgs& a) {
  const uint64_t wavePacks = (a.cols + 64 * T::kVec - 1) / (64 * T::kVec);
  // as above; two groups of four waves per CU, or one of eight or more, as each team adds
  // its sums to what the second kernel reads (16384 x 4096: 8 waves of 1 pack with four rows
  // ahead 75.5 us, 4 of 2 with one 82, twice the groups 84; 32768 x 2048: 4 waves of 1 with two
  // rows ahead and two groups 76.9, one group 105; 65536 x 1024: 1 wave of 2 with three ahead
  // 78.9, one 85.7)
  if (wavePacks <= 1) return launchNormGrad<T, P, 1, 1, 3, 2>(dev, a);
  if (wavePacks <= 2) return launchNormGrad<T, P, 1, 2, 3, 2>(dev, a);
  if (wavePacks <= 4) return launchNormGrad<T, P, 4, 1, 2, 2>(dev, a);
  if (wavePacks <= 8) return launchNormGrad<T, P, 8, 1, 4, 1>(dev, a);
  if (wavePacks <= 16) return launchNormGrad<T, P, 8, 2, 2, 1>(dev, a);
  if constexpr (T::kVec == 8) {
    if (wavePacks <= 32) return launchNormGrad<T, P, 16, 2, 1, 1>(dev, a);
  } else {
    if (wavePacks <= 32) return launchNormGrad<T, P, 8, 4, 1, 1>(dev, a);
    if (wavePacks <= 64) return launchNormGrad<T, P, 16, 4, 1, 1>(dev, a);
  }
  return launchLongGrad<T, P>(dev, a);
}

template <typename Args, typename F32, typename Same16, typename Wide16, typename SameB, typename WideB>
int byTypes(int type, int paramType, polar_hip_device* dev, const Args& a, F32 f32, Same16 same16, Wide16 wide16,
            SameB sameB, WideB wideB) {
  if (type == POLAR_HIP_F32) return f32(dev, a);
  const bool wide = paramType == POLAR_HIP_F32;
  if (type == POLAR_HIP_F16) return wide ? wide16(dev, a) : same16(dev, a);
  return wide ? wideB(dev, a) : sameB(dev, a);
}

// largest row: its length is exact in fp32, the divisor of the means
constexpr uint64_t kMaxCols = 1ull << 24;

} // namespace

extern "C" {

int polar_hip_flayernorm(polar_hip_device* dev, int type, const void* x, uint64_t xStride, int paramType,
                         const void* weight, const void* bias, float eps, void* y, uint64_t yStride, float* mean,
                         float* rstd, uint64_t rows, uint64_t cols) {
  POLAR_HIP_REQUIRE(dev != nullptr, "dev is null");
  POLAR_HIP_REQUIRE(knownType(type), "unknown element type");
  POLAR_HIP_REQUIRE(paramType == type || paramType == POLAR_HIP_F32, "parameters are fp32 or of the tensor's type");
  POLAR_HIP_REQUIRE(eps >= 0.0f && std::isfinite(eps), "eps must be finite and not negative");
  POLAR_HIP_REQUIRE(cols >= 1 && cols <= kMaxCols, "rows of 1 to 2^24 elements");
  if (rows == 0) return POLAR_HIP_OK;
  POLAR_HIP_REQUIRE(x && y, "null tensor");
  POLAR_HIP_REQUIRE(xStride >= cols && yStride >= cols, "a row's stride is shorter than the row");
  POLAR_HIP_REQUIRE(addressable(rows, std::max(xStride, yStride), sizeOf(type)), "tensor too large");
  POLAR_HIP_REQUIRE(alignedTo(x, sizeOf(type)) && alignedTo(y, sizeOf(type)) && alignedTo(weight, sizeOf(paramType)) &&
                        alignedTo(bias, sizeOf(paramType)) && alignedTo(mean, 4) && alignedTo(rstd, 4),
                    "misaligned pointer");
  POLAR_HIP_REQUIRE(x != y || xStride == yStride, "in place needs equal strides");
  POLAR_HIP_TRY(hipSetDevice(dev->ordinal));
  const NormArgs a{x, xStride, weight, bias, eps, y, yStride, mean, rstd, rows, cols};
  return byTypes(type, paramType, dev, a, norm<TypeF32, TypeF32>, norm<TypeF16, TypeF16>, norm<TypeF16, TypeF32>,
                 norm<TypeBF16, TypeBF16>, norm<TypeBF16, TypeF32>);
}

int polar_hip_flayernorm_grad(polar_hip_device* dev, int type, const void* dy, uint64_t dyStride, const void* x,
                              uint64_t xStride, int paramType, const void* weight, const float* mean,
                              const float* rstd, float eps, void* dx, uint64_t dxStride, void* dweight, void* dbias,
                              uint64_t rows, uint64_t cols) {
  POLAR_HIP_REQUIRE(dev != nullptr, "dev is null");
  POLAR_HIP_REQUIRE(knownType(type), "unknown element type");
  POLAR_HIP_REQUIRE(paramType == type || paramType == POLAR_HIP_F32, "parameters are fp32 or of the tensor's type");
  POLAR_HIP_REQUIRE((mean == nullptr) == (rstd == nullptr), "mean and rstd come together");
  POLAR_HIP_REQUIRE(mean != nullptr || (eps >= 0.0f && std::isfinite(eps)), "eps must be finite and not negative");
  POLAR_HIP_REQUIRE(cols >= 1 && cols <= kMaxCols, "rows of 1 to 2^24 elements");
  POLAR_HIP_REQUIRE(rows < (1ull << 31), "too many rows");
  POLAR_HIP_REQUIRE(rows == 0 || (dy && x), "null tensor");
  POLAR_HIP_REQUIRE(rows == 0 || (dyStride >= cols && xStride >= cols && (dx == nullptr || dxStride >= cols)),
                    "a row's stride is shorter than the row");
  POLAR_HIP_REQUIRE(addressable(rows, std::max({dyStride, xStride, dx ? dxStride : 0}), sizeOf(type)), "tensor too large");
  POLAR_HIP_REQUIRE(alignedTo(dy, sizeOf(type)) && alignedTo(x, sizeOf(type)) && alignedTo(dx, sizeOf(type)) &&
                        alignedTo(weight, sizeOf(paramType)) && alignedTo(dweight, sizeOf(paramType)) &&
                        alignedTo(dbias, sizeOf(paramType)) && alignedTo(mean, 4) && alignedTo(rstd, 4),
                    "misaligned pointer");
  POLAR_HIP_REQUIRE(dx == nullptr || ((dx != dy || dxStride == dyStride) && (dx != x || dxStride == xStride)),
                    "in place needs equal strides");
  if (dx == nullptr && dweight == nullptr && dbias == nullptr) return POLAR_HIP_OK;
  POLAR_HIP_TRY(hipSetDevice(dev->ordinal));
  const NormGradArgs a{dy, dyStride, x, xStride, weight, mean, rstd, eps, dx, dxStride, dweight, dbias, rows, cols};
  if (rows == 0) // sums over no rows
    return paramType == POLAR_HIP_F32   ? launchParams<TypeF32>(dev, a, nullptr, 0)
           : paramType == POLAR_HIP_F16 ? launchParams<TypeF16>(dev, a, nullptr, 0)
                                        : launchParams<TypeBF16>(dev, a, nullptr, 0);
  return byTypes(type, paramType, dev, a, normGrad<TypeF32, TypeF32>, normGrad<TypeF16, TypeF16>,
                 normGrad<TypeF16, TypeF32>, normGrad<TypeBF16, TypeBF16>, normGrad<TypeBF16, TypeF32>);
}

} // extern "C"
