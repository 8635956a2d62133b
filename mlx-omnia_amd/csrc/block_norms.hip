// The norms around a block, with its gate and scales: the gated norm of a mixer's output in
// groups, and the join of two blocks. Everything in fp32 from the bf16 inputs to one rounding
// for each output; the sums of squares are fp32 (8 to 16384 terms: at most 16 in turn, then in a tree
// over a lane's places and the lanes and, of a row, over up to eight waves in turn: under 30 roundings of
// 2^-24). Both read each tensor once and write each result once, and
// are bound by that from a few hundred rows on, by the launch below.
#include "common.hpp"
#include "host.hpp"

namespace omnia {
namespace {

// A lane's sum of squares: up to 16 one after another; of more vectors their first values, second and so
// on each by themselves, then in a tree. (Of 128 one after another small ones behind a large one were
// lost; with 16 in a tree 8,192 rows of 4,096 with the gate first took 38 us for 36.2.)
template <int kVectors>
__device__ __forceinline__ float squares(const float (&y)[kVectors][8]) {
  constexpr int kSums = kVectors <= 2 ? 1 : 8;
  float sums[8] = {};
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[j % kSums] = __builtin_fmaf(y[i][j], y[i][j], sums[j % kSums]);
  }
  if constexpr (kSums == 1) return sums[0];
  return ((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7]));
}

// 1 / (1 + exp(-z)): exact ends (an exponential that overflows gives 0).
__device__ __forceinline__ float sigmoid(float z) { return 1.0f / (1.0f + __expf(-z)); }

struct GatedArgs {
  const uint16_t *x, *gate, *weight;
  int64_t x_stride, gate_stride;
  uint16_t* out;
  int64_t items;     // rows * groups
  int groups, vectors, weight_step;
  float inverse_group, eps;
  int silu;
};

// A group of values per kLanes lanes, kVectors 16-byte vectors each. (Where the gate stands is known when
// it is built: asked for in the kernel, groups of 512 with the gate first took 37.4 -> 41.5 us.)
template <int kLanes, int kVectors, bool kGateFirst>
__global__ __launch_bounds__(256) void gated_rms_norm_kernel(GatedArgs a) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  if (item >= a.items) return;   // whole groups of lanes
  const int64_t row = item / a.groups;
  const int group = static_cast<int>(item - row * a.groups);
  const uint16_t* x = a.x + row * a.x_stride + static_cast<int64_t>(group) * a.vectors * 8;
  const uint16_t* gate = a.gate + row * a.gate_stride + static_cast<int64_t>(group) * a.vectors * 8;
  const uint16_t* weight = a.weight + static_cast<int64_t>(group) * a.weight_step;
  u32x4 xs[kVectors], gs[kVectors], ws[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int at = lane + i * kLanes;
    const bool there = at < a.vectors;
    xs[i] = there ? *reinterpret_cast<const u32x4*>(x + at * 8) : u32x4{0, 0, 0, 0};
    gs[i] = there ? *reinterpret_cast<const u32x4*>(gate + at * 8) : u32x4{0, 0, 0, 0};
    ws[i] = there ? *reinterpret_cast<const u32x4*>(weight + at * 8) : u32x4{0, 0, 0, 0};
  }
  // The gate where the formula has it: behind the norm it may overflow with a value that the norm makes small.
  float y[kVectors][8];
  const auto gated = [&](int i) {
    float z[8];
    unpack8(gs[i], z);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i][j] *= (a.silu ? z[j] : 1.0f) * sigmoid(z[j]);
  };
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    unpack8(xs[i], y[i]);
    if constexpr (kGateFirst) gated(i);
  }
  const float sum = group_sum<kLanes>(squares(y));
  const float inverse = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum, a.inverse_group, a.eps));
  uint16_t* out = a.out + item * (a.vectors * 8);
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int at = lane + i * kLanes;
    float w[8];
    unpack8(ws[i], w);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i][j] = y[i][j] * inverse * w[j];
    if constexpr (!kGateFirst) gated(i);
    if (at < a.vectors) *reinterpret_cast<u32x4*>(out + at * 8) = pack8(y[i]);
  }
}

struct BlockArgs {
  const uint16_t *x, *block, *gate, *post, *pre;
  int64_t gate_stride;
  uint16_t *summed, *normalized;
  int vectors;
  float hidden, post_eps, pre_eps, residual_scale, block_scale;
  int sigmoid;
};

// The sum over the workgroup, the same in every lane: each wave's, then those in turn.
template <int kWaves>
__device__ __forceinline__ float block_sum(float v, float* parts) {
  v = wave_sum_f32(v);
  if constexpr (kWaves == 1) return v;
  if (threadIdx.x % kWave == 0) parts[threadIdx.x / kWave] = v;
  lds_barrier();
  v = parts[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v += parts[w];
  return v;
}

// A row per workgroup of kWaves, kVectors 16-byte vectors a lane, read past the caches (8,192 rows of
// 5,120 with a gate: 76.2 -> 71.8 us; the stores past them as well 72.0, and what follows reads those).
template <int kWaves, int kVectors>
__global__ __launch_bounds__(64 * kWaves) void block_norm_kernel(BlockArgs a) {
  constexpr int kThreads = 64 * kWaves;
  __shared__ float parts[2][kWaves];
  const int64_t row = blockIdx.x;
  const int64_t first = row * a.vectors * 8;
  u32x4 xs[kVectors], bs[kVectors], gs[kVectors], posts[kVectors], pres[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int at = threadIdx.x + i * kThreads;
    const bool there = at < a.vectors;
    const u32x4 zero = u32x4{0, 0, 0, 0};
    bs[i] = there ? load_nt(reinterpret_cast<const u32x4*>(a.block + first + at * 8)) : zero;
    xs[i] = there ? load_nt(reinterpret_cast<const u32x4*>(a.x + first + at * 8)) : zero;
    gs[i] = there && a.gate ? load_nt(reinterpret_cast<const u32x4*>(a.gate + row * a.gate_stride + at * 8)) : zero;
    posts[i] = there && a.post ? *reinterpret_cast<const u32x4*>(a.post + at * 8) : zero;
    pres[i] = there ? *reinterpret_cast<const u32x4*>(a.pre + at * 8) : zero;
  }
  float s[kVectors][8];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) unpack8(bs[i], s[i]);
  if (a.post != nullptr) {
    const float inverse = 1.0f / __builtin_sqrtf(block_sum<kWaves>(squares(s), parts[0]) / a.hidden + a.post_eps);
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      float w[8];
      unpack8(posts[i], w);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] = s[i][j] * inverse * w[j];
    }
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    float x[8], g[8];
    unpack8(xs[i], x);
    unpack8(gs[i], g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (a.gate != nullptr) s[i][j] *= a.sigmoid ? sigmoid(g[j]) : g[j];
      s[i][j] = __builtin_fmaf(a.block_scale, s[i][j], a.residual_scale * x[j]);
    }
  }
  const float inverse = 1.0f / __builtin_sqrtf(block_sum<kWaves>(squares(s), parts[1]) / a.hidden + a.pre_eps);
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const int at = threadIdx.x + i * kThreads;
    if (at >= a.vectors) continue;
    *reinterpret_cast<u32x4*>(a.summed + first + at * 8) = pack8(s[i]);
    float w[8];
    unpack8(pres[i], w);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = s[i][j] * inverse * w[j];
    *reinterpret_cast<u32x4*>(a.normalized + first + at * 8) = pack8(w);
  }
}

template <int kLanes, int kVectors>
void launch_gated(const GatedArgs& a, int64_t blocks, bool gate_first, hipStream_t stream) {
  if (gate_first) gated_rms_norm_kernel<kLanes, kVectors, true><<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(a);
  else gated_rms_norm_kernel<kLanes, kVectors, false><<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(a);
}

template <int kWaves, int kVectors>
void launch_block(const BlockArgs& a, int64_t rows, hipStream_t stream) {
  block_norm_kernel<kWaves, kVectors><<<dim3(static_cast<unsigned>(rows)), 64 * kWaves, 0, stream>>>(a);
}

}  // namespace
}  // namespace omnia

extern "C" int32_t omnia_gated_rms_norm(const uint16_t* x, int64_t x_stride, const uint16_t* gate, int64_t gate_stride,
                                        const uint16_t* weight, int64_t weight_width, int64_t rows, int64_t width,
                                        int64_t group, float eps, int32_t silu, int32_t gate_first, uint16_t* out,
                                        hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(group > 0 && group % 8 == 0 && group <= 8192, "gated_rms_norm: group must be a multiple of 8, at most 8192");
  OMNIA_REQUIRE(width > 0 && width % group == 0 && width < (int64_t{1} << 24), "gated_rms_norm: width must be whole groups");
  OMNIA_REQUIRE(weight_width == group || weight_width == width, "gated_rms_norm: the weight must cover a group or a row");
  OMNIA_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31), "gated_rms_norm: bad row count");
  if (rows == 0) return 0;
  OMNIA_REQUIRE(x && gate && weight && out, "gated_rms_norm: null pointer");
  OMNIA_REQUIRE(aligned16(x) && aligned16(gate) && aligned16(weight) && aligned16(out),
                "gated_rms_norm: pointers must be 16-byte aligned");
  OMNIA_REQUIRE(x_stride % 8 == 0 && gate_stride % 8 == 0 && x_stride >= width && gate_stride >= width,
                "gated_rms_norm: row strides must be multiples of 8 covering the row");
  const int64_t groups = width / group;
  const int vectors = static_cast<int>(group / 8);
  // Two vectors a lane, and past a wave more: 8,192 rows of 4,096 (201 MB) took 37.2, 36.7 and 48.2 us with
  // one, two and four in groups of 64, 41, 35.8 and 38 of 128, 40.2, 36.4 (5.5 TB/s) and 37.8 of 512. (Read
  // past the caches, groups of 64 43.1 for 37.2, the others as they are.)
  const int lanes = vectors <= 8 ? 4 : vectors <= 16 ? 8 : vectors <= 32 ? 16 : vectors <= 64 ? 32 : 64;
  const int64_t blocks = (rows * groups + 256 / lanes - 1) / (256 / lanes);
  OMNIA_REQUIRE(fits_launch(blocks, 256), "gated_rms_norm: too many groups for one launch");
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  const GatedArgs a{x, gate, weight, x_stride, gate_stride, out, rows * groups, static_cast<int>(groups), vectors,
                    weight_width == width ? static_cast<int>(group) : 0, 1.0f / static_cast<float>(group), eps, silu};
  const auto launch = lanes == 4 ? launch_gated<4, 2> : lanes == 8 ? launch_gated<8, 2> : lanes == 16 ? launch_gated<16, 2>
                      : lanes == 32 ? launch_gated<32, 2> : vectors <= 128 ? launch_gated<64, 2>
                      : vectors <= 256 ? launch_gated<64, 4> : vectors <= 512 ? launch_gated<64, 8> : launch_gated<64, 16>;
  launch(a, blocks, gate_first != 0, stream);
  return launched("gated_rms_norm");
}

extern "C" int32_t omnia_block_norm(const uint16_t* x, const uint16_t* block, const uint16_t* gate, int64_t gate_stride,
                                    int32_t sigmoid, const uint16_t* post_weight, float post_eps,
                                    const uint16_t* pre_weight, float pre_eps, float residual_scale, float block_scale,
                                    int64_t rows, int64_t hidden, uint16_t* summed, uint16_t* normalized,
                                    hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(hidden > 0 && hidden % 8 == 0 && hidden <= 16384, "block_norm: hidden must be a multiple of 8, at most 16384");
  OMNIA_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31), "block_norm: bad row count");
  if (rows == 0) return 0;
  OMNIA_REQUIRE(x && block && pre_weight && summed && normalized, "block_norm: null pointer");
  OMNIA_REQUIRE(aligned16(x) && aligned16(block) && aligned16(gate) && aligned16(post_weight) && aligned16(pre_weight) &&
                    aligned16(summed) && aligned16(normalized),
                "block_norm: pointers must be 16-byte aligned");
  OMNIA_REQUIRE(gate == nullptr || gate_stride == 0 || (gate_stride % 8 == 0 && gate_stride >= hidden),
                "block_norm: the gate's row stride must be 0 or a multiple of 8 covering the row");
  const int vectors = static_cast<int>(hidden / 8);
  // The fewest waves that hold the row a vector a lane, and past eight more vectors a lane.
  const int waves = vectors <= 64 ? 1 : vectors <= 128 ? 2 : vectors <= 256 ? 4 : 8;
  OMNIA_REQUIRE(fits_launch(rows, 64 * waves), "block_norm: too many rows for one launch");
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  const BlockArgs a{x, block, gate, post_weight, pre_weight, gate_stride, summed, normalized, vectors,
                    static_cast<float>(hidden), post_eps, pre_eps, residual_scale, block_scale, sigmoid};
  if (waves == 1) launch_block<1, 1>(a, rows, stream);
  else if (waves == 2) launch_block<2, 1>(a, rows, stream);
  else if (waves == 4) launch_block<4, 1>(a, rows, stream);
  else if (vectors <= 512) launch_block<8, 1>(a, rows, stream);
  else if (vectors <= 1024) launch_block<8, 2>(a, rows, stream);
  else launch_block<8, 4>(a, rows, stream);
  return launched("block_norm");
}
