// Linear attention with a decay for each head (the mixers whose state stands in place of a
// cache of rows):
//   S_t = exp(g_t) S_{t-1} + w_t k_t v_t^T,   o_t = scale * q_t S_t
// over each sequence's new tokens, S [DK, DV] in fp32 read from and left in the pool of states.
//
// Steps: a workgroup takes one head of one sequence with its whole state in registers (64 KB at
// 128 x 128, 16 vectors of 16 bytes a lane, all asked for at once), so a step of one token reads
// and writes the state once and is bound by that.
#include "common.hpp"
#include "host.hpp"

namespace omnia {
namespace {

struct LinearArgs {
  const uint16_t *q, *k, *v;
  const float *decay, *strength;
  float* states;
  const int32_t* steps;
  uint16_t* out;
  int64_t q_stride, k_stride, v_stride, decay_stride, strength_stride;
  int slots, tokens, heads, group;
  float scale;
};

template <int DK, int DV>
__global__ __launch_bounds__(256) void linear_step_kernel(LinearArgs a) {
  constexpr int kLanes = DV / 4;              // lanes of a state row
  constexpr int kRows = 256 / kLanes;         // rows of a pass
  constexpr int kPasses = DK / kRows;
  constexpr int kWaves = 4;
  __shared__ float key[2][DK], query[2][DK];
  __shared__ f32x4 sums[2][kWaves][kLanes];
  const int entry = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const int slot = a.steps[3 * entry], first = a.steps[3 * entry + 1], count = a.steps[3 * entry + 2];
  if (slot < 0 || slot >= a.slots || first < 0 || count <= 0 || count > a.tokens - first) return;
  const int column = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  float* state = a.states + (static_cast<int64_t>(slot) * a.heads + head) * (DK * DV) + row * DV + 4 * column;
  f32x4 s[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) s[i] = *reinterpret_cast<const f32x4*>(state + i * kRows * DV);
  const int shared = head / a.group;
  for (int t = 0; t < count; ++t) {
    const int64_t token = first + t;
    const int turn = t & 1;
    if (threadIdx.x < DK) {
      key[turn][threadIdx.x] = bf16_to_f32(a.k[token * a.k_stride + shared * DK + threadIdx.x]);
    } else if (threadIdx.x < 2 * DK) {
      query[turn][threadIdx.x - DK] = bf16_to_f32(a.q[token * a.q_stride + shared * DK + threadIdx.x - DK]);
    }
    const uint2 raw = *reinterpret_cast<const uint2*>(a.v + token * a.v_stride + head * DV + 4 * column);
    // A slow decay is taken as S + (exp(g) - 1) S: exp(g) itself, rounded next to 1, would be off the
    // same way at every token of a sequence.
    const float rate = expm1f(a.decay[token * a.decay_stride + head]);
    const bool slow = rate > -0.5f;
    const float factor = slow ? rate : rate + 1.0f;
    const float strength = a.strength != nullptr ? a.strength[token * a.strength_stride + head] : 1.0f;
    const float v[4] = {bf16_lo(raw.x) * strength, bf16_hi(raw.x) * strength, bf16_lo(raw.y) * strength,
                        bf16_hi(raw.y) * strength};
    lds_barrier();
    float o[4] = {};
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const float kr = key[turn][row + i * kRows], qr = query[turn][row + i * kRows];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float next = __builtin_fmaf(s[i][j], factor, kr * v[j]);
        s[i][j] = slow ? s[i][j] + next : next;
        o[j] = __builtin_fmaf(qr, s[i][j], o[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int offset = kLanes; offset < kWave; offset *= 2) o[j] += __shfl_xor(o[j], offset, kWave);
    }
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave < kLanes) sums[turn][wave][column] = f32x4{o[0], o[1], o[2], o[3]};
    lds_barrier();
    // (The next token's rows go to the other half, and the one after's behind its barrier.)
    if (threadIdx.x < kLanes) {
      f32x4 total = sums[turn][0][column];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) total += sums[turn][w][column];
      uint2 packed;
      packed.x = pack_bf16(total[0] * a.scale, total[1] * a.scale);
      packed.y = pack_bf16(total[2] * a.scale, total[3] * a.scale);
      *reinterpret_cast<uint2*>(a.out + (token * a.heads + head) * DV + 4 * column) = packed;
    }
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) *reinterpret_cast<f32x4*>(state + i * kRows * DV) = s[i];
}

}  // namespace
}  // namespace omnia

extern "C" int32_t omnia_linear_attention(const omnia_linear_attention_t* c, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(c != nullptr, "linear_attention: null pointer");
  OMNIA_REQUIRE((c->key_dim == 64 || c->key_dim == 128) && (c->value_dim == 64 || c->value_dim == 128),
                "linear_attention: key_dim and value_dim must be 64 or 128");
  OMNIA_REQUIRE(c->key_heads > 0 && c->heads > 0 && c->heads <= 4096 && c->heads % c->key_heads == 0,
                "linear_attention: heads must be a multiple of key_heads");
  constexpr int64_t kMost = int64_t{1} << 24;
  OMNIA_REQUIRE(c->tokens >= 0 && c->tokens < kMost && c->step_count >= 0 && c->step_count <= c->tokens &&
                    c->slots >= 0 && c->slots < kMost,
                "linear_attention: bad token, step or slot count");
  if (c->step_count == 0) return 0;
  OMNIA_REQUIRE(c->queries && c->keys && c->values && c->log_decay && c->states && c->steps && c->out,
                "linear_attention: null pointer");
  OMNIA_REQUIRE(aligned16(c->queries) && aligned16(c->keys) && aligned16(c->values) && aligned16(c->states) &&
                    aligned16(c->out),
                "linear_attention: pointers must be 16-byte aligned");
  OMNIA_REQUIRE(c->query_stride % 8 == 0 && c->key_stride % 8 == 0 && c->value_stride % 8 == 0 &&
                    c->query_stride >= c->key_heads * c->key_dim && c->key_stride >= c->key_heads * c->key_dim &&
                    c->value_stride >= c->heads * c->value_dim && c->query_stride < kMost && c->key_stride < kMost &&
                    c->value_stride < kMost,
                "linear_attention: row strides must be multiples of 8 covering the heads, below 2^24");
  OMNIA_REQUIRE((c->decay_stride == 0 || c->decay_stride >= c->heads) &&
                    (c->strengths == nullptr || c->strength_stride >= c->heads),
                "linear_attention: decay and strength rows must cover the heads");
  const int64_t blocks = c->step_count * c->heads;
  OMNIA_REQUIRE(blocks < (int64_t{1} << 31), "linear_attention: too many steps");
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  const LinearArgs a{c->queries, c->keys, c->values, c->log_decay, c->strengths, c->states, c->steps, c->out,
                     c->query_stride, c->key_stride, c->value_stride, c->decay_stride, c->strength_stride,
                     static_cast<int>(c->slots), static_cast<int>(c->tokens), static_cast<int>(c->heads),
                     static_cast<int>(c->heads / c->key_heads), c->scale};
  const auto kernel = c->key_dim == 64
                          ? (c->value_dim == 64 ? linear_step_kernel<64, 64> : linear_step_kernel<64, 128>)
                          : (c->value_dim == 64 ? linear_step_kernel<128, 64> : linear_step_kernel<128, 128>);
  kernel<<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(a);
  return launched("linear_attention");
}
