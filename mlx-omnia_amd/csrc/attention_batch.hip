// Attention of a batch of sequences over a cache of pages, the rows that all of them share
// taken once.
//
// Every new token of the batch is normed, rotated and written at its own sequence's position
// by one launch; its attention is then cut into pieces of keys,
//   rows [0, prefix)            the same pages for every sequence: one workgroup multiplies a
//                               tile of queries from any of the sequences with them
//   rows [prefix, limit of q)   each sequence's own pages
// and each piece leaves (m, l, c) = (max, sum of 2^(s - m), sum of 2^(s - m) v) of its scores
// s = q . k * scale * log2(e). Pieces merge exactly: with M = max m_p,
//   l = sum l_p 2^(m_p - M),  out = sum c_p 2^(m_p - M) / (l + 2^(sink log2(e) - M)).
#include <cfloat>

#include "common.hpp"
#include "host.hpp"

namespace omnia {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4_lds __attribute__((ext_vector_type(4)));

// The tables of a pool, as the kernels follow them: every id is checked where it is read.
struct PageTables {
  const int32_t* tables;    // [sequences, width] page ids
  const int32_t* lengths;   // [sequences] rows before this step
  const int2* tokens;       // [tokens] (sequence, its how many-th new token)
  int sequences, width, pages, page_shift;

  // Rows of a token's sequence before it, or -1 for a sequence outside the tables.
  __device__ __forceinline__ int before(int2 token) const { return rows_before(token.x, token.y); }
  __device__ __forceinline__ int rows_before(int sequence, int j) const {
    return sequence >= 0 && sequence < sequences ? lengths[sequence] + j : -1;
  }
  // The page of a sequence's row, or -1 where there is none.
  __device__ __forceinline__ int page(int sequence, int row) const {
    const int index = row >> page_shift;
    if (sequence < 0 || sequence >= sequences || index < 0 || index >= width) return -1;
    const int id = tables[static_cast<int64_t>(sequence) * width + index];
    return id < pages ? id : -1;
  }
  // A kv head's row of a page, counted in rows of the pool.
  __device__ __forceinline__ int64_t row_of(int page, int kv_heads, int kv_head, int row) const {
    return ((static_cast<int64_t>(page) * kv_heads + kv_head) << page_shift) + (row & ((1 << page_shift) - 1));
  }
};

// ---- prologue -------------------------------------------------------------------------

struct BatchProjectArgs {
  const uint16_t* raw[3];   // queries, keys, values: rows of heads x D, `stride` apart
  int64_t stride[3];
  const uint16_t* gain[2];  // query and key norm weights [D], or null
  const float* cos;         // [angle_rows, pairs] rows `table_stride` floats apart
  const float* sin;
  int64_t table_stride, angle_rows;
  void* queries;            // [tokens, heads, D] bf16, or fp32 with `wide`
  uint16_t* pool[2];        // a layer's keys and values [pages, kv_heads, page_rows, D]
  PageTables at;
  int heads, kv_heads, tokens, pairs, wide;
  float mscale, eps;
};

// A head vector per D / 8 lanes, 16 bytes a lane, kHeads of one token in turn: what is the
// token's (sequence, position, page, angles) is looked up once for them, and their loads are
// under way together. (Its angles are four times a lane's bytes of a head: read for each head
// and with an index division, 7,000 tokens of 64 heads took 31 us.) The norm, the rotation and
// mscale stay in fp32 and are rounded once, where they are stored. Bound by its launch at a few
// tokens (where a head in turn is the faster: 128 tokens of 48 heads 5.3 us for 8.1) and by
// memory at a prompt.
template <int D, int kHeads>
__global__ __launch_bounds__(256) void attention_batch_project_kernel(BatchProjectArgs a) {
  constexpr int kLanes = D / 8, kGroups = 256 / kLanes;
  const int64_t token = blockIdx.x;
  const int lane = threadIdx.x % kLanes;
  const int first = static_cast<int>(blockIdx.y) * kGroups * kHeads + threadIdx.x / kLanes;
  const int slots = a.heads + 2 * a.kv_heads;
  u32x4 raw[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int slot = min(first + i * kGroups, slots - 1);
    const int part = slot < a.heads ? 0 : slot < a.heads + a.kv_heads ? 1 : 2;
    const int head = slot - (part == 0 ? 0 : part == 1 ? a.heads : a.heads + a.kv_heads);
    raw[i] = *reinterpret_cast<const u32x4*>(a.raw[part] + token * a.stride[part] + head * D + lane * 8);
  }
  const int2 whose = a.at.tokens[token];
  const int position = a.at.before(whose);
  const int page = position < 0 ? -1 : a.at.page(whose.x, position);
  const int half = a.pairs / 8;   // lanes of one half of the rotated block
  const bool turned = lane < 2 * half;
  const int partner = lane < half ? lane + half : turned ? lane - half : lane;
  float c[8], s[8];
  if (a.pairs > 0) {
    // Lanes past the rotated block read its first angles and keep their values; a position past
    // the table reads its last row.
    const int64_t row = min(static_cast<int64_t>(max(position, 0)), a.angle_rows - 1) * a.table_stride;
    const int at = turned ? (lane < half ? lane : lane - half) * 8 : 0;
    *reinterpret_cast<f32x4*>(c) = *reinterpret_cast<const f32x4*>(a.cos + row + at);
    *reinterpret_cast<f32x4*>(c + 4) = *reinterpret_cast<const f32x4*>(a.cos + row + at + 4);
    *reinterpret_cast<f32x4*>(s) = *reinterpret_cast<const f32x4*>(a.sin + row + at);
    *reinterpret_cast<f32x4*>(s + 4) = *reinterpret_cast<const f32x4*>(a.sin + row + at + 4);
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int slot = first + i * kGroups;
    if (slot >= slots) return;   // whole groups of lanes: their shuffles stay inside
    const int part = slot < a.heads ? 0 : slot < a.heads + a.kv_heads ? 1 : 2;
    const int head = slot - (part == 0 ? 0 : part == 1 ? a.heads : a.heads + a.kv_heads);
    u32x4 v = raw[i];
    float x[8];
    if (part < 2) {
      unpack8(v, x);
      const uint16_t* gain = a.gain[part];
      if (gain != nullptr) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += x[j] * x[j];
        sum = group_sum<kLanes>(sum);
        const float inv = 1.0f / sqrtf(sum / static_cast<float>(D) + a.eps);
        float w[8];
        unpack8(*reinterpret_cast<const u32x4*>(gain + lane * 8), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = w[j] * (x[j] * inv);
      }
      if (a.pairs > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float mine = x[j] * a.mscale;
          const float other = __shfl(mine, partner, kLanes);
          const float rotated = lane < half ? mine * c[j] - other * s[j] : other * s[j] + mine * c[j];
          x[j] = turned ? rotated : x[j];
        }
      }
      v = pack8(x);
    }
    if (part == 0) {
      const int64_t at = (token * a.heads + head) * D + lane * 8;
      if (a.wide != 0) {
        float* to = static_cast<float*>(a.queries) + at;
        *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(to + 4) = f32x4{x[4], x[5], x[6], x[7]};
      } else {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.queries) + at) = v;
      }
    } else if (page >= 0) {
      *reinterpret_cast<u32x4*>(a.pool[part - 1] + a.at.row_of(page, a.kv_heads, head, position) * D + lane * 8) = v;
    }
  }
}

constexpr float kLog2e = 1.4426950408889634f;

// A head's sink logit in the denominator: its own weight is 1, or 0 where it is -inf (or there
// is none), or NaN where it is +inf or a NaN. (Its maximum stays finite, so that it compares
// and cancels.)
struct SinkTerm {
  float top, weight;
  __device__ __forceinline__ SinkTerm(const uint16_t* sinks, int head) {
    const float logit = sinks != nullptr ? bf16_to_f32(sinks[head]) : -INFINITY;
    top = logit == -INFINITY ? -INFINITY : fminf(fmaxf(logit * kLog2e, -FLT_MAX), FLT_MAX);
    weight = __builtin_amdgcn_exp2f(logit - fmaxf(logit, -FLT_MAX));
  }
  // 1 / (total + sink) for a sum over the maximum `base` has; nothing attended gives 0.
  __device__ __forceinline__ float inverse(float base, float total) const {
    const float most = fmaxf(base, top);
    const float shift = most == -INFINITY ? 0.0f : most;
    const float shrink = __builtin_amdgcn_exp2f(base - shift);
    const float sum = __builtin_fmaf(total, shrink, weight * __builtin_amdgcn_exp2f(top - shift));
    return sum == 0.0f ? 0.0f : shrink / sum;
  }
};

// ---- attention ------------------------------------------------------------------------

struct BatchArgs {
  const void* q;            // [tokens, heads, D] bf16 or fp32
  const uint16_t* keys;     // a layer's [pages, kv_heads, page_rows, D]
  const uint16_t* values;
  const int4* tiles;        // own pieces: query rows [x, y) of sequence z, x of its w-th new token
  const uint16_t* sinks;    // [heads] or null
  uint16_t* out;            // [tokens, heads, D]
  float* partial;           // [tokens * heads, splits, D] contexts, then [tokens * heads, splits, 2]
  PageTables at;
  int heads, kv_heads, group, tokens, prefix, prefix_sequence, prefix_tiles, own_tiles;
  int prefix_splits, prefix_keys, own_splits, own_keys;   // splits of either part, keys of one
  float scale_log2;
  BatchProjectArgs fresh;   // with kFresh: the new tokens' raw rows, in place of q
};

constexpr int kWaveRows = 32, kWaves = 4, kTileRows = kWaveRows * kWaves, kTileKeys = 64, kNarrowRows = 16;

// A query row is one head of one token: of a kv head, row r is head r % group of token
// r / group.
//
// Scores are taken transposed, S^T = K Q^T on the matrix cores: a lane then holds the scores of
// one row, its state is a scalar a lane, and P^T is the B operand of O^T = V^T P^T as it stands,
// with the keys that a lane holds as the product's k index, in that order for both operands.
// V^T comes out of LDS by the transposing read.
//
// Queries of 32 bits go into the product as two bf16 parts, 16 of their 24 bits (queries of bf16
// are one), and so do the weights (split_weights_two): a weight is off by at most 2^-15 of
// itself, 1/128 of the half step that the result is rounded by. Their sum is taken before that,
// in fp32. The results' error is 0.0017 of their size, that of rounding them alone. One part of
// the weights made 0.0023 of it and, replayed, 150 us for 175 behind a document of 32,768 rows
// (128 tokens), 203 for 254 over prompts (1,828 tokens behind 4,096 rows), within 3 us where
// memory or launches bound.
//
// The maximum that the weights are taken under is raised only where a score passes it by more
// than 2^8: the sums have the room, and the rescaling of a row's context, which a growing
// maximum would ask for in nearly every tile, is rare.
constexpr float kSlack = 8.0f;

// Eight softmax weights (each zero, or a positive normal number) as two bf16 operands: the top
// half of the number cut off, less than 2^-7 of it left, and that rounded by at most 2^-8 of
// itself. Neither part is negative, and of a positive weight neither is zero: times an infinite
// value both give that infinity, as the weight itself would.
__device__ __forceinline__ void split_weights_two(const float (&p)[8], u32x4 (&parts)[2]) {
  float rest[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x0 = __float_as_uint(p[2 * j]), x1 = __float_as_uint(p[2 * j + 1]);
    parts[0][j] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
    rest[2 * j] = __builtin_amdgcn_fmed3f(p[2 * j] - __uint_as_float(x0 & 0xffff0000u), p[2 * j], 0x1p-126f);
    rest[2 * j + 1] = __builtin_amdgcn_fmed3f(p[2 * j + 1] - __uint_as_float(x1 & 0xffff0000u), p[2 * j + 1], 0x1p-126f);
  }
  parts[1] = pack8(rest);
}

// What the scheduler is told to group (sched_group_barrier's masks).
constexpr int kValu = 0x2, kMfma = 0x8, kVmemRead = 0x20, kDsRead = 0x100;

__device__ __forceinline__ u32x4 low_part(const float (&x)[8], const u32x4& high) {
  float h[8], rest[8];
  unpack8(high, h);
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i] - h[i];
  return pack8(rest);
}

// Eight consecutive values of a query, as they come (bf16, or fp32 in kParts 2) and as bf16
// operands, in kParts parts.
template <int kParts>
struct QueryEight {
  u32x4 raw[kParts];
  __device__ __forceinline__ void load(const void* q, int64_t at) {
    const u32x4* from = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(q) + at * kParts);
#pragma unroll
    for (int i = 0; i < kParts; ++i) raw[i] = from[i];
  }
  __device__ __forceinline__ void split(s16x8 (&parts)[kParts]) const {
    if constexpr (kParts == 1) {
      parts[0] = __builtin_bit_cast(s16x8, raw[0]);
    } else {
      float x[8];
      *reinterpret_cast<u32x4*>(x) = raw[0];
      *reinterpret_cast<u32x4*>(x + 4) = raw[1];
      const u32x4 high = pack8(x);
      parts[0] = __builtin_bit_cast(s16x8, high);
      parts[1] = __builtin_bit_cast(s16x8, low_part(x, high));
    }
  }
};

__device__ __forceinline__ s16x8 read_transposed(const uint16_t* first, const uint16_t* second) {
  typedef __attribute__((address_space(3))) s16x4_lds* LdsPtr;
  const s16x4_lds v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(first));
  const s16x4_lds v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(second));
  return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Raises the maximum where it has to be; the factor for what was summed under the old one.
__device__ __forceinline__ bool raise(float& top, float best, float& shrink) {
  if (__ballot(best > top + kSlack || (top == -INFINITY && best > top)) == 0) return false;
  const float next = fmaxf(top, best);
  shrink = __builtin_amdgcn_exp2f(top - (next == -INFINITY ? 0.0f : next));
  top = next;
  return true;
}

// The same from a token's raw row: eights of it kStep apart, from `at` on, normed and rotated as the
// prologue does. Its launch is spared (4 us of a step of one token a sequence); rotary pairs in
// whole kStep, so that both halves of a pair are the lane's.
template <int D, int kEights, int kStep>
struct FreshQueries {
  u32x4 raw[kEights], gain[kEights];
  f32x4 c[kEights / 2][2], s[kEights / 2][2];
  __device__ __forceinline__ void load(const BatchProjectArgs& a, int token, int head, int at) {
    const uint16_t* from = a.raw[0] + token * a.stride[0] + head * D + at;
#pragma unroll
    for (int i = 0; i < kEights; ++i) raw[i] = *reinterpret_cast<const u32x4*>(from + kStep * i);
    if (a.gain[0] != nullptr) {
#pragma unroll
      for (int i = 0; i < kEights; ++i) gain[i] = *reinterpret_cast<const u32x4*>(a.gain[0] + at + kStep * i);
    }
  }
  __device__ __forceinline__ void load_angles(const BatchProjectArgs& a, int position, int at) {
    if (a.pairs == 0) return;
    const int64_t row = min(static_cast<int64_t>(max(position, 0)), a.angle_rows - 1) * a.table_stride + at;
#pragma unroll
    for (int i = 0; i < kEights / 2; ++i) {
      const int64_t from = row + (kStep * i < a.pairs ? kStep * i : 0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        c[i][h] = *reinterpret_cast<const f32x4*>(a.cos + from + 4 * h);
        s[i][h] = *reinterpret_cast<const f32x4*>(a.sin + from + 4 * h);
      }
    }
  }
  template <int kPairs>
  __device__ __forceinline__ void rotate(float (&x)[kEights][8], float mscale) const {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float first = x[i][j] * mscale, second = x[i + kPairs][j] * mscale;
        x[i][j] = first * c[i][j / 4][j % 4] - second * s[i][j / 4][j % 4];
        x[i + kPairs][j] = first * s[i][j / 4][j % 4] + second * c[i][j / 4][j % 4];
      }
    }
  }
  // `whole`: the sum over the lanes that share the row.
  template <typename Whole>
  __device__ __forceinline__ void split(const BatchProjectArgs& a, s16x8 (&parts)[kEights][2], const Whole& whole) const {
    float x[kEights][8];
#pragma unroll
    for (int i = 0; i < kEights; ++i) unpack8(raw[i], x[i]);
    if (a.gain[0] != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kEights; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += x[i][j] * x[i][j];
      }
      const float inv = 1.0f / sqrtf(whole(sum) / static_cast<float>(D) + a.eps);
#pragma unroll
      for (int i = 0; i < kEights; ++i) {
        float w[8];
        unpack8(gain[i], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = w[j] * (x[i][j] * inv);
      }
    }
    if (a.pairs == kEights / 2 * kStep) {
      rotate<kEights / 2>(x, a.mscale);
    } else if constexpr (kEights >= 4) {
      if (a.pairs == kEights / 4 * kStep) rotate<kEights / 4>(x, a.mscale);
    }
#pragma unroll
    for (int i = 0; i < kEights; ++i) {
      const u32x4 high = pack8(x[i]);
      parts[i][0] = __builtin_bit_cast(s16x8, high);
      parts[i][1] = __builtin_bit_cast(s16x8, low_part(x[i], high));
    }
  }
};

__device__ __forceinline__ float pair_sum(float x) {   // over lanes l and l + 32
  uint32_t lower, upper;
  half_pair(__float_as_uint(x), lower, upper);
  return __uint_as_float(lower) + __uint_as_float(upper);
}
__device__ __forceinline__ float quarter_sum(float x) {   // over lanes l, l + 16, l + 32 and l + 48
  uint32_t a, b;
  row_pair(__float_as_uint(x), a, b);
  return pair_sum(__uint_as_float(a) + __uint_as_float(b));
}

// 32 rows on 32x32x16 MFMA: row = column lane % 32; of 32 keys lane half h holds the keys
// 8 i + 4 h + j, i and j below 4.
template <int D, int kParts>
struct WideRows {
  static constexpr int kSteps = D / 16, kBlocks = D / 32;
  s16x8 q[kSteps][kParts];  // Q^T as the B operand: k = 8 half + j of each 16-wide step
  f32x16 out[kBlocks];      // O^T: d = 32 b + 8 (e / 4) + 4 half + e % 4 of the column's row
  float top, total;         // the maximum (the whole row's) and the sum (this lane's keys)
  int key_at, value_at[kBlocks];
  struct Queries {
    QueryEight<kParts> of[kSteps];
    __device__ __forceinline__ Queries(const void* queries, int64_t row, int lane) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) of[s].load(queries, row * D + 8 * (lane / 32) + 16 * s);
    }
  };

  using Fresh = FreshQueries<D, kSteps, 16>;

  __device__ __forceinline__ void start(const Queries& queries, int lane) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) queries.of[s].split(q[s]);
    start(lane);
  }
  __device__ __forceinline__ void start(const Fresh& fresh, const BatchProjectArgs& a, int lane) {
    fresh.split(a, q, pair_sum);
    start(lane);
  }
  __device__ __forceinline__ void start(int lane) {
    const int column = lane % 32, half = lane / 32;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) out[b] = f32x16{};
    top = -INFINITY;
    total = 0.0f;
    // Where this lane reads: K row `column`, chunk 2 s + half; V keys 4 half + sub / 4, 4
    // values from 16 (lane / 16 % 2) + 4 (sub % 4) of each 32-wide block.
    key_at = column * D + ((half ^ turn_k(column)) * 8);
    const int sub = lane % 16;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int r = sub / 4;
      const int piece = (b * 4 + 2 * (lane / 16 % 2) + (sub % 4) / 2) ^ turn_v(r);
      value_at[b] = (4 * half + r) * D + piece * 8 + (sub % 2) * 4;
    }
  }
  // Chunks are permuted in LDS so that both operands' reads touch every bank once: K's 16
  // rows of one chunk, V's four rows of one 64-byte group.
  static __device__ __forceinline__ int turn_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
  static __device__ __forceinline__ int turn_v(int row) { return D == 128 ? (row & 3) << 2 : (row & 2) << 1; }

  // A tile of 64 keys from LDS. With `edge`, keys outside [first, last) of it or in a sixteen
  // that `absent` marks do not count. `issue(i)`, i below kSteps, asks for the next tile's
  // vectors between the products.
  template <typename Issue>
  __device__ __forceinline__ void take(const uint16_t* tile_k, const uint16_t* tile_v, float scale_log2, bool edge,
                                       int first, int last, uint32_t absent, int half, const Issue& issue) {
    f32x16 s[2] = {f32x16{}, f32x16{}};
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const s16x8 k = *reinterpret_cast<const s16x8*>(tile_k + kb * 32 * D + (key_at ^ (step * 16)));
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, k),
                                                          __builtin_bit_cast(bf16x8, q[step][part]), s[kb], 0, 0, 0);
        }
      }
      issue(step);
    }
    // The first values, read while the scores are still being multiplied.
    s16x8 v[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) v[b] = read_transposed(tile_v + value_at[b], tile_v + value_at[b] + 8 * D);
    // Keys two steps ahead of their products, a vector of the next tile beside each step's.
    __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
#pragma unroll
    for (int step = 0; step < kSteps - 2; ++step) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        __builtin_amdgcn_sched_group_barrier(kMfma, kParts, 0);
        __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kVmemRead, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMfma, 2 * kParts, 0);
    __builtin_amdgcn_sched_group_barrier(kVmemRead, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kDsRead, 2 * kBlocks, 0);
    __builtin_amdgcn_sched_group_barrier(kMfma, 2 * kParts, 0);
    if (edge) {
      // This lane's keys are 4 half and a constant each: compared with constants, since 32 keys
      // of its own were held in registers throughout the walk.
      first -= 4 * half;
      last -= 4 * half;
      asm volatile("" : "+v"(first), "+v"(last));
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const int in = (e / 16) * 32 + 8 * ((e % 16) / 4) + e % 4;
        const bool keep = in >= first && in < last && ((absent >> (in / 16)) & 1u) == 0;
        s[e / 16][e % 16] = keep ? s[e / 16][e % 16] : -INFINITY;
      }
    }
    __builtin_amdgcn_s_setprio(0);
    float best = s[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) best = fmaxf(best, s[e / 16][e % 16]);
    uint32_t lower, upper;
    half_pair(__float_as_uint(best), lower, upper);
    best = fmaxf(__uint_as_float(lower), __uint_as_float(upper)) * scale_log2;
    float shrink;
    if (raise(top, best, shrink)) {
      total *= shrink;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) out[b] *= shrink;
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int step = 0; step < 4; ++step) {   // 16 keys each
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[step / 2][(step % 2) * 8 + j], scale_log2, -base));
        sums[j % 4] += p[j];
      }
      u32x4 weights[2];
      split_weights_two(p, weights);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          out[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v[b]),
                                                           __builtin_bit_cast(bf16x8, weights[part]), out[b], 0, 0, 0);
        }
        if (step < 3) {
          const uint16_t* at = tile_v + (step + 1) * 16 * D + value_at[b];
          v[b] = read_transposed(at, at + 8 * D);
        }
      }
    }
    // A step's products beside the next one's weights (52 vector operations) and values; of the
    // first step's 44 ahead of any product (with all 52 two registers spilled).
    __builtin_amdgcn_sched_group_barrier(kValu, 44, 0);
#pragma unroll
    for (int step = 0; step < 3; ++step) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 2, 0);
        __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 0);
        __builtin_amdgcn_sched_group_barrier(kValu, 52 / kBlocks, 0);
      }
    }
    __builtin_amdgcn_sched_group_barrier(kMfma, 2 * kBlocks, 0);
    total += (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }

  // The values that were taken out of keys [low, end), for a row that sees those keys: they
  // have positive weights, so an infinity stays one and a NaN a NaN, whatever the weights are.
  template <typename ValueRow>
  __device__ __forceinline__ void put_odd(int low, int end, int half, const ValueRow& value_row) {
    for (int key = low; key < end; ++key) {
      const uint16_t* value = value_row(key);
      if (value == nullptr) continue;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = bf16_to_f32(value[b * 32 + 8 * (e / 4) + 4 * half + e % 4]);
          out[b][e] += fabsf(v) <= FLT_MAX ? 0.0f : v;
        }
      }
    }
  }

  // The row's sum, from both halves' keys.
  __device__ __forceinline__ float whole_total() const {
    uint32_t lower, upper;
    half_pair(__float_as_uint(total), lower, upper);
    return __uint_as_float(lower) + __uint_as_float(upper);
  }
};

// 16 rows on 16x16x32 MFMA: row = column lane % 16; of 32 keys the lane quarter h holds the
// keys 16 i + 4 h + j, i below 2 and j below 4.
template <int D, int kParts>
struct NarrowRows {
  static constexpr int kSteps = D / 32, kBlocks = D / 16;
  s16x8 q[kSteps][kParts];  // Q^T as the B operand: k = 8 quarter + j of each 32-wide step
  f32x4 out[kBlocks];       // O^T: d = 16 b + 4 quarter + e of the column's row
  float top, total;
  int key_at, value_at;
  struct Queries {
    QueryEight<kParts> of[kSteps];
    __device__ __forceinline__ Queries(const void* queries, int64_t row, int lane) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) of[s].load(queries, row * D + 8 * (lane / 16) + 32 * s);
    }
  };

  using Fresh = FreshQueries<D, kSteps, 32>;

  __device__ __forceinline__ void start(const Queries& queries, int lane) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) queries.of[s].split(q[s]);
    start(lane);
  }
  __device__ __forceinline__ void start(const Fresh& fresh, const BatchProjectArgs& a, int lane) {
    fresh.split(a, q, quarter_sum);
    start(lane);
  }
  __device__ __forceinline__ void start(int lane) {
    const int column = lane % 16, quarter = lane / 16;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) out[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    top = -INFINITY;
    total = 0.0f;
    // Where this lane reads: K row `column`, chunk 4 s + quarter; V key 4 quarter + column / 4,
    // 4 values from 4 (column % 4) of each 16-wide block (whose two chunks are 2 b and 2 b + 1).
    key_at = column * D + ((quarter ^ turn_k(column)) * 8);
    const int r = 4 * quarter + column / 4;
    value_at = r * D + ((column % 4 / 2) ^ turn_v(r)) * 8 + column % 2 * 4;
  }
  // Chunks are permuted in LDS so that both operands' reads touch every bank once: K's 16 rows
  // of one chunk, V's eight rows of two. (Rows 16 on are turned as the first 16.)
  static __device__ __forceinline__ int turn_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
  static __device__ __forceinline__ int turn_v(int row) { return D == 128 ? (row & 7) << 1 : (row & 6); }

  // A tile of 32 keys from LDS, as above.
  __device__ __forceinline__ void take(const uint16_t* tile_k, const uint16_t* tile_v, float scale_log2, bool edge,
                                       int first, int last, uint32_t absent, int quarter) {
    f32x4 s[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const s16x8 k = *reinterpret_cast<const s16x8*>(tile_k + kb * 16 * D + (key_at ^ (step * 32)));
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k),
                                                          __builtin_bit_cast(bf16x8, q[step][part]), s[kb], 0, 0, 0);
        }
      }
    }
    if (edge) {
      first -= 4 * quarter;
      last -= 4 * quarter;
      asm volatile("" : "+v"(first), "+v"(last));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int in = (e / 4) * 16 + e % 4;
        const bool keep = in >= first && in < last && ((absent >> (in / 16)) & 1u) == 0;
        s[e / 4][e % 4] = keep ? s[e / 4][e % 4] : -INFINITY;
      }
    }
    float best = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) best = fmaxf(best, s[e / 4][e % 4]);
    uint32_t x, y;
    row_pair(__float_as_uint(best), x, y);
    best = fmaxf(__uint_as_float(x), __uint_as_float(y));
    half_pair(__float_as_uint(best), x, y);
    best = fmaxf(__uint_as_float(x), __uint_as_float(y)) * scale_log2;
    float shrink;
    if (raise(top, best, shrink)) {
      total *= shrink;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) out[b] *= shrink;
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j / 4][j % 4], scale_log2, -base));
    total += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    u32x4 weights[2];
    split_weights_two(p, weights);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const uint16_t* at = tile_v + (value_at ^ (b * 16));
      const s16x8 v = read_transposed(at, at + 16 * D);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        out[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v),
                                                         __builtin_bit_cast(bf16x8, weights[part]), out[b], 0, 0, 0);
      }
    }
  }

  template <typename ValueRow>
  __device__ __forceinline__ void put_odd(int low, int end, int quarter, const ValueRow& value_row) {
    for (int key = low; key < end; ++key) {
      const uint16_t* value = value_row(key);
      if (value == nullptr) continue;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = bf16_to_f32(value[b * 16 + 4 * quarter + e]);
          out[b][e] += fabsf(v) <= FLT_MAX ? 0.0f : v;
        }
      }
    }
  }

  // The row's sum, from the four quarters' keys.
  __device__ __forceinline__ float whole_total() const {
    uint32_t x, y;
    row_pair(__float_as_uint(total), x, y);
    const float two = __uint_as_float(x) + __uint_as_float(y);
    half_pair(__float_as_uint(two), x, y);
    return __uint_as_float(x) + __uint_as_float(y);
  }
};

// Takes the values that are not finite out of eight; whether there were any.
__device__ __forceinline__ bool take_out_odd(u32x4& v) {
  bool found = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t word = v[j];
    const bool lo = (word & 0x7f80u) == 0x7f80u, hi = (word & 0x7f800000u) == 0x7f800000u;
    v[j] = word & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
    found = found || lo || hi;
  }
  return found;
}

// The pages of a sequence as a wave walks its rows upwards. Tiles start at multiples of 16
// rows and pages hold 16 or more, so 16 rows from a multiple of 16 lie in one page; lane l
// holds the entry of the l-th sixteen of 1,024 rows, and the ones of the next 1,024 are on
// their way before they are asked for. What is loaded is looked at where it is used, and checked
// there: with the checks beside the loads each was waited for in turn, 3 us before the first keys
// of a piece were asked for.
struct PageWalk {
  const PageTables& at;
  const int32_t* line;      // of the sequence's table, or of the first one's where there is none
  bool known;               // whether there is
  int window, now, next;

  __device__ __forceinline__ int fetch(int w) const {
    const int index = (w * 1024 + static_cast<int>(threadIdx.x) % kWave * 16) >> at.page_shift;
    return line[min(index, at.width - 1)];
  }
  __device__ __forceinline__ PageWalk(const PageTables& tables, int s, int row) : at(tables) {
    known = s >= 0 && s < at.sequences;
    line = at.tables + static_cast<int64_t>(known ? s : 0) * at.width;
    window = row / 1024;
    now = fetch(window);
    next = fetch(window + 1);
  }
  // Before rows of `row`'s window are asked for (no further than the next one's).
  __device__ __forceinline__ void reach(int row) {
    if (row / 1024 == window) return;
    window = row / 1024;
    now = next;
    next = fetch(window + 1);
  }
  // The page of the sixteen at `row` (the same in every lane), below 0 for none.
  __device__ __forceinline__ int page(int row) const {
    const int id = __builtin_amdgcn_readlane(now, row / 16 % 64);
    return known && (row >> at.page_shift) < at.width && id < at.pages ? id : -1;
  }
};

// What a workgroup does: which rows of which kv head with which keys of whose pages.
struct Piece {
  bool shared, mixed;       // mixed: rows that see different keys
  int first_row, end_row, kv_head, split, low, high, sequence;
  int token;                // own: the first row is of this new token of the sequence
  int before;               // own: a row's token t sees the keys up to before + t
};

// As far as the block's number and its tile say, so that the pages are asked for at once.
__device__ __forceinline__ void find_piece(const BatchArgs& a, Piece& p) {
  const int rows = a.tokens * a.group;
  const int pairs = a.kv_heads * a.prefix_splits;
  const int prefix_blocks = pairs * a.prefix_tiles;
  int block = blockIdx.x;
  p.shared = block < prefix_blocks;
  if (p.shared) {
    // The row tiles that read the same keys go to one XCD, one after another.
    int pair;
    if (pairs % kXcds == 0) {
      const int turn = block / kXcds;
      pair = block % kXcds + turn / a.prefix_tiles * kXcds;
      p.first_row = turn % a.prefix_tiles * kTileRows;
    } else {
      pair = block % pairs;
      p.first_row = block / pairs * kTileRows;
    }
    p.end_row = min(p.first_row + kTileRows, rows);
    p.kv_head = pair % a.kv_heads;
    p.split = pair / a.kv_heads;
    p.low = p.split * a.prefix_keys;
    p.high = min(p.low + a.prefix_keys, a.prefix);
    p.sequence = a.prefix_sequence;
    p.mixed = false;
  } else {
    block -= prefix_blocks;
    p.kv_head = block % a.kv_heads;
    block /= a.kv_heads;
    p.split = block / a.own_tiles;
    const int4 tile = a.tiles[block % a.own_tiles];
    p.first_row = min(max(tile.x, 0), rows - 1);
    p.end_row = min(min(max(tile.y, p.first_row + 1), rows), p.first_row + kTileRows);
    p.sequence = tile.z;
    p.token = tile.w;
    p.low = a.prefix + p.split * a.own_keys;
  }
}

// The keys of an own piece, by its sequence's length; whether there is anything to do.
__device__ __forceinline__ bool find_keys(const BatchArgs& a, Piece& p) {
  if (!p.shared) {
    const int first = p.first_row / a.group, last = (p.end_row - 1) / a.group;
    p.before = a.at.rows_before(p.sequence, p.token) - first;
    p.high = min(p.low + a.own_keys, p.before + last + 1);
    p.mixed = last != first;
    if (p.low >= p.high) {
      // No row of the tile reaches this split, nor is it merged; where it is the only one, its
      // rows come as zeros.
      if (a.prefix_splits + a.own_splits > 1) return false;
      p.high = p.low;
    }
  }
  if (p.sequence < 0 || p.sequence >= a.at.sequences) p.high = p.low;
  return true;
}

// The values of a sequence's row, or null for a row on no page.
template <int D>
__device__ __forceinline__ auto value_row(const BatchArgs& a, const Piece& p) {
  return [&a, &p](int key) -> const uint16_t* {
    const int page = a.at.page(p.sequence, key);
    return page < 0 ? nullptr : a.values + a.at.row_of(page, a.kv_heads, p.kv_head, key) * D;
  };
}

// What a piece leaves of row `at` (of token, head and split) for the merge.
template <int D>
__device__ __forceinline__ void store_part(const BatchArgs& a, int64_t at, int d, const f32x4& v) {
  *reinterpret_cast<f32x4*>(a.partial + at * D + d) = v;
}
template <int D>
__device__ __forceinline__ void store_state(const BatchArgs& a, int64_t at, float top, float total) {
  const int64_t splits = a.prefix_splits + a.own_splits;
  *reinterpret_cast<float2*>(a.partial + static_cast<int64_t>(a.tokens) * a.heads * splits * D + 2 * at) =
      float2{top, total};
}

// 16 bytes a lane from global memory straight to LDS: lane l's come to `to` + 16 l.
__device__ __forceinline__ void load_to_lds(const uint16_t* from, uint16_t* to) {
  typedef __attribute__((address_space(1))) const void* Global;
  typedef __attribute__((address_space(3))) void* Local;
  __builtin_amdgcn_global_load_lds((Global)from, (Local)to, 16, 0, 0);
}

// Up to 128 rows, 32 a wave: the four waves share the tiles of 64 keys, through two LDS stages;
// the next tile is on its way to the one while the other is multiplied. (A piece of a few tiles
// starts at the rate that a CU takes its 64 KB of queries and its keys from the caches, 3 us: with
// the first two tiles asked for together it was none the faster, 40.5 us for 39.9.)
template <int D, int kParts, bool kFresh>
__device__ __forceinline__ void wide_piece(const BatchArgs& a, Piece p, PageWalk& walk, uint16_t* stage0, 
                                           uint16_t* stage1, int* flags) {
  int *odd = flags, *short_rows = flags + 1;
  using Rows = WideRows<D, kParts>;
  constexpr int kChunks = D / 8;
  constexpr int kLoads = kTileKeys * kChunks / 256;   // 16-byte vectors a thread brings, each of K and V
  constexpr int kTile = kTileKeys * D;                // elements of one tile
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int column = lane % 32, half = lane / 32;
  const int row = min(p.first_row + wave * kWaveRows + column, p.end_row - 1);
  const bool live = p.first_row + wave * kWaveRows + column < p.end_row;
  const bool working = p.first_row + wave * kWaveRows < p.end_row;   // the wave
  const int token = row / a.group, head = p.kv_head * a.group + row % a.group;
  const int2 whose = p.shared ? a.at.tokens[token] : int2{0, 0};   // asked for ahead of its use
  // Up to here every row sees the keys: up to the first row's limit, or all the shared ones
  // (that a sequence stops before their end is not expected of a plan, but served: below).
  int common = p.mixed ? p.before + p.first_row / a.group + 1 : p.high;

  // Thread t's vector i is chunk t % kChunks of row (t + 256 i) / kChunks of a tile, of one
  // sixteen for the whole wave.
  const int chunk = threadIdx.x % kChunks;
  const int stage_row = threadIdx.x / kChunks;   // of vector 0
  const uint32_t from_k = (stage_row % 16) * D + (chunk ^ Rows::turn_k(stage_row)) * 8;
  const uint32_t from_v = (stage_row % 16) * D + (chunk ^ Rows::turn_v(stage_row)) * 8;
  const int sixteen = D == 128 ? 0 : __builtin_amdgcn_readfirstlane(wave / 2);   // of vector 0
  bool whole = false;    // of the tile asked for: every row there, and seen by all rows
  uint32_t absent = 0;   // its sixteens without a page
  int64_t base[kLoads];
  auto find = [&](int tile) {
    const int key0 = tile * kTileKeys;
    walk.reach(key0);
    absent = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) absent |= walk.page(key0 + 16 * i) < 0 ? 1u << i : 0u;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = key0 + 16 * (D == 128 ? i : 2 * i + sixteen);
      base[i] = a.at.row_of(max(walk.page(at), 0), a.kv_heads, p.kv_head, at) * D;
    }
    whole = absent == 0 && key0 >= p.low && key0 + kTileKeys <= min(p.high, common);
  };
  // Its i-th vectors, keys and then values (rows of any page are in the pool, counted or not).
  auto ask = [&](int i, uint16_t* stage) {
    uint16_t* to = stage + (256 * (i % kLoads) + wave * kWave) * 8;
    if (i < kLoads) {
      load_to_lds(a.keys + base[i % kLoads] + from_k, to);
    } else {
      load_to_lds(a.values + base[i % kLoads] + from_v, to + kTile);
    }
  };
  auto ask_all = [&](uint16_t* stage) {
#pragma unroll
    for (int i = 0; i < 2 * kLoads; ++i) ask(i, stage);
  };
  // Any other tile: a row outside [low, high), or of no page, comes as zeros (a zero weight
  // times what the page happens to hold could be a NaN), and so does a value that is not
  // finite: a row that does not see it would have zero times it. Those that see it get it at
  // the end.
  auto patch = [&](int tile, uint16_t* stage) {
#pragma unroll 1
    for (int i = 0; i < kLoads; ++i) {
      const int first = tile * kTileKeys + 16 * (D == 128 ? i : 2 * i + sixteen);
      const int page = walk.page(first);
      const int at = stage_row + 256 / kChunks * i;
      const int key = tile * kTileKeys + at;
      u32x4 k = u32x4{0, 0, 0, 0}, v = u32x4{0, 0, 0, 0};
      if (page >= 0 && key >= p.low && key < p.high) {
        const int64_t base = a.at.row_of(page, a.kv_heads, p.kv_head, first) * D;
        k = *reinterpret_cast<const u32x4*>(a.keys + base + from_k);
        v = *reinterpret_cast<const u32x4*>(a.values + base + from_v);
      }
      if (take_out_odd(v)) *odd = 1;
      *reinterpret_cast<u32x4*>(stage + at * D + chunk * 8) = k;
      *reinterpret_cast<u32x4*>(stage + kTile + at * D + chunk * 8) = v;
    }
  };
  // The tile asked for is in LDS, of every wave.
  auto arrive = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
    lds_barrier();
  };

  const int tiles = (p.high + kTileKeys - 1) / kTileKeys;   // past the last
  int tile = p.low / kTileKeys;
  if (threadIdx.x == 0) *odd = *short_rows = 0;
  lds_barrier();
  Rows rows;
  int limit;
  const bool known = whose.x >= 0 && whose.x < a.at.sequences;
  const auto last = [&](int length) { return !p.shared ? p.before + token : known ? length + whose.y : -1; };
  if constexpr (kFresh) {
    typename Rows::Fresh fresh;
    fresh.load(a.fresh, token, head, 8 * half);
    const int length = a.at.lengths[known ? whose.x : 0];
    find(tile);
    if (whole && tile < tiles) ask_all(stage0);
    limit = last(length) + 1;
    fresh.load_angles(a.fresh, limit - 1, 8 * half);
    rows.start(fresh, a.fresh, lane);
  } else {
    const typename Rows::Queries queries(a.q, static_cast<int64_t>(token) * a.heads + head, lane);
    find(tile);
    if (whole && tile < tiles) ask_all(stage0);
    const int length = a.at.lengths[known ? whose.x : 0];
    rows.start(queries, lane);
    limit = last(length) + 1;
  }
  if (p.shared && limit < p.high) *short_rows = 1;
  if (tile < tiles && !whole) patch(tile, stage0);
  arrive();
  if (*short_rows != 0) {
    common = 0;
    if (tile < tiles && whole) {
      patch(tile, stage0);
      lds_barrier();
    }
    whole = false;
  }
  // The stages by name, not by a turning index: the compiler then sees that what is on its way
  // to the one is not what is read from the other, and does not wait for it.
  // The next tile is asked for between the products (ahead of them, 1,828 tokens of prompts took
  // 203 us for 196, with one part of the weights), whatever it is, without a branch that they would wait at, and patched once it
  // has arrived. Behind the last it is that one again: a piece of four tiles takes up to a
  // hundredth longer.
  static_assert(Rows::kSteps == 2 * kLoads, "a vector of the next tile a step of the products");
  auto turn = [&](const uint16_t* here, uint16_t* there) {
    const bool edge = !whole;
    const uint32_t holes = absent;
    const int key0 = tile * kTileKeys;
    find(min(tile + 1, tiles - 1));
    if (working) {
      rows.take(here, here + kTile, a.scale_log2, edge, p.low - key0, min(p.high, limit) - key0, holes, half,
                [&](int i) {
                  ask(i, there);
                });
    } else {
      ask_all(there);
    }
    ++tile;
    arrive();
    if (!whole && tile < tiles) {
      patch(tile, there);
      lds_barrier();
    }
  };
  while (tile < tiles) {
    turn(stage0, stage1);
    if (tile >= tiles) break;
    turn(stage1, stage0);
  }
  if (*odd != 0) rows.put_odd(p.low, min(p.high, limit), half, value_row<D>(a, p));

  const float total = rows.whole_total();
  if (!live) return;
  const int splits = a.prefix_splits + a.own_splits;
  const int64_t at = static_cast<int64_t>(token) * a.heads + head;
  if (splits > 1) {
    const int64_t part = at * splits + (p.shared ? p.split : a.prefix_splits + p.split);
#pragma unroll
    for (int b = 0; b < Rows::kBlocks; ++b) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        store_part<D>(a, part, b * 32 + 8 * i + 4 * half,
                      f32x4{rows.out[b][4 * i], rows.out[b][4 * i + 1], rows.out[b][4 * i + 2], rows.out[b][4 * i + 3]});
      }
    }
    if (half == 0) store_state<D>(a, part, rows.top, total);
    return;
  }
  const SinkTerm sink(a.sinks, head);
  const float inverse = sink.inverse(rows.top, total);
#pragma unroll
  for (int b = 0; b < Rows::kBlocks; ++b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint2 packed;
      packed.x = pack_bf16(rows.out[b][4 * i] * inverse, rows.out[b][4 * i + 1] * inverse);
      packed.y = pack_bf16(rows.out[b][4 * i + 2] * inverse, rows.out[b][4 * i + 3] * inverse);
      *reinterpret_cast<uint2*>(a.out + at * D + b * 32 + 8 * i + 4 * half) = packed;
    }
  }
}

// The row that a token adds for a kv head, 16 bytes a lane: its key in the first D / 8 lanes, normed
// and rotated as the prologue does, its value in as many more.
template <int D>
struct NewRow {
  static constexpr int kLanes = D / 8;
  u32x4 raw, gain;
  f32x4 c[2], s[2];
  __device__ __forceinline__ void load(const BatchProjectArgs& a, int token, int head, int position, int lane) {
    const int mine = lane % kLanes, part = lane / kLanes % 2, half = a.pairs / 8;
    raw = *reinterpret_cast<const u32x4*>(a.raw[1 + part] + token * a.stride[1 + part] + head * D + mine * 8);
    if (a.gain[1] != nullptr) gain = *reinterpret_cast<const u32x4*>(a.gain[1] + mine * 8);
    if (a.pairs == 0) return;
    const int64_t from = min(static_cast<int64_t>(max(position, 0)), a.angle_rows - 1) * a.table_stride +
                         (mine < half ? mine : mine < 2 * half ? mine - half : 0) * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      c[h] = *reinterpret_cast<const f32x4*>(a.cos + from + 4 * h);
      s[h] = *reinterpret_cast<const f32x4*>(a.sin + from + 4 * h);
    }
  }
  __device__ __forceinline__ u32x4 finish(const BatchProjectArgs& a, int lane) const {
    const int mine = lane % kLanes, part = lane / kLanes % 2, half = a.pairs / 8;
    float x[8];
    unpack8(raw, x);
    if (a.gain[1] != nullptr) {
      float sum = 0.0f, w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += x[j] * x[j];
      sum = group_sum<kLanes>(sum);
      const float inv = 1.0f / sqrtf(sum / static_cast<float>(D) + a.eps);
      unpack8(gain, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = w[j] * (x[j] * inv);
    }
    if (a.pairs > 0) {
      const bool turned = mine < 2 * half;
      const int partner = mine < half ? mine + half : turned ? mine - half : mine;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float self = x[j] * a.mscale, other = __shfl(self, partner, kLanes);
        const float cj = c[j / 4][j % 4], sj = s[j / 4][j % 4];
        const float rotated = mine < half ? self * cj - other * sj : other * sj + self * cj;
        x[j] = turned ? rotated : x[j];
      }
    }
    return part == 0 ? pack8(x) : raw;
  }
};

// A wave's walk over a piece with up to 16 rows: every `stride`-th tile of 32 keys from `tile`
// on, through an LDS buffer of its own, without a barrier. Leaves the rows' state in `rows`.
template <int D, int kParts, bool kStream, bool kFresh>
__device__ __forceinline__ void narrow_walk(const BatchArgs& a, Piece& p, PageWalk& walk, NarrowRows<D, kParts>& rows,
                                            int tile, int stride, uint16_t* tile_k) {
  using Rows = NarrowRows<D, kParts>;
  constexpr int kKeys = 32;
  constexpr int kChunks = D / 8, kRowsALoad = kWave / kChunks;   // 4 or 8
  constexpr int kLoads = kKeys / kRowsALoad;                     // 16-byte vectors a lane stages, each of K and V
  uint16_t* tile_v = tile_k + kKeys * D;
  const int lane = threadIdx.x % kWave, column = lane % 16, quarter = lane / 16;
  const int row = min(p.first_row + column, p.end_row - 1);
  const int token = row / a.group, head = p.kv_head * a.group + row % a.group;
  const int2 whose = p.shared ? a.at.tokens[token] : int2{0, 0};

  const int first_tile = tile, tiles = (p.high + kKeys - 1) / kKeys;   // past the last
  const int chunk = lane % kChunks, stage_row = lane / kChunks;
  const uint32_t offset = stage_row * D + chunk * 8;
  u32x4 stage_k[kLoads], stage_v[kLoads];
  bool whole = false;
  uint32_t absent = 0;
  const auto load = [](const uint16_t* from) {
    return kStream ? load_nt(reinterpret_cast<const u32x4*>(from)) : *reinterpret_cast<const u32x4*>(from);
  };
  auto load_tile = [&](int t) {
    const int key0 = t * kKeys;
    walk.reach(key0);
    absent = 0;
    int64_t first[kKeys / 16];
#pragma unroll
    for (int i = 0; i < kKeys / 16; ++i) {
      const int page = walk.page(key0 + 16 * i);
      absent |= page < 0 ? 1u << i : 0u;
      first[i] = a.at.row_of(max(page, 0), a.kv_heads, p.kv_head, key0 + 16 * i) * D;
    }
    whole = __builtin_amdgcn_readfirstlane(absent == 0 && key0 >= p.low && key0 + kKeys <= p.high ? 1 : 0) != 0;
    // Every row, counted or not (a row of any page is in the pool): without branches the queries,
    // asked for before, are waited for alone.
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int in = i * kRowsALoad;   // of the tile, the load's first row
      stage_k[i] = load(a.keys + first[in / 16] + (in % 16) * D + offset);
      stage_v[i] = load(a.values + first[in / 16] + (in % 16) * D + offset);
    }
  };

  bool odd = false;   // a value of this wave's keys was taken out, by this lane
  int limit;
  u32x4 new_row;   // the new token's key (lanes below D / 8) and value (as many more), and where it is
  int new_at = -1;
  if constexpr (kFresh) {
    // Own rows are of one token, whose position is known: all it needs is asked for ahead of the keys.
    typename Rows::Fresh fresh;
    NewRow<D> added;
    fresh.load(a.fresh, token, head, 8 * quarter);
    const bool shared = !kStream && p.shared;
    if (!shared) {
      limit = p.before + token + 1;
      const int position = __builtin_amdgcn_readfirstlane(limit - 1);
      fresh.load_angles(a.fresh, position, 8 * quarter);
      if (position >= p.low && position < p.high) {
        new_at = position;
        added.load(a.fresh, __builtin_amdgcn_readfirstlane(token), p.kv_head, position, lane);
      }
    }
    load_tile(tile);
    if (shared) {
      limit = a.at.before(whose) + 1;
      fresh.load_angles(a.fresh, limit - 1, 8 * quarter);
    }
    rows.start(fresh, a.fresh, lane);
    if (new_at >= 0) new_row = added.finish(a.fresh, lane);
  } else {
    const typename Rows::Queries queries(a.q, static_cast<int64_t>(token) * a.heads + head, lane);
    load_tile(tile);
    rows.start(queries, lane);
    limit = (p.shared ? a.at.before(whose) : p.before + token) + 1;
  }
  if (p.shared && __ballot(limit < p.high) != 0) p.mixed = true;   // the same rows in every wave
  while (tile < tiles) {
    const int key0 = tile * kKeys;
    const bool edge = __builtin_amdgcn_readfirstlane(p.mixed || !whole ? 1 : 0) != 0;
    const uint32_t holes = absent;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int in = i * kRowsALoad, key = key0 + in + stage_row;
        const bool there = ((absent >> (in / 16)) & 1u) == 0 && key >= p.low && key < p.high;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          stage_k[i][j] = there ? stage_k[i][j] : 0u;
          stage_v[i][j] = there ? stage_v[i][j] : 0u;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * kRowsALoad + stage_row;
      if (p.mixed) odd = take_out_odd(stage_v[i]) || odd;
      *reinterpret_cast<u32x4*>(tile_k + at * D + (chunk ^ Rows::turn_k(at)) * 8) = stage_k[i];
      *reinterpret_cast<u32x4*>(tile_v + at * D + (chunk ^ Rows::turn_v(at)) * 8) = stage_v[i];
    }
    // The new row, over what its place in the pool held: this wave is its only reader here.
    if (kFresh && new_at >= 0 && tile == new_at / kKeys) {
      const int at = new_at % kKeys, mine = lane % kChunks, part = lane / kChunks;
      const int turn = part == 0 ? Rows::turn_k(at) : Rows::turn_v(at);
      const int page = walk.page(new_at);
      if (page >= 0 && part < 2) {
        *reinterpret_cast<u32x4*>((part == 0 ? tile_k : tile_v) + at * D + (mine ^ turn) * 8) = new_row;
        const int64_t to = a.at.row_of(page, a.kv_heads, p.kv_head, new_at) * D + mine * 8;
        *reinterpret_cast<u32x4*>(a.fresh.pool[part] + to) = new_row;
      }
    }
    const int following = tile + stride;
    if (following < tiles) load_tile(following);
    // The wave's lanes read what the others stored: LDS takes a wave's operations in order.
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
    rows.take(tile_k, tile_v, a.scale_log2, edge, p.low - key0, min(p.high, limit) - key0, holes, quarter);
    tile = following;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  }
  // A wave that took any out puts back its own tiles'.
  if (__ballot(odd) != 0) {
    const auto any = value_row<D>(a, p);
    rows.put_odd(max(p.low, first_tile * kKeys), min(p.high, limit), quarter, [&](int key) {
      return (key / kKeys - first_tile) % stride == 0 ? any(key) : nullptr;
    });
  }
}

// Four values of a row at `d`: for the merge, or the result where there is one piece a row.
template <int D>
__device__ __forceinline__ void store_four(const BatchArgs& a, const Piece& p, int row, int d, float top, float total,
                                           const f32x4& v) {
  const int splits = a.prefix_splits + a.own_splits;
  const int head = p.kv_head * a.group + row % a.group;
  const int64_t at = static_cast<int64_t>(row / a.group) * a.heads + head;
  if (splits > 1) {
    const int64_t part = at * splits + (p.shared ? p.split : a.prefix_splits + p.split);
    store_part<D>(a, part, d, v);
    if (d == 0) store_state<D>(a, part, top, total);
    return;
  }
  const SinkTerm sink(a.sinks, head);
  const float inverse = sink.inverse(top, total);
  uint2 packed;
  packed.x = pack_bf16(v[0] * inverse, v[1] * inverse);
  packed.y = pack_bf16(v[2] * inverse, v[3] * inverse);
  *reinterpret_cast<uint2*>(a.out + at * D + d) = packed;
}

// Up to 16 rows: the four waves hold the same rows, take every fourth tile each and merge at the
// end.
template <int D, int kParts, bool kFresh>
__device__ __forceinline__ void narrow_piece(const BatchArgs& a, Piece p, PageWalk& walk, uint16_t* stage0,
                                             uint16_t* stage1) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int column = lane % 16, quarter = lane / 16;
  NarrowRows<D, kParts> rows;
  narrow_walk<D, kParts, false, kFresh>(a, p, walk, rows, p.low / 32 + wave, kWaves,
                         (wave < 2 ? stage0 : stage1) + wave % 2 * 2 * 32 * D);

  // The waves' states and contexts meet in LDS: row c's context of wave w at [w][c] of the one
  // stage, its top and sum in the other.
  const float total = rows.whole_total();
  const int count = p.end_row - p.first_row;
  float* parts = reinterpret_cast<float*>(stage0);
  float2* states = reinterpret_cast<float2*>(stage1);
  lds_barrier();
  if (column < count) {
#pragma unroll
    for (int b = 0; b < D / 16; ++b) {
      *reinterpret_cast<f32x4*>(parts + (wave * kNarrowRows + column) * D + b * 16 + 4 * quarter) = rows.out[b];
    }
    if (quarter == 0) states[wave * kNarrowRows + column] = float2{rows.top, total};
  }
  lds_barrier();
  for (int item = threadIdx.x; item < count * (D / 4); item += 256) {
    const int r = item / (D / 4), d = item % (D / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, states[w * kNarrowRows + r].x);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 state = states[w * kNarrowRows + r];
      const float factor = __builtin_amdgcn_exp2f(state.x - base);
      const f32x4 part = *reinterpret_cast<const f32x4*>(parts + (w * kNarrowRows + r) * D + d);
      sum = __builtin_fmaf(state.y, factor, sum);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(part[i], factor, v[i]);
    }
    store_four<D>(a, p, p.first_row + r, d, top, sum, v);
  }
}

template <int D, int kParts, bool kFresh = false>
__global__ __launch_bounds__(256, 2) void attention_batch_kernel(BatchArgs a) {
  // K and V of a tile each; a narrow piece's waves have half of one each, and its contexts of
  // four waves fill the first.
  __shared__ __attribute__((aligned(16))) uint16_t stage0[2 * kTileKeys * D], stage1[2 * kTileKeys * D];
  static_assert(sizeof(stage0) == kWaves * kNarrowRows * D * sizeof(float) && sizeof(stage0) == 2 * 2 * 32 * D * 2,
                "a stage holds what a narrow piece puts there");
  __shared__ int flags[2];   // a value was taken out; a row ends before the shared ones do
  Piece p;
  find_piece(a, p);
  PageWalk walk(a.at, p.sequence, p.low);
  if (!find_keys(a, p)) return;
  if (p.end_row - p.first_row <= kNarrowRows) {
    narrow_piece<D, kParts, kFresh>(a, p, walk, stage0, stage1);
  } else {
    wide_piece<D, kParts, kFresh>(a, p, walk, stage0, stage1, flags);
  }
}

// Own pieces alone, a wave each, so that none waits for another: 24 sequences of up to 16,000
// rows take 92 us, with the four waves of a workgroup on one piece 115. Bound by memory, at 5.5
// to 6.2 TB/s; what is read is past the caches' size, so it goes by them (24 of 4,776 rows: 103
// -> 91 us; where it fits, it may be there still, and a nontemporal load costs a tenth). Pieces
// of a tile of more than 16 rows take them 16 at a time.
template <int D, int kParts, bool kFresh = false>
__global__ __launch_bounds__(64, 2) void attention_own_kernel(BatchArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t tile[2 * 32 * D];
  Piece p;
  find_piece(a, p);
  const int first = p.first_row, end = p.end_row, token = p.token;
  for (int row = first; row < end; row += kNarrowRows) {
    p.first_row = row;
    p.end_row = min(row + kNarrowRows, end);
    PageWalk walk(a.at, p.sequence, p.low);
    p.token = token + row / a.group - first / a.group;
    if (!find_keys(a, p)) continue;
    const int column = threadIdx.x % 16, quarter = threadIdx.x / 16;
    NarrowRows<D, kParts> rows;
    narrow_walk<D, kParts, true, kFresh>(a, p, walk, rows, p.low / 32, 1, tile);
    const float total = rows.whole_total();
    if (column >= p.end_row - p.first_row) continue;
#pragma unroll
    for (int b = 0; b < D / 16; ++b) {
      store_four<D>(a, p, p.first_row + column, b * 16 + 4 * quarter, rows.top, total, rows.out[b]);
    }
  }
}

// Merges a row's pieces. A piece that the row does not reach was not written and is not read.
// A row that attends nothing comes as zeros.
//
// D / 4 lanes hold a piece's context; kGroups of them take every kGroups-th piece of a row and
// meet in LDS, so that a few rows of many pieces (16 tokens of 32 heads, 33 pieces: 9.1 us with
// one group) are not a chain of loads on a few CUs.
template <int D, int kGroups>
__global__ __launch_bounds__(256) void attention_batch_merge_kernel(BatchArgs a) {
  constexpr int kLanes = D / 4, kRows = 256 / kLanes / kGroups;   // of one piece; rows of a workgroup
  constexpr int kAtOnce = 4;
  __shared__ float2 group_state[kGroups > 1 ? kRows * kGroups : 1];
  __shared__ f32x4 group_sum[kGroups > 1 ? kRows * kGroups * kLanes : 1];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes % kGroups, in = threadIdx.x / kLanes / kGroups;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + in;   // token * heads + head
  const int64_t rows = static_cast<int64_t>(a.tokens) * a.heads;
  const int64_t row_at = row < rows ? row : rows - 1;
  const int64_t token = row_at / a.heads;
  const int own = a.at.before(a.at.tokens[token]) + 1 - a.prefix;
  const int splits = a.prefix_splits + a.own_splits;
  const int count = a.prefix_splits + min(own <= 0 ? 0 : (own + a.own_keys - 1) / a.own_keys, a.own_splits);
  const float2* states = reinterpret_cast<const float2*>(a.partial + rows * splits * D) + row_at * splits;
  const float* parts = a.partial + row_at * splits * D + lane * 4;
  const int head = static_cast<int>(row_at - token * a.heads);
  const SinkTerm sink(a.sinks, head);
  float top = -INFINITY, total = 0.0f;
  f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int first = group; first < count; first += kAtOnce * kGroups) {
    float2 state[kAtOnce];
    f32x4 part[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int s = min(first + i * kGroups, count - 1);
      state[i] = states[s];
      part[i] = *reinterpret_cast<const f32x4*>(parts + static_cast<int64_t>(s) * D);
    }
    float next = top;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) next = fmaxf(next, state[i].x);
    const float base = next == -INFINITY ? 0.0f : next;
    const float shrink = __builtin_amdgcn_exp2f(top - base);
    total *= shrink;
    sum *= shrink;
    top = next;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (first + i * kGroups < count) {
        const float factor = __builtin_amdgcn_exp2f(state[i].x - base);
        total = __builtin_fmaf(state[i].y, factor, total);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = __builtin_fmaf(part[i][j], factor, sum[j]);
      }
    }
  }
  if constexpr (kGroups > 1) {
    if (lane == 0) group_state[in * kGroups + group] = float2{top, total};
    group_sum[(in * kGroups + group) * kLanes + lane] = sum;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) top = fmaxf(top, group_state[in * kGroups + g].x);
    const float base = top == -INFINITY ? 0.0f : top;
    total = 0.0f;
    sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float2 state = group_state[in * kGroups + g];
      const f32x4 part = group_sum[(in * kGroups + g) * kLanes + lane];
      const float factor = __builtin_amdgcn_exp2f(state.x - base);
      total = __builtin_fmaf(state.y, factor, total);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = __builtin_fmaf(part[j], factor, sum[j]);
    }
  }
  if (row >= rows) return;
  const float inverse = sink.inverse(top, total);
  uint2 packed;
  packed.x = pack_bf16(sum[0] * inverse, sum[1] * inverse);
  packed.y = pack_bf16(sum[2] * inverse, sum[3] * inverse);
  *reinterpret_cast<uint2*>(a.out + row * D + lane * 4) = packed;
}

template <int D>
void launch_merge(const BatchArgs& a, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.tokens) * a.heads;
  const auto launch = [&](auto kernel, int groups) {
    const int64_t of_one = 256 / (D / 4) / groups;
    kernel<<<dim3(static_cast<unsigned>((rows + of_one - 1) / of_one)), 256, 0, stream>>>(a);
  };
  // A group has four pieces under way at once.
  const int splits = a.prefix_splits + a.own_splits;
  if (splits <= 4) {
    launch(attention_batch_merge_kernel<D, 1>, 1);
  } else if (splits <= 20) {
    launch(attention_batch_merge_kernel<D, 4>, 4);
  } else {
    launch(attention_batch_merge_kernel<D, 256 / (D / 4)>, 256 / (D / 4));
  }
}

// How the keys are cut: the shared rows and the sequences' own each into pieces of a multiple
// of 64 keys. A wide piece leaves 128 rows of context for the merge and takes a while to start; a
// narrow one leaves a few rows and is short, so that sequences of different lengths fill the card
// evenly.
struct Plan {
  int64_t prefix, prefix_tiles, prefix_splits, prefix_keys, own_splits, own_keys;
  bool own_alone;   // own pieces only, a wave each
};

constexpr int64_t kSlots = 512, kNarrowBlocks = 2048, kNarrowKeys = 512, kMaxSplits = 64;
constexpr int64_t kOwnKeys = 256, kOwnPieces = 2048;

// Most pieces of a row: the merge reads them all again, up to 64 at once, but a few kv heads of a
// few sequences have to fill the card (two of one sequence of 400,000 rows: 64 pieces each 251 us, 512 86).
int64_t most_splits(int64_t blocks) {
  const int64_t fill = 2 * kSlots / (blocks < 1 ? 1 : blocks);
  return fill > kMaxSplits ? fill : kMaxSplits;
}

// `splits` pieces of whole tiles of 64 keys for each of `blocks` workgroups, or as many as those
// leave, and the keys of one.
int64_t cut(int64_t blocks, int64_t keys, int64_t splits, int64_t& each) {
  const int64_t most = most_splits(blocks);
  splits = splits < 1 ? 1 : splits > most ? most : splits;
  const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys;
  const int64_t of_one = (tiles + splits - 1) / splits;
  each = of_one * kTileKeys;
  return (tiles + of_one - 1) / of_one;
}

// What wide pieces were measured to take, in us: one on a CU waits for its keys, two share the
// matrix cores and the start's loads. That was with one part of the weights; with two a tile takes
// 1.5 and 2.15, and 2.4 and 3.35. Cut by those, it comes out even (replayed): three prompts of 300
// tokens behind 512 rows 54.8 -> 49.6, nine of 120 behind 2,048 124 -> 117, but 40 of 20 behind
// 8,192 216 -> 230 and 128 tokens behind 32,768 181 -> 187, so they stay.
struct WideCost {
  double start, tile, start_both, tile_both, tile_bytes;
};
constexpr WideCost kCost64{4.0, 1.2, 5.0, 1.6, 16384.0}, kCost128{5.5, 2.0, 7.5, 2.57, 32768.0};
constexpr double kBytesPerUs = 6e6, kLaunchUs = 4.0;

// `count` pieces of `tiles` tiles, of which `row_tiles` read the same keys. (Alone, the start takes
// less where there are fewer to share the caches' rate: 256 pieces of four tiles 20.0 us, 128 and 64
// of them 18.0, the launch included; 0.65 and 0.7 are fitted to such replays.)
double wide_us(const WideCost& c, int64_t count, int64_t tiles, int64_t row_tiles) {
  const auto round = [&](int64_t n) {
    if (n <= 0) return 0.0;
    const bool both = n > kSlots / 2;
    const double memory = n * c.tile_bytes / row_tiles / kBytesPerUs, tile = both ? c.tile_both : c.tile;
    return (both ? c.start_both : c.start * (0.65 + 0.7 * n / kSlots)) + tiles * (memory > tile ? memory : tile);
  };
  return count / kSlots * round(kSlots) + round(count % kSlots);
}

// What runs beside wide pieces and is merged with them: whether there is anything, how many pieces
// start after them, what one takes, and what all of them take where they have the card to
// themselves. `fresh`: one token a sequence, whose prologue is spared where all pieces run at once.
struct Beside {
  bool any, fresh;
  int64_t blocks;
  double pieces, us, all_us;
};

// Wide pieces of `keys` keys, of which the part `filled` is there, for each of `blocks` workgroups:
// as many as are expected to be done first, with their partial results (`row_us` for
// a piece of every row) and the merge's launch, and what is beside them and finds no slot
// meanwhile. Against as many as fill the slots, of 256 keys or more (replayed): 128 tokens behind
// 32,768 rows with up to 1,024 own each 202 -> 181 us, 128 behind 4,096 105 -> 81, 96 behind 4,000
// 53 -> 50, 100 of two kv heads behind 8,192 46 -> 42, nine prompts of up to 100 tokens behind
// 2,048 88 -> 68.
int64_t wide_splits(int64_t blocks, int64_t keys, double filled, const WideCost& c, int64_t row_tiles, double row_us,
                    const Beside& beside, int64_t& each) {
  const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys;
  int64_t best = 1;
  double least = 0.0;
  for (int64_t splits = 1; splits <= most_splits(blocks) && splits <= tiles; ++splits) {
    const int64_t of_one = (tiles + splits - 1) / splits;
    if ((tiles + of_one - 1) / of_one != splits) continue;   // as another one
    // Of pieces that are not all there, as many whole ones as they amount to.
    const int64_t count = static_cast<int64_t>(blocks * splits * filled) + (filled < 1.0 ? 1 : 0);
    double us = wide_us(c, count, of_one, row_tiles);
    if (beside.pieces > 0) {
      // Beside the others one takes a quarter longer, and with every slot taken the last wait: 0.8,
      // 1.05 and 15 of 16 are fitted to the replays above together, not measured apart.
      const double meanwhile = count < kSlots ? 0.8 * (kSlots - count) * us / beside.us : 0.0;
      if (count > kSlots / 16 * 15) us *= 1.05;
      if (meanwhile < beside.pieces) us += (beside.pieces - meanwhile) / beside.pieces * beside.all_us;
      if (beside.fresh && count + beside.blocks > kSlots) us += kLaunchUs;
    }
    if (splits > 1 || beside.any) us += kLaunchUs + splits * row_us;
    if (splits == 1 || us < least) {
      least = us;
      best = splits;
    }
  }
  return cut(blocks, keys, best, each);
}

// Narrow pieces of `keys` keys, of which the part `filled` is there, for each of `blocks`
// workgroups, and the keys of one; `taken` workgroups start before them.
int64_t narrow_splits(int64_t blocks, int64_t keys, double filled, int64_t taken, int64_t& each) {
  if (filled < 0.5) blocks = static_cast<int64_t>(blocks * 2.0 * filled) + 1;
  const auto fill = [&](int64_t target, int64_t least) {
    const int64_t splits = (target + blocks - 1) / blocks, by_keys = keys / least;
    return splits < by_keys ? splits : by_keys;
  };
  // Short ones where slots that are left would be empty, else longer (384 beside 312 others: 45.0
  // us in two pieces each, 42.5 in one).
  const int64_t splits = fill(kNarrowBlocks, kNarrowKeys);
  const int64_t slots = taken >= kSlots ? kSlots : taken > kSlots / 2 ? kSlots / 2 : kSlots - taken;
  return cut(blocks, keys, blocks * splits < slots ? fill(slots, kNarrowKeys / 4) : splits, each);
}

// `own_total`: the own rows of every tile's sequence together, or 0 where they are not known and
// taken to be spread up to own_rows (in prompts: to be as many).
Plan plan_for(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t prefix, int64_t own_rows,
              int64_t own_total, int64_t own_tiles) {
  Plan p{};
  const int64_t rows = tokens * (heads / kv_heads);
  const int64_t shared_tiles = (rows + kTileRows - 1) / kTileRows;
  // Where the sequences' own tiles are nearly as full as shared ones (prompts), each walks the
  // shared rows as well: as many products, and nothing to merge. At 1.06 as many tiles, nine
  // prompts of 120 tokens, that is even (behind 2,048 rows 116 us shared, 117 walked, behind 8,192
  // 307 and 309), at 1.24, of 100, it is not (98 and 110, 233 and 285), nor mostly at 1.2, of 50 (69
  // and 62, 134 and 156).
  // So do a few sequences of a few rows: one piece a row, and again nothing to merge (2 of 229
  // rows: 16 -> 13.4 us a step).
  const bool few = prefix + own_rows <= kNarrowKeys && kv_heads * own_tiles <= kSlots;
  p.prefix = own_tiles * 8 <= shared_tiles * 9 || few ? 0 : prefix;
  if (own_total > 0) own_total += (prefix - p.prefix) * own_tiles;
  own_rows += prefix - p.prefix;
  p.prefix_tiles = p.prefix > 0 ? shared_tiles : 0;
  p.prefix_keys = p.own_keys = kTileKeys;
  const int64_t own_blocks = kv_heads * own_tiles;
  const bool narrow = rows <= kNarrowRows * own_tiles, any_own = own_rows > 0 && own_tiles > 0;
  const WideCost& cost = head_dim == 64 ? kCost64 : kCost128;
  const double whole = static_cast<double>(own_rows) * own_tiles;
  const double total = own_total <= 0 ? (narrow ? whole / 2.0 : whole) : own_total < whole ? own_total : whole;
  const double filled = whole > 0.0 ? total / whole : 1.0;
  // A piece's contexts of all rows, written and read.
  const double row_us = static_cast<double>(tokens) * heads * head_dim * 8.0 / kBytesPerUs;
  if (p.prefix > 0 && shared_tiles > 0) {
    const int64_t blocks = kv_heads * shared_tiles;
    if (rows <= kNarrowRows) {
      p.prefix_splits = narrow_splits(blocks, p.prefix, 1.0, 0, p.prefix_keys);
    } else {
      Beside own{any_own, false, own_blocks, 0.0, 1.0, 0.0};
      if (any_own && narrow) {
        const int64_t of_one = own_rows < kNarrowKeys ? own_rows : kNarrowKeys;
        own.fresh = own_tiles == tokens && heads <= kNarrowRows * kv_heads;
        own.pieces = own_blocks * (filled * own_rows / kNarrowKeys + 0.5);
        if (own.pieces < own_blocks) own.pieces = static_cast<double>(own_blocks);
        own.us = 3.0 + 0.011 * of_one;   // 128 pieces, launch included: 5.8 us of 128 keys, 7.0 of 192
      } else if (any_own) {
        own.pieces = static_cast<double>(own_blocks);
        own.us = cost.start + (own_rows + kTileKeys - 1) / kTileKeys * cost.tile;
      }
      own.all_us = own.pieces / kSlots * own.us;
      const double bytes = narrow ? kv_heads * total * head_dim * 4.0 : 0.0;
      if (own.all_us < bytes / kBytesPerUs) own.all_us = bytes / kBytesPerUs;
      p.prefix_splits = wide_splits(blocks, p.prefix, 1.0, cost, shared_tiles, row_us, own, p.prefix_keys);
    }
  }
  if (!any_own) return p;
  p.own_alone = p.prefix == 0 && narrow && 2.0 * kv_heads * total >= kOwnPieces * kOwnKeys;
  if (p.own_alone) {
    // All at once where that is possible: a wave that has done its piece leaves the others more
    // of the memory's rate, until the last ones cannot take it. Short ones where a few sequences
    // have most of the rows (64 sequences of up to 567, but one of 4,000, of 3 tokens: 92 -> 48 us;
    // eight of up to 8,000, of 6 tokens, 39 -> 43).
    const int64_t even = filled < 0.5 ? static_cast<int64_t>(own_blocks * 2.0 * filled) + 1 : own_blocks;
    const int64_t fill = (kOwnPieces + even - 1) / even;
    const int64_t most = own_rows / kOwnKeys, least = own_rows / (4 * kOwnKeys);
    p.own_splits = cut(own_blocks, own_rows, fill > most ? most : fill < least ? least : fill, p.own_keys);
  } else if (narrow) {
    p.own_splits = narrow_splits(own_blocks, own_rows, filled, kv_heads * p.prefix_tiles * p.prefix_splits, p.own_keys);
  } else {
    p.own_splits = wide_splits(own_blocks, own_rows, filled, cost, own_tiles, row_us,
                               Beside{p.prefix > 0, false, 0, 0.0, 1.0, 0.0}, p.own_keys);
  }
  return p;
}

bool geometry_served(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t prefix,
                     int64_t own_rows, int64_t own_tiles) {
  constexpr int64_t kMaxRows = int64_t{1} << 30;
  return (head_dim == 64 || head_dim == 128) && kv_heads > 0 && heads > 0 && heads <= 4096 && heads % kv_heads == 0 &&
         tokens >= 0 && tokens * heads < kMaxRows && prefix >= 0 && prefix < kMaxRows && own_rows >= 0 &&
         own_rows < kMaxRows && own_tiles >= 0 && own_tiles < kMaxRows;
}

int64_t query_bytes(int64_t tokens, int64_t heads, int64_t head_dim) {
  return (tokens * heads * head_dim * static_cast<int64_t>(sizeof(float)) + 255) / 256 * 256;
}

int page_shift_of(int64_t page_rows) {
  for (int shift = 4; shift <= 8; ++shift) {
    if (page_rows == int64_t{1} << shift) return shift;
  }
  return -1;
}

// Whether the attention projects a step's rows itself, without the prologue's launch: one token a
// sequence, of up to 16 rows, with pairs that a lane holds both halves of, where the pieces run at
// once (one a sequence and kv head counted: of more some are past its rows). Each projects its
// queries, which costs it a microsecond or two: 33 sequences of 64 heads 28.1 -> 23.4 us, but 96
// of 32 with 696 pieces 43.7 -> 44.6. Waves alone have several rounds and gain all the same (24
// sequences of up to 16,000 rows: 94.5 -> 93.1).
bool takes_fresh(const omnia_attention_batch_step_t& s) {
  if (s.one_token_each == 0 || s.tokens <= 0 || s.own_tiles != s.tokens || s.rotary_pairs % 32 != 0 ||
      !geometry_served(s.tokens, s.heads, s.kv_heads, s.head_dim, s.prefix, s.own_rows, s.own_tiles) ||
      s.heads > kNarrowRows * s.kv_heads) {
    return false;
  }
  const Plan p = plan_for(s.tokens, s.heads, s.kv_heads, s.head_dim, s.prefix, s.own_rows, s.own_total, s.own_tiles);
  return p.own_alone || s.kv_heads * (p.prefix_tiles * p.prefix_splits + s.own_tiles) <= kSlots;
}

// Whether a step's prologue is refused.
int32_t project_refused(const omnia_attention_batch_step_t& s, const void* queries) {
  OMNIA_REQUIRE(geometry_served(s.tokens, s.heads, s.kv_heads, s.head_dim, 0, 0, 0), "attention_batch_project: bad geometry");
  OMNIA_REQUIRE(s.rotary_pairs >= 0 && s.rotary_pairs % 8 == 0 && 2 * s.rotary_pairs <= s.head_dim,
                "attention_batch_project: rotary_pairs must be a multiple of 8 within the head");
  OMNIA_REQUIRE(page_shift_of(s.page_rows) > 0, "attention_batch_project: page_rows must be 16, 32, 64, 128 or 256");
  OMNIA_REQUIRE(s.pages > 0 && s.pages < (int64_t{1} << 31) && s.sequences > 0 && s.sequences < (int64_t{1} << 31) &&
                    s.width > 0 && s.width < (int64_t{1} << 31) / s.page_rows,
                "attention_batch_project: bad tables");
  if (s.tokens == 0) return 0;
  OMNIA_REQUIRE(s.raw_queries && s.raw_keys && s.raw_values && queries && s.keys && s.values && s.tables && s.lengths &&
                    s.token_map,
                "attention_batch_project: null pointer");
  OMNIA_REQUIRE(aligned16(s.raw_queries) && aligned16(s.raw_keys) && aligned16(s.raw_values) && aligned16(queries) &&
                    aligned16(s.keys) && aligned16(s.values) && aligned16(s.query_weight) && aligned16(s.key_weight),
                "attention_batch_project: pointers must be 16-byte aligned");
  OMNIA_REQUIRE(s.query_stride % 8 == 0 && s.key_stride % 8 == 0 && s.value_stride % 8 == 0 &&
                    s.query_stride >= s.heads * s.head_dim && s.key_stride >= s.kv_heads * s.head_dim &&
                    s.value_stride >= s.kv_heads * s.head_dim,
                "attention_batch_project: row strides must be multiples of 8 covering the heads");
  OMNIA_REQUIRE(s.rotary_pairs == 0 || (s.cos_rows && s.sin_rows && aligned16(s.cos_rows) && aligned16(s.sin_rows) &&
                                        s.table_stride % 4 == 0 && s.table_stride >= s.rotary_pairs && s.angle_rows > 0),
                "attention_batch_project: angle rows must be 16-byte aligned and cover the pairs");
  return 0;
}

BatchProjectArgs project_args(const omnia_attention_batch_step_t& s, void* queries, int32_t wide) {
  return BatchProjectArgs{{s.raw_queries, s.raw_keys, s.raw_values}, {s.query_stride, s.key_stride, s.value_stride},
                          {s.query_weight, s.key_weight}, s.cos_rows, s.sin_rows, s.table_stride, s.angle_rows, queries,
                          {s.keys, s.values},
                          {s.tables, s.lengths, reinterpret_cast<const int2*>(s.token_map),
                           static_cast<int>(s.sequences), static_cast<int>(s.width), static_cast<int>(s.pages),
                           page_shift_of(s.page_rows)},
                          static_cast<int>(s.heads), static_cast<int>(s.kv_heads), static_cast<int>(s.tokens),
                          static_cast<int>(s.rotary_pairs), wide != 0 ? 1 : 0, s.mscale, s.eps};
}

int32_t project(const omnia_attention_batch_step_t& s, void* queries, int32_t wide, hipStream_t stream) {
  int32_t rc = project_refused(s, queries);
  if (rc != 0 || s.tokens == 0) return rc;
  rc = check_device(stream);
  if (rc != 0) return rc;
  const BatchProjectArgs a = project_args(s, queries, wide);
  // Up to four heads in turn, the same number in every workgroup of a token (7,133 tokens of 80
  // heads of 64, 32 at once: three in turn 30.6 us, four 31.8; 4,000 of 12 heads of 128, 16 at
  // once: one 9.9, four 13.6). Below 1,024 tokens one is the faster (900 of 80: 9.0 for 9.3).
  const int64_t at_once = 256 / (s.head_dim / 8), rounds = (s.heads + 2 * s.kv_heads + at_once - 1) / at_once;
  const int64_t parts = s.tokens < 1024 ? rounds : (rounds + 3) / 4;   // at most 768
  const dim3 grid(static_cast<unsigned>(s.tokens), static_cast<unsigned>(parts));
  const auto launch = [&](auto one, auto two, auto three, auto four) {
    const int64_t turns = (rounds + parts - 1) / parts;
    (turns == 1 ? one : turns == 2 ? two : turns == 3 ? three : four)<<<grid, 256, 0, stream>>>(a);
  };
  if (s.head_dim == 64) {
    launch(attention_batch_project_kernel<64, 1>, attention_batch_project_kernel<64, 2>,
           attention_batch_project_kernel<64, 3>, attention_batch_project_kernel<64, 4>);
  } else {
    launch(attention_batch_project_kernel<128, 1>, attention_batch_project_kernel<128, 2>,
           attention_batch_project_kernel<128, 3>, attention_batch_project_kernel<128, 4>);
  }
  return launched("attention_batch_project");
}

}  // namespace
}  // namespace omnia

extern "C" int32_t omnia_attention_batch_project(
    const uint16_t* raw_queries, int64_t query_stride, const uint16_t* raw_keys, int64_t key_stride,
    const uint16_t* raw_values, int64_t value_stride, const uint16_t* query_weight, const uint16_t* key_weight,
    const float* cos_rows, const float* sin_rows, int64_t table_stride, int64_t angle_rows, int64_t rotary_pairs,
    float mscale, float eps, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, void* queries,
    int32_t wide_queries, uint16_t* keys, uint16_t* values, int64_t pages, int64_t page_rows, const int32_t* tables, int64_t sequences,
    int64_t width, const int32_t* lengths, const int32_t* token_map, hipStream_t stream) {
  using namespace omnia;
  omnia_attention_batch_step_t s{};
  s.raw_queries = raw_queries;
  s.raw_keys = raw_keys;
  s.raw_values = raw_values;
  s.query_stride = query_stride;
  s.key_stride = key_stride;
  s.value_stride = value_stride;
  s.query_weight = query_weight;
  s.key_weight = key_weight;
  s.cos_rows = cos_rows;
  s.sin_rows = sin_rows;
  s.table_stride = table_stride;
  s.angle_rows = angle_rows;
  s.rotary_pairs = rotary_pairs;
  s.mscale = mscale;
  s.eps = eps;
  s.tokens = tokens;
  s.heads = heads;
  s.kv_heads = kv_heads;
  s.head_dim = head_dim;
  s.keys = keys;
  s.values = values;
  s.pages = pages;
  s.page_rows = page_rows;
  s.tables = tables;
  s.sequences = sequences;
  s.width = width;
  s.lengths = lengths;
  s.token_map = token_map;
  return project(s, queries, wide_queries, stream);
}

extern "C" int64_t omnia_attention_batch_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads,
                                                         int64_t head_dim, int64_t prefix, int64_t own_rows,
                                                         int64_t own_total, int64_t own_tiles) {
  using namespace omnia;
  if (!geometry_served(tokens, heads, kv_heads, head_dim, prefix, own_rows, own_tiles) || own_total < 0) return -EINVAL;
  const Plan p = plan_for(tokens, heads, kv_heads, head_dim, prefix, own_rows, own_total, own_tiles);
  const int64_t splits = p.prefix_splits + p.own_splits;
  return splits == 1 ? 0 : splits * tokens * heads * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

namespace omnia {
namespace {
// `fresh`: the step's prologue, where the kernels take the new tokens' raw rows in place of queries.
int32_t attend(const BatchProjectArgs* fresh, const void* queries, int32_t wide_queries, const uint16_t* keys,
                                         const uint16_t* values, int64_t pages, int64_t page_rows, const int32_t* tables, int64_t sequences,
                                         int64_t width, const int32_t* lengths, const int32_t* token_map,
                                         int64_t tokens, const int32_t* tiles, int64_t own_tiles, int64_t prefix,
                                         int64_t prefix_sequence, int64_t own_rows, int64_t own_total,
                                         int64_t heads, int64_t kv_heads, int64_t head_dim,
                                         const uint16_t* sinks, float scale, void* workspace, int64_t workspace_bytes,
                                         uint16_t* out, hipStream_t stream) {
  OMNIA_REQUIRE(geometry_served(tokens, heads, kv_heads, head_dim, prefix, own_rows, own_tiles) && own_total >= 0,
                "attention_batch: head_dim 64 or 128, heads a multiple of kv_heads, fewer than 2^30 rows");
  const int shift = page_shift_of(page_rows);
  OMNIA_REQUIRE(shift > 0, "attention_batch: page_rows must be 16, 32, 64, 128 or 256");
  OMNIA_REQUIRE(pages > 0 && pages < (int64_t{1} << 31) && sequences > 0 && sequences < (int64_t{1} << 31) &&
                    width > 0 && width < (int64_t{1} << 31) / page_rows,
                "attention_batch: bad tables");
  OMNIA_REQUIRE(prefix == 0 || (prefix_sequence >= 0 && prefix_sequence < sequences),
                "attention_batch: no such sequence to read the shared rows through");
  OMNIA_REQUIRE(scale > 0.0f && scale * kLog2e < INFINITY, "attention_batch: the scale must be positive, below 2^127");
  if (tokens == 0) return 0;
  OMNIA_REQUIRE(queries && keys && values && tables && lengths && token_map && out && (own_tiles == 0 || tiles),
                "attention_batch: null pointer");
  OMNIA_REQUIRE(aligned16(queries) && aligned16(keys) && aligned16(values) && aligned16(out) && aligned16(tiles),
                "attention_batch: pointers must be 16-byte aligned");
  const int64_t need = omnia_attention_batch_workspace_bytes(tokens, heads, kv_heads, head_dim, prefix, own_rows,
                                                             own_total, own_tiles);
  OMNIA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
                "attention_batch: workspace too small (omnia_attention_batch_workspace_bytes) or not aligned");
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  const Plan p = plan_for(tokens, heads, kv_heads, head_dim, prefix, own_rows, own_total, own_tiles);
  const BatchArgs a{queries, keys, values, reinterpret_cast<const int4*>(tiles), sinks, out,
                    static_cast<float*>(workspace),
                    {tables, lengths, reinterpret_cast<const int2*>(token_map), static_cast<int>(sequences),
                     static_cast<int>(width), static_cast<int>(pages), shift},
                    static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(heads / kv_heads),
                    static_cast<int>(tokens), static_cast<int>(p.prefix), static_cast<int>(prefix_sequence),
                    static_cast<int>(p.prefix_tiles), static_cast<int>(own_tiles), static_cast<int>(p.prefix_splits), static_cast<int>(p.prefix_keys),
                    static_cast<int>(p.own_splits), static_cast<int>(p.own_keys), scale * kLog2e,
                    fresh != nullptr ? *fresh : BatchProjectArgs{}};
  const int64_t blocks = kv_heads * (p.prefix_tiles * p.prefix_splits + own_tiles * p.own_splits);
  OMNIA_REQUIRE(blocks < (int64_t{1} << 31), "attention_batch: too many tiles");
  const bool wide = wide_queries != 0;
  if (p.own_alone) {
    const auto kernel = head_dim == 64
                            ? (fresh ? attention_own_kernel<64, 2, true> : wide ? attention_own_kernel<64, 2> : attention_own_kernel<64, 1>)
                            : (fresh ? attention_own_kernel<128, 2, true> : wide ? attention_own_kernel<128, 2> : attention_own_kernel<128, 1>);
    kernel<<<dim3(static_cast<unsigned>(blocks)), 64, 0, stream>>>(a);
  } else if (blocks > 0) {
    const auto kernel = head_dim == 64
                            ? (fresh ? attention_batch_kernel<64, 2, true> : wide ? attention_batch_kernel<64, 2> : attention_batch_kernel<64, 1>)
                            : (fresh ? attention_batch_kernel<128, 2, true> : wide ? attention_batch_kernel<128, 2> : attention_batch_kernel<128, 1>);
    kernel<<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(a);
  }
  if (p.prefix_splits + p.own_splits != 1) {
    head_dim == 64 ? launch_merge<64>(a, stream) : launch_merge<128>(a, stream);
  }
  return launched("attention_batch");
}
}  // namespace
}  // namespace omnia

extern "C" int32_t omnia_attention_batch(const void* queries, int32_t wide_queries, const uint16_t* keys,
                                         const uint16_t* values, int64_t pages, int64_t page_rows, const int32_t* tables, int64_t sequences,
                                         int64_t width, const int32_t* lengths, const int32_t* token_map,
                                         int64_t tokens, const int32_t* tiles, int64_t own_tiles, int64_t prefix,
                                         int64_t prefix_sequence, int64_t own_rows, int64_t own_total,
                                         int64_t heads, int64_t kv_heads, int64_t head_dim,
                                         const uint16_t* sinks, float scale, void* workspace, int64_t workspace_bytes,
                                         uint16_t* out, hipStream_t stream) {
  return omnia::attend(nullptr, queries, wide_queries, keys, values, pages, page_rows, tables, sequences, width, lengths,
                       token_map, tokens, tiles, own_tiles, prefix, prefix_sequence, own_rows, own_total, heads, kv_heads,
                       head_dim, sinks, scale, workspace, workspace_bytes, out, stream);
}

extern "C" int64_t omnia_attention_batch_step_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                    int64_t prefix, int64_t own_rows, int64_t own_total,
                                                    int64_t own_tiles) {
  using namespace omnia;
  const int64_t more = omnia_attention_batch_workspace_bytes(tokens, heads, kv_heads, head_dim, prefix, own_rows,
                                                             own_total, own_tiles);
  return more < 0 ? more : query_bytes(tokens, heads, head_dim) + more;
}

extern "C" int32_t omnia_attention_batch_step(const omnia_attention_batch_step_t* s, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(s != nullptr, "attention_batch_step: null pointer");
  if (s->queries != nullptr) return project(*s, s->queries, 0, stream);
  const int64_t need = omnia_attention_batch_step_bytes(s->tokens, s->heads, s->kv_heads, s->head_dim, s->prefix,
                                                        s->own_rows, s->own_total, s->own_tiles);
  OMNIA_REQUIRE(need >= 0, "attention_batch_step: bad geometry");
  OMNIA_REQUIRE(need == 0 || (s->workspace && s->workspace_bytes >= need && aligned16(s->workspace)),
                "attention_batch_step: workspace too small (omnia_attention_batch_step_bytes) or not aligned");
  const int64_t queries = query_bytes(s->tokens, s->heads, s->head_dim);
  const bool fresh = takes_fresh(*s);
  const int32_t rc = fresh ? project_refused(*s, s->workspace) : project(*s, s->workspace, 1, stream);
  if (rc != 0) return rc;
  const BatchProjectArgs rows = project_args(*s, s->workspace, 1);
  return attend(fresh ? &rows : nullptr, s->workspace, 1, s->keys, s->values, s->pages, s->page_rows, s->tables,
                s->sequences, s->width, s->lengths, s->token_map, s->tokens, s->tiles, s->own_tiles, s->prefix,
                s->prefix_sequence, s->own_rows, s->own_total, s->heads, s->kv_heads, s->head_dim, s->sinks, s->scale,
                static_cast<char*>(s->workspace) + queries, s->workspace_bytes - queries, s->out, stream);
}
