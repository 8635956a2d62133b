// Linear attention with a decay for each head (the mixers whose state stands in place of a
// cache of rows):
//   S_t = exp(g_t) S_{t-1} + w_t k_t v_t^T,   o_t = scale * q_t S_t
// over each sequence's new tokens, S [DK, DV] in fp32 read from and left in the pool of states.
//
// Steps: a workgroup takes one head of one sequence with its whole state in registers (64 KB at
// 128 x 128, all asked for at once), so a step of one token reads and writes the state once and is
// bound by that: 64 requests of 32 heads of 128 x 128, 268 MB over pools in turn, take 47 us (5.7 TB/s),
// 200 of 64 heads of 128 x 64, 839 MB, 149 us (5.6 TB/s); a plain copy reaches 6.5. Both go past the
// caches, as the states of all layers do not stay in them: 57.5 -> 50.2 us and 167 -> 156 when the lanes
// held 16 and 8 vectors (45 -> 50 for one pool of 134 MB over and over, half of which the last-level
// cache keeps).
//
// Prompts: a workgroup takes one head of one piece of a sequence, 64 tokens at a time on the matrix
// unit. Where the sequences are too few to fill the card each is cut into pieces: the pieces' own
// parts of the state first (k and v alone), then the states ahead of each, then the pieces' contexts.
// 32,768 tokens of 32 heads of 128 x 128 take 422 us back to back, and in the kernel trace 126 the parts, 12 the
// states between and 345 the contexts, at 0.77 and 0.76 PFLOP/s of products (97 and 262 GFLOP with the parts
// that 32 bits cost; a large product of bf16 alone reaches 1.2). 8,192 tokens of 64 heads of 128 x 64 take 123 us,
// in the trace 39, 12 and 96. By the counters the contexts' vector instructions take 63% of the cycles and the
// matrix unit's 53 (45 of 128 x 64), the LDS 22 without a conflict, and the clock is at 1.8 to 2 of 2.4 GHz.
#include "common.hpp"
#include "host.hpp"

namespace omnia {
namespace {

struct LinearArgs {
  const uint16_t *q, *k, *v;
  const float *decay, *strength;
  float* states;
  const int32_t *steps, *runs, *chains;
  uint16_t* out;
  float *carried, *totals;   // the workspace: states ahead of pieces, and pieces' log2 decays
  int64_t q_stride, k_stride, v_stride, decay_stride, strength_stride;
  int slots, tokens, heads, group, pieces;
  float scale;
};

// A decay of a state s: s * factor, or a slow one's as s + s * factor (exp(g) - 1): exp(g) itself, rounded
// next to 1, would be off the same way at every token or chunk of a sequence, and what a fast one leaves
// would be as a difference from 1.
struct Decay {
  float factor;
  bool slow;
};
__device__ __forceinline__ Decay decay_of(float g) {
  const float rate = expm1f(g);
  const bool slow = rate > -0.5f;
  return {slow ? rate : expf(g), slow};
}

// Two to four vectors a lane: 200 requests of 64 heads of 128 x 64 took 156 us with eight, 64 of 32 of
// 128 x 128 50.1 with 16 and 47.5 with four; of 64 x 64, 128 of 32 heads, 25.3 with four and 31.7 with one.
// (The states go out at the end: right behind the last token's update it was 49.8 for 47.5.)
constexpr int step_threads(int64_t state) { return state >= 64 * 128 ? 1024 : 256; }
template <int DK, int DV>
constexpr int kStepThreads = step_threads(DK * DV);

template <int DK, int DV>
__global__ __launch_bounds__((kStepThreads<DK, DV>)) void linear_step_kernel(LinearArgs a) {
  constexpr int kThreads = kStepThreads<DK, DV>;
  constexpr int kLanes = DV / 4;              // lanes of a state row
  constexpr int kRows = kThreads / kLanes;    // rows of a pass
  constexpr int kPasses = DK / kRows;
  constexpr int kWaves = kThreads / kWave;
  __shared__ float key[2][DK], query[2][DK];
  __shared__ f32x4 sums[2][kWaves][kLanes];
  const int entry = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const int slot = a.steps[3 * entry], first = a.steps[3 * entry + 1], count = a.steps[3 * entry + 2];
  if (slot < 0 || slot >= a.slots || first < 0 || count <= 0 || count > a.tokens - first) return;
  const int column = threadIdx.x % kLanes, row = threadIdx.x / kLanes;
  float* state = a.states + (static_cast<int64_t>(slot) * a.heads + head) * (DK * DV) + row * DV + 4 * column;
  f32x4 s[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) s[i] = load_nt(reinterpret_cast<const f32x4*>(state + i * kRows * DV));
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
    const Decay decay = decay_of(a.decay[token * a.decay_stride + head]);
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
        const float next = __builtin_fmaf(s[i][j], decay.factor, kr * v[j]);
        s[i][j] = decay.slow ? s[i][j] + next : next;
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
  for (int i = 0; i < kPasses; ++i) store_nt(reinterpret_cast<f32x4*>(state + i * kRows * DV), s[i]);
}

// ---- prompts: 64 tokens at a time ---------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4_lds __attribute__((ext_vector_type(4)));

constexpr int kChunk = 64;
constexpr int kNoLds = 0x7f;   // what a scheduling barrier lets through: all but LDS's instructions
constexpr double kLog2e = 1.4426950408889634074;

// Where 16-byte piece `piece` of row `row` lies in its row of a tile of D columns: rows of one
// piece (the products' operands) and four rows of one 64-byte group (the transposed reads) touch
// every bank once.
template <int D>
__device__ __forceinline__ int turn_of(int row) {
  return D == 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
}

// Eight fp32 numbers as bf16 operands of the matrix unit: the top halves, cut off (`x` keeps what
// is left of each, exactly).
__device__ __forceinline__ s16x8 cut(float (&x)[8]) {
  u32x4 part;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x0 = __float_as_uint(x[2 * j]), x1 = __float_as_uint(x[2 * j + 1]);
    part[j] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
    x[2 * j] -= __uint_as_float(x0 & 0xffff0000u);
    x[2 * j + 1] -= __uint_as_float(x1 & 0xffff0000u);
  }
  return __builtin_bit_cast(s16x8, part);
}

__device__ __forceinline__ f32x16 product(s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Inclusive sums over the lanes of a wave: within rows of 16, then the rows' last onto the rows behind.
template <int ctrl, int rows>
__device__ __forceinline__ double moved(double value) {   // zeros where no lane is moved from
  const uint64_t bits = __builtin_bit_cast(uint64_t, value);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), ctrl, rows, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), ctrl, rows, 0xf, false);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ double prefix_sum(double value) {
  value += moved<0x111, 0xf>(value);   // row_shr 1, 2, 4, 8
  value += moved<0x112, 0xf>(value);
  value += moved<0x114, 0xf>(value);
  value += moved<0x118, 0xf>(value);
  value += moved<0x142, 0xa>(value);   // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
  value += moved<0x143, 0xc>(value);
  return value;
}
// The last lane's value, in every lane.
__device__ __forceinline__ double last_lane(double value) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, value);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(bits), kWave - 1);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(bits >> 32), kWave - 1);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
// log2 of a decay. Past 2^-160 it leaves nothing of 32 bits, as that does; sums of -inf would differ
// by NaN, and of larger ones lose more.
__device__ __forceinline__ double log2_of(float g) { return g < -110.0f ? -160.0 : g * kLog2e; }

// 16 bytes a lane from global memory straight to LDS: lane l's come to `to` + 16 l.
__device__ __forceinline__ void load_to_lds(const void* from, uint16_t* to) {
  typedef __attribute__((address_space(1))) const void* Global;
  typedef __attribute__((address_space(3))) void* Local;
  __builtin_amdgcn_global_load_lds((Global)from, (Local)to, 16, 0, 0);
}

// A workgroup barrier for what waves exchange through LDS that leaves loads straight to LDS in flight
// (lds_barrier's fence, to which those are writes to LDS, waits for them: 32,768 tokens of 32 heads of
// 128 x 128 378.5 us for 376, 8,192 of 64 heads of 128 x 64 119.5 for 118).
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Brings a chunk's rows of D columns to LDS, with kThreads lanes; each row's 16-byte pieces lie
// turned (turn_of).
template <int D, int kThreads>
struct Rows {
  static constexpr int kPieces = D / 8;
  static constexpr int kPass = kThreads / kPieces;               // rows of a pass
  static constexpr int kTurns = kPass >= 16 ? 1 : 16 / kPass;    // passes whose pieces are turned otherwise
  static constexpr int kPasses = kChunk / kPass;
  static_assert(kPass * kPieces == kThreads && kPasses * kPass == kChunk, "whole passes");
  uint32_t stride;   // bytes
  uint32_t first;    // of this lane's row in the first pass
  uint32_t piece[kTurns];
  __device__ __forceinline__ Rows(int64_t row_stride)
      : stride(static_cast<uint32_t>(2 * row_stride)), first(threadIdx.x / kPieces * stride) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      piece[i] = ((threadIdx.x % kPieces) ^ turn_of<D>(threadIdx.x / kPieces + i * kPass)) * 16;
    }
  }
  // Rows past the last of `tokens` come as the last: their weights are zeros, and where that last row
  // is not finite, so is all that it meets.
  __device__ __forceinline__ void ask(const uint16_t* rows, int tokens, uint16_t* tile, int wave) const {
    const char* from = reinterpret_cast<const char*>(rows);
    uint16_t* to = tile + wave * kWave * 8;
    const uint32_t last = static_cast<uint32_t>(tokens - 1) * stride;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      load_to_lds(from + (min(first + i * kPass * stride, last) + piece[i % kTurns]), to + i * kThreads * 8);
    }
  }
};

// Sixteen rows' values of a column each lane and k's rows with them (of every 32 of the state's rows):
// s += k^T (left v), the scaled values in three parts.
template <int kTiles>
__device__ __forceinline__ void add_products(f32x16 (&s)[kTiles], const s16x8& values, const f32x4 (&left)[2],
                                             const s16x8 (&k)[kTiles]) {
  float x[8];
  unpack8(__builtin_bit_cast(u32x4, values), x);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= left[e / 4][e % 4];
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    const s16x8 v = cut(x);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) s[i] = product(k[i], v, s[i]);
  }
}

// Eight rows of a tile transposed, `at` in the first of them and the other four 8 rows on (whose
// pieces' turn is another by 2).
__device__ __forceinline__ s16x8 transposed(const uint16_t* tile, int at, int width) {
  typedef __attribute__((address_space(3))) s16x4_lds* LdsPtr;
  const s16x4_lds low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(tile + at));
  const s16x4_lds high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(tile + 8 * width + (at ^ 16)));
  return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Where a lane's i-th four of its state's rows lie in the workspace's states: lane by lane, 16 bytes each.
template <int DK, int DV>
__device__ __forceinline__ uint32_t held_at(int wave, int lane, int i) {
  return ((wave % (DV / 32) * (DK / 8) + i) * kWave + lane) * 4;
}

// The same of a decay given as log2.
constexpr float kLn2 = 0.693147180559945f;
__device__ __forceinline__ Decay decay_of_log2(float log2) {
  const float rate = expm1f(log2 * kLn2);
  const bool slow = rate > -0.5f;
  return {slow ? rate : __builtin_amdgcn_exp2f(log2), slow};
}

// What a chunk's decays come to, with G their sums in log2: exp(G) as fraction 2^exponent, w * scale / fraction,
// w exp(G_end - G), and G_end as a Decay.
struct Gates {
  int exponent[kChunk];
  float fraction[kChunk], strength[kChunk], left[kChunk], factor;
  int slow, pad[2];
};

// A piece of a sequence, for kHeads heads of a key head: a wave holds 32 columns of a head's state in
// the matrix unit's accumulators over all of the piece's chunks. In a chunk, with G the sums of g up
// to a token in it:
//   P[t, s] = exp(G_t - G_s) w_s (q_t . k_s), s <= t              each 32 x 32 of it by one wave
//   o_t = scale (exp(G_t) q_t S + P v),   S' = exp(G_end) S + k^T (exp(G_end - G_s) w_s v_s)
// The accumulators' order of rows is that of the products' operands over 16 rows once the state's
// rows are numbered 16 j + 8 half + 0..7 (lane (half, c) holds its column c of those), for which k is
// transposed in that order: S is an operand of q S, and the columns of P that a wave has made one of
// P v, as they are. S, P and the scaled v, fp32 all of them, enter their products as three bf16 parts,
// which hold all 24 bits, as the steps multiply them. (With S and P in two parts, of 16 bits, 12 sequences
// up to 1,501 tokens of 32 heads of 128 x 128 took 94 us for 105, 32,768 tokens 368 for 406, 8,192 of 64 heads
// of 128 x 64 115.5 for 126; the contexts then differed from those of fp32 products by 1.3e-4 of their size,
// and by 2 to 5e-5 now, as sums in another order do.) G is summed in fp64, and what the state's factors are made
// of are its differences in fp64: a fast decay ahead of a slow one would swallow the slow one's. P's weights
// are products of exp(G_t) and exp(-G_s), each a number of [1, 2) or (1/2, 1] times a power of two of its
// own, so that the fast decays' powers cancel exactly: what is left is a few fp32 roundings, and no
// exponential for each of P's numbers. Factors below 2^-126 are zeros.
// The next chunk's rows go straight to LDS while this one's are multiplied: k to the other of two
// tiles, v, which is held as operands from the start, and q, done with after the first half, to the
// same (k and v where P lies only when it is done with). Its decays are summed by the wave that has no
// part of P.
template <int DK, int DV, int kHeads>
__global__ __launch_bounds__(2 * DV * kHeads, 2) void linear_chunk_kernel(LinearArgs a) {
  constexpr int kWidth = DV * kHeads, kWaves = kWidth / 32, kThreads = 64 * kWaves;
  constexpr int kTiles = DK / 32, kSteps = DK / 16;
  __shared__ __attribute__((aligned(16))) uint16_t tile_q[kChunk * DK], tile_k0[kChunk * DK], tile_k1[kChunk * DK];
  // P^T: heads, parts, (t, 16 s), lanes: 1 KB each. Of 128 x 128, and of two heads, it lies where v did,
  // which is read first, or the LDS would hold one workgroup a CU for two; v of the next chunk is then
  // asked for later. Two heads' of 128 x 64 take the place of the next chunk's k with it: one part
  // of each lies in either, four pieces of the third behind them and the other two apart.
  constexpr int kWeights = kHeads * 3 * 6, kHeld = kChunk * kWidth / 8 / kWave;   // KB
  constexpr bool kOver = kHeads == 2 || (DK == 128 && DV == 128), kOverNext = DK == 128 && kHeads == 2;
  __shared__ u32x4 held[(kOver && !kOverNext ? kWeights : kHeld) * kWave], apart[(!kOver ? kWeights : kOverNext ? 4 : 1) * kWave];
  uint16_t* const tile_v = reinterpret_cast<uint16_t*>(held);
  const auto weight_at = [&](uint16_t* next_k, int h, int part, int frag) {
    u32x4 *const own = (kOver ? held : apart) + threadIdx.x % kWave, *const next = reinterpret_cast<u32x4*>(next_k) + threadIdx.x % kWave;
    if (!kOverNext) return own + ((h * 3 + part) * 6 + frag) * kWave;
    if (part < 2) return (part == 0 ? own : next) + (h * 6 + frag) * kWave;
    return frag < 4 ? (h == 0 ? own : next) + (12 + frag) * kWave : apart + threadIdx.x % kWave + (h * 2 + frag - 4) * kWave;
  };
  __shared__ __attribute__((aligned(16))) Gates gates0[kHeads], gates1[kHeads];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int half = lane / 32, column = lane % 32;
  const int blocks = a.heads / kHeads;
  const int entry = blockIdx.x / blocks, head0 = blockIdx.x % blocks * kHeads;
  const int mine = wave * 32 / DV, head = head0 + mine;   // the wave's
  const int32_t* run = a.runs + 5 * entry;
  const int slot = run[0], first = run[1], count = run[2], in = run[3], kind = run[4];
  if (slot < 0 || slot >= a.slots || first < 0 || count <= 0 || count > a.tokens - first || in < -1 ||
      in >= a.pieces || (in < 0 && kind != 3)) {
    return;
  }
  const int shared = head0 / a.group;
  constexpr int64_t kState = DK * DV;
  const int64_t state_at = (static_cast<int64_t>(slot) * a.heads + head) * kState;
  uint32_t own = 8 * half * DV + 32 * wave % DV + column;   // this lane's first row and its column

  const Rows<DK, kThreads> rows_q(a.q_stride), rows_k(a.k_stride);
  const Rows<kWidth, kThreads> rows_v(a.v_stride);
  auto ask_q = [&](int chunk) {
    rows_q.ask(a.q + (first + chunk) * a.q_stride + shared * DK, min(kChunk, count - chunk), tile_q, wave);
  };
  auto ask_k = [&](int chunk, uint16_t* tile) {
    rows_k.ask(a.k + (first + chunk) * a.k_stride + shared * DK, min(kChunk, count - chunk), tile, wave);
  };
  auto ask_v = [&](int chunk) {
    rows_v.ask(a.v + (first + chunk) * a.v_stride + head0 * DV, min(kChunk, count - chunk), tile_v, wave);
  };
  ask_k(0, tile_k0);
  ask_q(0);
  ask_v(0);

  // The decays of the chunk after next are asked for a chunk ahead of their sums.
  float ahead_g[kHeads], ahead_w[kHeads];
  auto ask_gates = [&](int chunk) {
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const int64_t token = first + min(chunk + lane, count - 1);
      ahead_g[h] = a.decay[token * a.decay_stride + head0 + h];
      ahead_w[h] = a.strength != nullptr ? a.strength[token * a.strength_stride + head0 + h] : 1.0f;
    }
  };
  auto sum_gates = [&](int chunk, Gates* gates) {
    const bool there = lane < count - chunk;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const float g = ahead_g[h], w = there ? ahead_w[h] : 0.0f;
      const double log2 = there ? log2_of(g) : 0.0;
      const double sum = prefix_sum(log2);
      const double end = last_lane(sum);
      const double whole = __builtin_floor(sum);
      const float rest = static_cast<float>(sum - whole);   // (NaN of a sum that is not finite)
      gates[h].exponent[lane] = static_cast<int>(__builtin_fmin(whole, 0x1p24));
      gates[h].fraction[lane] = __builtin_amdgcn_exp2f(rest);
      gates[h].strength[lane] = w * a.scale * __builtin_amdgcn_exp2f(-rest);
      gates[h].left[lane] = there ? __builtin_amdgcn_exp2f(static_cast<float>(end - sum)) * w : 0.0f;
      const Decay decay = decay_of_log2(static_cast<float>(end));
      gates[h].factor = decay.factor;   // (by every lane)
      gates[h].slow = decay.slow;
    }
  };
  if (wave == kWaves - 1) {
    ask_gates(0);
    sum_gates(0, gates0);
    ask_gates(kChunk);
  }

  f32x16 s[kTiles];
  {
    if (in >= 0) {
      const float* from = a.carried + (static_cast<int64_t>(in) * a.heads + head) * kState;
#pragma unroll
      for (int i = 0; i < 4 * kTiles; ++i) {
        const f32x4 four = *reinterpret_cast<const f32x4*>(from + held_at<DK, DV>(wave, lane, i));
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i / 4][4 * (i % 4) + e] = four[e];
      }
    } else {
      const float* from = a.states + state_at;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[i][e] = from[own + (32 * i + 16 * (e / 8) + e % 8) * DV];
      }
    }
  }

  // Where this lane reads (elements; the first, in bytes): row `column` of a tile's first 32, piece `half`, whose other
  // pieces and columns are an xor away; transposed, rows 4 half + sub / 4 (8 rows on: their turn is
  // another by 2), the four columns 4 (sub % 4) of 16, of k those that make the state's order.
  const int sub = lane % 16, row = 4 * half + sub / 4;
  const int four = (sub % 2) * 2 + sub % 4 / 2;
  const int plain = 2 * (column * DK + (half ^ turn_of<DK>(column)) * 8);   // bytes
  const int turned_k = row * DK + ((2 * (lane / 16 % 2) + four / 2) ^ turn_of<DK>(row)) * 8 + four % 2 * 4;
  const int turned_v =
      row * kWidth + ((4 * wave + 2 * (lane / 16 % 2) + sub % 4 / 2) ^ turn_of<kWidth>(row)) * 8 + sub % 2 * 4;
  // The part of P^T that a wave makes: 32 tokens t by 32 s, (0, 0), (1, 1) and (1, 0). (A fourth wave's is
  // not used.)
  const int part_t = wave == 0 ? 0 : 1, part_s = wave == 1 ? 1 : 0;

  auto take = [&](int chunk, const uint16_t* tile_k, uint16_t* next_k, const Gates* all, Gates* next) {
    const int64_t token0 = first + chunk;
    const int tokens = min(kChunk, count - chunk);
    const bool more = chunk + kChunk < count;
    const Gates& gates = all[mine];
    // Pinned: what the walk's reads start from is a few numbers, and not one for each of them.
    int at_k = turned_k, at_v = turned_v, at_q = plain, at_s = plain + 64 * part_s * DK, at_t = plain + 64 * part_t * DK;
    asm volatile("" : "+v"(at_k), "+v"(at_v), "+v"(at_q), "+v"(at_s), "+v"(at_t));
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this chunk's rows
    lds_barrier();
    s16x8 values[4];
#pragma unroll
    for (int step = 0; step < 4; ++step) values[step] = transposed(tile_v + step * 16 * kWidth, at_v, kWidth);
    // The products of P^T; here and below each step's operands are asked for ahead of the last one's products.
    const auto read = [&](const uint16_t* tile, int at, int step) {
      return *reinterpret_cast<const s16x8*>(reinterpret_cast<const char*>(tile) + (at ^ (32 * step)));
    };
    s16x8 q[2][2], kq[2];
    const auto fetch = [&](int step) {
      kq[step % 2] = read(tile_k, at_s, step);
      q[step % 2][1] = read(tile_q, at_t, step);
      __builtin_amdgcn_sched_barrier(kNoLds);
    };
    f32x16 p = f32x16{};
    fetch(0);
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      if (step + 1 < kSteps) fetch(step + 1);
      p = product(kq[step % 2], q[step % 2][1], p);
    }
    float odd[4] = {};
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const u32x4 raw = __builtin_bit_cast(u32x4, values[step]);
#pragma unroll
      for (int j = 0; j < 4; ++j) odd[j] = dot2_bf16(raw[j], 0u, odd[j]);   // NaN behind a value that is not finite
    }
    const float none = (odd[0] + odd[1]) + (odd[2] + odd[3]);
    const bool slow = __ballot(none != none) != 0;   // of the wave
    if (slow) {
      // Zero times such a value is a NaN where a token does not see it: these columns a token at a time.
      for (int t = 0; t < tokens; ++t) {
        const Decay decay = decay_of(a.decay[(token0 + t) * a.decay_stride + head]);
        const int column_v = 32 * wave + column;
        const float w = a.strength != nullptr ? a.strength[(token0 + t) * a.strength_stride + head] : 1.0f;
        const float v = w * bf16_to_f32(tile_v[t * kWidth + ((column_v / 8) ^ turn_of<kWidth>(t)) * 8 + column_v % 8]);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int at = t * DK + ((4 * i + 2 * j + half) ^ turn_of<DK>(t)) * 8;
            float kr[8], qr[8];
            unpack8(*reinterpret_cast<const u32x4*>(tile_k + at), kr);
            unpack8(*reinterpret_cast<const u32x4*>(tile_q + at), qr);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float next = __builtin_fmaf(s[i][8 * j + e], decay.factor, kr[e] * v);
              s[i][8 * j + e] = decay.slow ? s[i][8 * j + e] + next : next;
              sum = __builtin_fmaf(qr[e], s[i][8 * j + e], sum);
            }
          }
        }
        uint32_t low, high;
        half_pair(__float_as_uint(sum), low, high);
        sum = __uint_as_float(low) + __uint_as_float(high);
        if (half == 0) {
          a.out[((token0 + t) * a.heads + head) * DV + 32 * wave % DV + column] = f32_to_bf16(sum * a.scale);
        }
      }
    }
    meet();   // v is done with
    if (wave == kWaves - 1 && more) {
      sum_gates(chunk + kChunk, next);
      ask_gates(chunk + 2 * kChunk);
    }

    // 16 rows s of a part of P^T, weighed: a few at a time, to stand between the products.
    struct Unit {
      int exponent;
      float fraction, x[8];
      i32x4 exponents[2];
      f32x4 strengths[2];
    };
    const auto look = [&](Unit& u, int h, int j, int tt, int ts) {
      const int t = 32 * tt + column, at = 32 * ts + 16 * j + 4 * half;
      u.exponent = all[h].exponent[t];
      u.fraction = all[h].fraction[t];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u.exponents[i] = *reinterpret_cast<const i32x4*>(&all[h].exponent[at + 8 * i]);
        u.strengths[i] = *reinterpret_cast<const f32x4*>(&all[h].strength[at + 8 * i]);
      }
    };
    const auto weigh = [&](Unit& u, int j, int tt, int ts, int from, int end) {
      // Past this token's place in the part: none of them where the part is not on the diagonal.
      const int bound = tt == ts ? column - 4 * half - 16 * j : 32;
#pragma unroll
      for (int e = from; e < end; ++e) {
        const int i = e / 4, n = e % 4;
        const float decayed = __builtin_amdgcn_ldexpf(u.strengths[i][n], u.exponent - u.exponents[i][n]) * u.fraction;
        float weight = p[8 * j + e] * decayed;
        // Chosen, not multiplied by zero: a later token's key may not be finite. (Pinned, or the
        // compiler branches around each of them.)
        asm("" : "+v"(weight));
        u.x[e] = 8 * i + n <= bound ? weight : 0.0f;
      }
    };
    const auto keep_weights = [&](Unit& u, int h, int j, int tt, int ts, bool kept) {
      const int frag = 2 * tt + 2 * ts + j;
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        const u32x4 cut_off = __builtin_bit_cast(u32x4, cut(u.x));
        if (kept) *weight_at(next_k, h, part, frag) = cut_off;
      }
    };
    // q S, in two halves with P's weights between the products and the next chunk's rows ahead of them.
    f32x16 o[2] = {f32x16{}, f32x16{}};
    const auto fetch_q = [&](int step) {
#pragma unroll
      for (int i = 0; i < 2; ++i) q[step % 2][i] = read(tile_q + 32 * i * DK, at_q, step);
      __builtin_amdgcn_sched_barrier(kNoLds);
    };
    // (Ahead of the waves that are in their other half, and have more products: 1 to 3% of all prompts.)
    __builtin_amdgcn_s_setprio(1);
    fetch_q(0);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      constexpr int kUnitSteps = kSteps / 2 / kHeads, kShare = 8 / kUnitSteps;   // steps of a unit, weights of a step
      if (more) {
        if (part == 0 && !kOverNext) ask_k(chunk + kChunk, next_k);
        else if (part == 1 && !kOver) ask_v(chunk + kChunk);
      }
#pragma unroll
      for (int n = 0; n < kHeads; ++n) {   // 2 kHeads units in all
        const int h = (part * kHeads + n) / 2, j = (part * kHeads + n) % 2;
        Unit unit;
        look(unit, h, j, part_t, part_s);
        __builtin_amdgcn_sched_barrier(kNoLds);
#pragma unroll
        for (int i = 0; i < kUnitSteps; ++i) {
          const int step = (part * kHeads + n) * kUnitSteps + i, now = step % 2;
          if (step + 1 < kSteps) fetch_q(step + 1);
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = s[step / 2][8 * (step % 2) + e];
#pragma unroll
          for (int third = 0; third < 3; ++third) {
            const s16x8 cut_off = cut(x);
            o[0] = product(cut_off, q[now][0], o[0]);
            o[1] = product(cut_off, q[now][1], o[1]);
          }
          weigh(unit, j, part_t, part_s, kShare * i, kShare * (i + 1));
        }
        keep_weights(unit, h, j, part_t, part_s, wave < 3);
      }
    }
    if (kWaves < 3 && wave == kWaves - 1) {
      p = f32x16{};
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        p = product(read(tile_k, at_q, step), read(tile_q + 32 * DK, at_q, step), p);
      }
#pragma unroll
      for (int n = 0; n < 2 * kHeads; ++n) {
        Unit unit;
        look(unit, n / 2, n % 2, 1, 0);
        weigh(unit, n % 2, 1, 0, 0, 8);
        keep_weights(unit, n / 2, n % 2, 1, 0, true);
      }
    }
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const int t = 32 * tt + column;
      o[tt] *= __builtin_amdgcn_ldexpf(gates.fraction[t], gates.exponent[t]) * a.scale;
    }
    const auto ask_rest = [&] {
      meet();   // P is done with
      if (kOverNext && more) ask_k(chunk + kChunk, next_k);
      if (more) ask_v(chunk + kChunk);
    };
    meet();   // P is there, q is done with
    if (more) ask_q(chunk + kChunk);
    if (slow) {
      if (kOver) ask_rest();
      return;
    }
    __builtin_amdgcn_s_setprio(0);
    // The first products' operands are asked for ahead of the decay, and each step's ahead of the last one's.
    s16x8 parts[2][3], kt[2][kTiles];   // of P's 32 t by 16 s
    f32x4 left[2][2];
    const auto fetch_state = [&](int step) {
#pragma unroll
      for (int i = 0; i < 2; ++i) left[step % 2][i] = *reinterpret_cast<const f32x4*>(&gates.left[16 * step + 8 * i + 4 * half]);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) kt[step % 2][i] = transposed(tile_k + step * 16 * DK, at_k ^ (32 * i), DK);
      __builtin_amdgcn_sched_barrier(kNoLds);
    };
    // P's parts of 32 t by 16 s in turn: (t, s / 32, s / 16 % 2).
    constexpr int kTurn[6][3] = {{0, 0, 0}, {1, 0, 0}, {0, 0, 1}, {1, 0, 1}, {1, 1, 0}, {1, 1, 1}};
    const auto fetch_part = [&](int turn) {
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        const int frag = 2 * kTurn[turn][0] + 2 * kTurn[turn][1] + kTurn[turn][2];
        parts[turn % 2][part] = __builtin_bit_cast(s16x8, *weight_at(next_k, mine, part, frag));
      }
      __builtin_amdgcn_sched_barrier(kNoLds);
    };
    const float factor = gates.factor;
    const bool slowly = __builtin_amdgcn_readfirstlane(gates.slow) != 0;
    fetch_part(0);
    // Rows past the last are out of the buffer, and not written.
    const int64_t bytes = static_cast<int64_t>(a.heads) * DV * 2;   // of a row
    const auto to = __builtin_amdgcn_make_buffer_rsrc(a.out + (token0 * a.heads + head) * DV, 0,
                                                      static_cast<int>((tokens - 1) * bytes + DV * 2), 0x00027000);
    const auto times = [&](int turn) {
      const int tt = kTurn[turn][0], step = 2 * kTurn[turn][1] + kTurn[turn][2];
#pragma unroll
      for (int part = 0; part < 3; ++part) o[tt] = product(values[step], parts[turn % 2][part], o[tt]);
    };
    const auto store = [&](int tt) {
      const int at = (32 * tt + column) * static_cast<int>(bytes) + (32 * wave % DV + 8 * half) * 2;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // A lane's fours 2 i and 2 i + 1 against the other half's: eight columns each.
        u32x4 packed;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int e = 8 * i + 2 * n;
          const auto both = __builtin_amdgcn_permlane32_swap(pack_bf16(o[tt][e], o[tt][e + 1]),
                                                             pack_bf16(o[tt][e + 4], o[tt][e + 5]), false, false);
          packed[n] = both[0];
          packed[2 + n] = both[1];
        }
        __builtin_amdgcn_raw_buffer_store_b128(packed, to, at + 32 * i, 0, 0);
      }
    };
#pragma unroll
    for (int turn = 0; turn < 6; ++turn) {
      if (turn + 1 < 6) fetch_part(turn + 1);
      if (turn == 5) {
        fetch_state(0);
        store(0);
      }
      times(turn);
    }
    if (kOver) ask_rest();
    store(1);
    if (slowly) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[i][e] = __builtin_fmaf(s[i][e], factor, s[i][e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) s[i] *= factor;
    }
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const int now = step % 2;
      if (step + 1 < 4) fetch_state(step + 1);
      add_products(s, values[step], left[now], kt[now]);
    }
  };
  for (int chunk = 0; chunk < count; chunk += 2 * kChunk) {
    take(chunk, tile_k0, tile_k1, gates0, gates1);
    if (chunk + kChunk < count) take(chunk + kChunk, tile_k1, tile_k0, gates1, gates0);
  }
  if ((kind & 2) == 0) return;
  float* to = a.states + state_at;
  asm volatile("" : "+v"(own));   // the addresses made anew: kept over the walk, they were spilled
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
#pragma unroll
    for (int e = 0; e < 16; ++e) to[own + (32 * i + 16 * (e / 8) + e % 8) * DV] = s[i][e];
  }
}

// What a piece adds to the state, for the pieces behind it: k^T (exp(G_end - G_s) w_s v_s) over all of
// its chunks, from the last to the first, so that what stands behind a chunk is known and the sums are
// never scaled. The first piece's is the state behind it: the sequence's own, decayed, comes on top at
// the end (and is kept for the piece's contexts, since the last piece writes over it).
template <int DK, int DV, int kHeads>
__global__ __launch_bounds__(2 * DV * kHeads, 2) void linear_part_kernel(LinearArgs a) {
  constexpr int kWidth = DV * kHeads, kWaves = kWidth / 32, kThreads = 64 * kWaves;
  constexpr int kTiles = DK / 32;
  __shared__ __attribute__((aligned(16))) uint16_t tile_k0[kChunk * DK], tile_k1[kChunk * DK];
  __shared__ __attribute__((aligned(16))) uint16_t tile_v0[kChunk * kWidth], tile_v1[kChunk * kWidth];
  __shared__ __attribute__((aligned(16))) float left0[kHeads][kChunk], left1[kHeads][kChunk];
  __shared__ float whole[kHeads];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int half = lane / 32, column = lane % 32;
  const int blocks = a.heads / kHeads;
  const int entry = blockIdx.x / blocks, head0 = blockIdx.x % blocks * kHeads;
  const int mine = wave * 32 / DV, head = head0 + mine;   // the wave's
  const int32_t* run = a.runs + 5 * entry;
  const int slot = run[0], first = run[1], count = run[2], in = run[3], kind = run[4];
  if (slot < 0 || slot >= a.slots || first < 0 || count <= 0 || count > a.tokens - first || in < 0 ||
      in + 1 >= a.pieces || (kind & 2) != 0) {
    return;
  }
  const int shared = head0 / a.group;
  constexpr int64_t kState = DK * DV;

  const Rows<DK, kThreads> rows_k(a.k_stride);
  const Rows<kWidth, kThreads> rows_v(a.v_stride);
  auto ask = [&](int chunk, uint16_t* tile_k, uint16_t* tile_v) {
    const int64_t token = first + chunk;
    const int tokens = min(kChunk, count - chunk);
    rows_k.ask(a.k + token * a.k_stride + shared * DK, tokens, tile_k, wave);
    rows_v.ask(a.v + token * a.v_stride + head0 * DV, tokens, tile_v, wave);
  };
  const int last = (count - 1) / kChunk * kChunk;
  ask(last, tile_k0, tile_v0);

  // The decays of the chunk after next are asked for a chunk ahead of their sums.
  float ahead_g[kHeads], ahead_w[kHeads];
  auto ask_gates = [&](int chunk) {
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const int64_t token = first + min(max(chunk, 0) + lane, count - 1);
      ahead_g[h] = a.decay[token * a.decay_stride + head0 + h];
      ahead_w[h] = a.strength != nullptr ? a.strength[token * a.strength_stride + head0 + h] : 1.0f;
    }
  };
  double behind[kHeads] = {};   // the log2 decays behind the chunk
  auto sum_gates = [&](int chunk, float (*left)[kChunk]) {
    const bool there = lane < count - chunk;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const double sum = prefix_sum(there ? log2_of(ahead_g[h]) : 0.0);
      behind[h] += last_lane(sum);
      left[h][lane] = there ? __builtin_amdgcn_exp2f(static_cast<float>(behind[h] - sum)) * ahead_w[h] : 0.0f;
    }
  };
  if (wave == kWaves - 1) {
    ask_gates(last);
    sum_gates(last, left0);
    ask_gates(last - kChunk);
  }

  const int sub = lane % 16, row = 4 * half + sub / 4;   // as in the kernel above
  const int four = (sub % 2) * 2 + sub % 4 / 2;
  const int turned_k = row * DK + ((2 * (lane / 16 % 2) + four / 2) ^ turn_of<DK>(row)) * 8 + four % 2 * 4;
  const int turned_v =
      row * kWidth + ((4 * wave + 2 * (lane / 16 % 2) + sub % 4 / 2) ^ turn_of<kWidth>(row)) * 8 + sub % 2 * 4;

  f32x16 s[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) s[i] = f32x16{};
  auto take = [&](int chunk, const uint16_t* tile_k, uint16_t* next_k, const uint16_t* tile_v, uint16_t* next_v,
                  const float (*all)[kChunk], float (*next)[kChunk]) {
    int at_k = turned_k, at_v = turned_v;
    asm volatile("" : "+v"(at_k), "+v"(at_v));
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this chunk's rows
    lds_barrier();
    if (chunk > 0) ask(chunk - kChunk, next_k, next_v);
    s16x8 values[2], k[2][kTiles];
    f32x4 left[2][2];
    const auto fetch = [&](int step) {
#pragma unroll
      for (int i = 0; i < 2; ++i) left[step % 2][i] = *reinterpret_cast<const f32x4*>(&all[mine][16 * step + 8 * i + 4 * half]);
      values[step % 2] = transposed(tile_v + step * 16 * kWidth, at_v, kWidth);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) k[step % 2][i] = transposed(tile_k + step * 16 * DK, at_k ^ (32 * i), DK);
      __builtin_amdgcn_sched_barrier(kNoLds);
    };
    fetch(0);
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const int now = step % 2;
      if (step + 1 < 4) fetch(step + 1);
      add_products(s, values[now], left[now], k[now]);
    }
    if (wave == kWaves - 1 && chunk > 0) {
      sum_gates(chunk - kChunk, next);
      ask_gates(chunk - 2 * kChunk);
    }
  };
  for (int chunk = last; chunk >= 0; chunk -= 2 * kChunk) {
    take(chunk, tile_k0, tile_k1, tile_v0, tile_v1, left0, left1);
    if (chunk >= kChunk) take(chunk - kChunk, tile_k1, tile_k0, tile_v1, tile_v0, left1, left0);
  }

  if (wave == kWaves - 1 && lane == 0) {
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      whole[h] = static_cast<float>(behind[h]);
      a.totals[static_cast<int64_t>(in + 1) * a.heads + head0 + h] = whole[h];
    }
  }
  lds_barrier();
  const bool opens = (kind & 1) != 0;
  const float keep = __builtin_amdgcn_exp2f(whole[mine]);
  const float* from = a.states + (static_cast<int64_t>(slot) * a.heads + head) * kState;
  float* kept = a.carried + (static_cast<int64_t>(in) * a.heads + head) * kState;
  float* to = kept + a.heads * kState;
  const uint32_t own = 8 * half * DV + 32 * wave % DV + column;
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    float before[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) before[e] = opens ? from[own + (32 * i + 16 * (e / 8) + e % 8) * DV] : 0.0f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t at = held_at<DK, DV>(wave, lane, 4 * i + n);
      f32x4 sums;
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[e] = __builtin_fmaf(before[4 * n + e], keep, s[i][4 * n + e]);
      if (opens) {
        *reinterpret_cast<f32x4*>(kept + at) = f32x4{before[4 * n], before[4 * n + 1], before[4 * n + 2], before[4 * n + 3]};
      } else {
        sums = f32x4{s[i][4 * n], s[i][4 * n + 1], s[i][4 * n + 2], s[i][4 * n + 3]};   // (not 0 times what keep may be)
      }
      *reinterpret_cast<f32x4*>(to + at) = sums;
    }
  }
}

// The states ahead of a sequence's third piece on, from what each piece before added:
// X_p = 2^total X_{p-1} + U_p, in place, eight pieces' asked for together. (With pieces that sum them
// as they begin, and no launch for it, 12 sequences in up to three pieces took 94.2 us for 93.7.)
__global__ __launch_bounds__(256) void linear_carry_kernel(LinearArgs a, int state) {
  constexpr int kAhead = 8;
  const int per_head = state / (256 * 4);   // workgroups
  const int part = blockIdx.x % per_head;
  const int head = blockIdx.x / per_head % a.heads, chain = blockIdx.x / per_head / a.heads;
  const int at = a.chains[2 * chain], count = a.chains[2 * chain + 1];
  if (at < 0 || count < 3 || count > a.pieces - at) return;
  const int64_t between = static_cast<int64_t>(a.heads) * state;
  float* x = a.carried + (static_cast<int64_t>(at + 1) * a.heads + head) * state + (part * 256 + threadIdx.x) * 4;
  const float* totals = a.totals + static_cast<int64_t>(at) * a.heads + head;
  f32x4 sum = *reinterpret_cast<const f32x4*>(x);
  for (int p = 2; p < count; p += kAhead) {
    f32x4 own[kAhead];
    float keep[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int n = min(p + i, count - 1);
      own[i] = *reinterpret_cast<const f32x4*>(x + (n - 1) * between);
      keep[i] = totals[static_cast<int64_t>(n) * a.heads];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (p + i >= count) break;
      const Decay decay = decay_of_log2(keep[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float next = __builtin_fmaf(sum[j], decay.factor, own[i][j]);
        sum[j] = decay.slow ? sum[j] + next : next;
      }
      *reinterpret_cast<f32x4*>(x + (p + i - 1) * between) = sum;
    }
  }
}

// Heads of a workgroup of the prompts' kernels: two of 64 columns where they share a key head, in four
// waves that share the chunk's q and k in LDS, else one. Two workgroups a CU, which are not in step,
// do better than one of twice the waves and heads: 8,192 tokens of 64 heads of 128 x 64 119 us for
// 123.5 with four of them together, 12 sequences up to 1,501 of 32 heads of 128 x 128 97.2 for 101.1 with two.
int shared_heads(int64_t group, int64_t value_dim) { return value_dim == 64 && group % 2 == 0 ? 2 : 1; }

template <int DK, int DV, int kHeads>
void launch_runs(const LinearArgs& a, int64_t runs, int64_t handed_on, int64_t chains, hipStream_t stream) {
  const auto grid = [&](int64_t count) { return dim3(static_cast<unsigned>(count * (a.heads / kHeads))); };
  if (handed_on > 0) linear_part_kernel<DK, DV, kHeads><<<grid(handed_on), 2 * DV * kHeads, 0, stream>>>(a);
  if (chains > 0) {
    const auto blocks = static_cast<unsigned>(chains * a.heads * (DK * DV / 1024));
    linear_carry_kernel<<<dim3(blocks), 256, 0, stream>>>(a, DK * DV);
  }
  linear_chunk_kernel<DK, DV, kHeads><<<grid(runs), 2 * DV * kHeads, 0, stream>>>(a);
}

template <int DK, int DV>
void launch_linear(const LinearArgs& a, int64_t steps, int64_t runs, int64_t handed_on, int64_t chains, hipStream_t stream) {
  if (steps > 0) linear_step_kernel<DK, DV><<<dim3(static_cast<unsigned>(steps * a.heads)), kStepThreads<DK, DV>, 0, stream>>>(a);
  if (runs == 0) return;
  if constexpr (DV == 64) {
    if (shared_heads(a.group, DV) == 2) return launch_runs<DK, DV, 2>(a, runs, handed_on, chains, stream);
  }
  launch_runs<DK, DV, 1>(a, runs, handed_on, chains, stream);
}

}  // namespace
}  // namespace omnia

extern "C" int64_t omnia_linear_attention_places(int64_t heads, int64_t key_heads, int64_t key_dim, int64_t value_dim) {
  if (heads <= 0 || heads > 4096 || key_heads <= 0 || heads % key_heads != 0 || (key_dim != 64 && key_dim != 128) ||
      (value_dim != 64 && value_dim != 128)) {
    return -EINVAL;
  }
  return 2 * 256 * omnia::shared_heads(heads / key_heads, value_dim);   // two workgroups a CU
}

extern "C" int64_t omnia_linear_attention_workspace_bytes(int64_t heads, int64_t key_dim, int64_t value_dim, int64_t pieces) {
  if (heads <= 0 || heads > 4096 || (key_dim != 64 && key_dim != 128) || (value_dim != 64 && value_dim != 128) ||
      pieces < 0 || pieces >= (int64_t{1} << 24)) {
    return -EINVAL;
  }
  return pieces * heads * (key_dim * value_dim + 1) * static_cast<int64_t>(sizeof(float));
}

extern "C" int32_t omnia_linear_attention(const omnia_linear_attention_t* c, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(c != nullptr, "linear_attention: null pointer");
  OMNIA_REQUIRE((c->key_dim == 64 || c->key_dim == 128) && (c->value_dim == 64 || c->value_dim == 128),
                "linear_attention: key_dim and value_dim must be 64 or 128");
  OMNIA_REQUIRE(c->key_heads > 0 && c->heads > 0 && c->heads <= 4096 && c->heads % c->key_heads == 0,
                "linear_attention: heads must be a multiple of key_heads");
  constexpr int64_t kMost = int64_t{1} << 24;
  OMNIA_REQUIRE(c->tokens >= 0 && c->tokens < kMost && c->slots >= 0 && c->slots < kMost && c->step_count >= 0 &&
                    c->run_count >= 0 && c->step_count + c->run_count <= c->tokens,
                "linear_attention: bad token, slot, step or run count");
  OMNIA_REQUIRE(c->handed_on >= 0 && c->handed_on <= c->run_count && c->chain_count >= 0 && c->chain_count <= c->handed_on &&
                    c->pieces >= c->handed_on && c->pieces <= c->run_count,
                "linear_attention: bad piece or chain count");
  if (c->step_count + c->run_count == 0) return 0;
  OMNIA_REQUIRE(c->queries && c->keys && c->values && c->log_decay && c->states && c->out &&
                    (c->steps || c->step_count == 0) && (c->runs || c->run_count == 0) && (c->chains || c->chain_count == 0),
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
  const int64_t need = omnia_linear_attention_workspace_bytes(c->heads, c->key_dim, c->value_dim, c->pieces);
  OMNIA_REQUIRE(need == 0 || (c->workspace && c->workspace_bytes >= need && aligned16(c->workspace)),
                "linear_attention: workspace too small (omnia_linear_attention_workspace_bytes) or not aligned");
  const int64_t state = c->key_dim * c->value_dim;
  OMNIA_REQUIRE(fits_launch(c->step_count * c->heads, step_threads(state)) && fits_launch(c->run_count * c->heads, 2 * c->value_dim) &&
                    fits_launch(c->chain_count * c->heads, state / 4),
                "linear_attention: too many steps or runs for one launch");
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  float* carried = static_cast<float*>(c->workspace);
  const LinearArgs a{c->queries, c->keys, c->values, c->log_decay, c->strengths, c->states, c->steps, c->runs, c->chains,
                     c->out, carried, carried + c->pieces * c->heads * c->key_dim * c->value_dim,
                     c->query_stride, c->key_stride, c->value_stride, c->decay_stride, c->strength_stride,
                     static_cast<int>(c->slots), static_cast<int>(c->tokens), static_cast<int>(c->heads),
                     static_cast<int>(c->heads / c->key_heads), static_cast<int>(c->pieces), c->scale};
  const auto launch = c->key_dim == 64 ? (c->value_dim == 64 ? launch_linear<64, 64> : launch_linear<64, 128>)
                                       : (c->value_dim == 64 ? launch_linear<128, 64> : launch_linear<128, 128>);
  launch(a, c->step_count, c->run_count, c->handed_on, c->chain_count, stream);
  return launched("linear_attention");
}
