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
  __device__ __forceinline__ int before(int2 token) const {
    return token.x >= 0 && token.x < sequences ? lengths[token.x] + token.y : -1;
  }
  // The page of a sequence's row, or -1 where there is none.
  __device__ __forceinline__ int page(int sequence, int row) const {
    const int index = row >> page_shift;
    if (index >= width) return -1;
    const int id = tables[static_cast<int64_t>(sequence) * width + index];
    return id < pages ? id : -1;
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
  uint16_t* queries;        // [tokens, heads, D]
  uint16_t* pool[2];        // a layer's keys and values [pages, kv_heads, page_rows, D]
  PageTables at;
  int heads, kv_heads, tokens, pairs;
  float mscale, eps;
};

// One head vector of one token per D / 8 lanes, 16 bytes a lane. The norm, the rotation and
// mscale stay in fp32 and are rounded once, where they are stored.
template <int D>
__global__ __launch_bounds__(256) void attention_batch_project_kernel(BatchProjectArgs a) {
  constexpr int kLanes = D / 8;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int slots = a.heads + 2 * a.kv_heads;
  const int64_t token = item / slots;
  int head = static_cast<int>(item % slots);
  if (token >= a.tokens) return;   // whole groups of lanes: their shuffles stay inside
  const int part = head < a.heads ? 0 : head < a.heads + a.kv_heads ? 1 : 2;
  head -= part == 0 ? 0 : part == 1 ? a.heads : a.heads + a.kv_heads;
  u32x4 v = *reinterpret_cast<const u32x4*>(a.raw[part] + token * a.stride[part] + head * D + lane * 8);
  const int2 whose = a.at.tokens[token];
  const int position = a.at.before(whose);
  if (part < 2) {
    float x[8];
    unpack8(v, x);
    const uint16_t* gain = a.gain[part];
    if (gain != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
      sum = group_sum<kLanes>(sum);
      const float inv = 1.0f / sqrtf(sum / static_cast<float>(D) + a.eps);
      float w[8];
      unpack8(*reinterpret_cast<const u32x4*>(gain + lane * 8), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = w[i] * (x[i] * inv);
    }
    if (a.pairs > 0) {
      const int half = a.pairs / 8;   // lanes of one half of the rotated block
      const int first = lane < half ? lane : lane - half;
      const int partner = lane < half ? lane + half : lane - half;
      // Lanes past the rotated block read its first angles and keep their values; a position
      // past the table reads its last row.
      const int64_t row = min(static_cast<int64_t>(max(position, 0)), a.angle_rows - 1) * a.table_stride;
      const int at = lane < 2 * half ? first * 8 : 0;
      float c[8], s[8];
      *reinterpret_cast<f32x4*>(c) = *reinterpret_cast<const f32x4*>(a.cos + row + at);
      *reinterpret_cast<f32x4*>(c + 4) = *reinterpret_cast<const f32x4*>(a.cos + row + at + 4);
      *reinterpret_cast<f32x4*>(s) = *reinterpret_cast<const f32x4*>(a.sin + row + at);
      *reinterpret_cast<f32x4*>(s + 4) = *reinterpret_cast<const f32x4*>(a.sin + row + at + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float mine = x[i] * a.mscale;
        const float other = __shfl(mine, partner < kLanes ? partner : lane, kLanes);
        const float turned = lane < half ? mine * c[i] - other * s[i] : other * s[i] + mine * c[i];
        x[i] = lane < 2 * half ? turned : x[i];
      }
    }
    v = pack8(x);
  }
  if (part == 0) {
    *reinterpret_cast<u32x4*>(a.queries + (token * a.heads + head) * D + lane * 8) = v;
    return;
  }
  const int page = position < 0 ? -1 : a.at.page(whose.x, position);
  if (page < 0) return;
  const int row = position & ((1 << a.at.page_shift) - 1);
  const int64_t to = ((static_cast<int64_t>(page) * a.kv_heads + head) << a.at.page_shift) + row;
  *reinterpret_cast<u32x4*>(a.pool[part - 1] + to * D + lane * 8) = v;
}

// ---- attention ------------------------------------------------------------------------

struct BatchArgs {
  const uint16_t* q;        // [tokens, heads, D]
  const uint16_t* keys;     // a layer's [pages, kv_heads, page_rows, D]
  const uint16_t* values;
  const int2* tiles;        // own pieces: query rows [x, y) of one sequence
  const uint16_t* sinks;    // [heads] or null
  uint16_t* out;            // [tokens, heads, D]
  float* partial;           // [tokens * heads, splits, D] contexts, then [tokens * heads, splits, 2]
  PageTables at;
  int heads, kv_heads, group, tokens, prefix, prefix_tiles, own_tiles;
  int prefix_splits, prefix_keys, own_splits, own_keys;   // splits of either part, keys of one
  float scale_log2;
};

constexpr int kWaveRows = 32, kWaves = 4, kTileRows = kWaveRows * kWaves, kTileKeys = 64;

// A query row is one head of one token: of a kv head, row r is head r % group of token
// r / group. A workgroup takes 128 of them (32 a wave) and walks its piece's keys in tiles of
// 64 through two LDS buffers, the next tile's rows in registers while this one is multiplied.
//
// Scores are taken transposed, S^T = K Q^T on 32x32x16 MFMA: a lane then holds 32 scores of
// one row (column lane % 32), so the softmax needs one cross-lane step, its state is a scalar
// a lane, and P^T is the B operand of O^T = V^T P^T as it stands: the MFMA's k index of lane
// half h, element j names key 8 (j / 4) + 4 h + j % 4, for both operands. V^T comes out of LDS
// by the transposing read.
//
// The weights are rounded to bf16 for that product, half a step of 2^-8 each, once more than
// the result's own rounding; their sum is taken before it, in fp32. (The weights' errors are
// independent and average out over the attended rows.)
//
// Tiles start at multiples of 64 rows and pages hold 16 or more, so 16 rows from a multiple of
// 16 lie in one page: its id is looked up once for them.
template <int D>
__global__ __launch_bounds__(256, 2) void attention_batch_kernel(BatchArgs a) {
  constexpr int kSteps = D / 16, kBlocks = D / 32, kChunks = D / 8;
  constexpr int kLoads = kTileKeys * kChunks / 256;   // 16-byte vectors a thread stages, each of K and V
  constexpr int kTile = kTileKeys * D;                // elements of one tile
  __shared__ __attribute__((aligned(16))) uint16_t lds[4 * kTile];   // K, V of two stages
  __shared__ unsigned long long odd_rows[3];   // of a stage: rows whose values are not all finite

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int column = lane % 32, half = lane / 32;
  const int rows = a.tokens * a.group;

  // Which piece: the shared rows' first, for a kv head and a split the row tiles side by side.
  const int prefix_blocks = a.kv_heads * a.prefix_splits * a.prefix_tiles;
  int block = xcd_contiguous_block(blockIdx.x, gridDim.x);
  const bool shared = block < prefix_blocks;
  int first_row, end_row, split, kv_head;
  if (shared) {
    first_row = block % a.prefix_tiles * kTileRows;
    end_row = min(first_row + kTileRows, rows);
    block /= a.prefix_tiles;
    split = block % a.prefix_splits;
    kv_head = block / a.prefix_splits;
  } else {
    block -= prefix_blocks;
    split = block % a.own_splits;
    block /= a.own_splits;
    kv_head = block % a.kv_heads;
    const int2 tile = a.tiles[block / a.kv_heads];
    first_row = min(max(tile.x, 0), rows - 1);
    end_row = min(min(max(tile.y, first_row + 1), rows), first_row + kTileRows);
  }
  // This lane's row, and the rows it may see; a workgroup's keys end where the last one's do.
  const int row = min(first_row + wave * kWaveRows + column, end_row - 1);
  const bool live = first_row + wave * kWaveRows + column < end_row;
  const int token = row / a.group, head = kv_head * a.group + row % a.group;
  const int2 whose = a.at.tokens[token];
  const int limit = min(a.at.before(whose) + 1, shared ? a.prefix : INT32_MAX);
  const int low = shared ? split * a.prefix_keys : a.prefix + split * a.own_keys;
  int high;   // past the last key of any row
  bool mixed; // rows that see different keys
  int sequence;
  {
    const int2 first = a.at.tokens[first_row / a.group], last = a.at.tokens[(end_row - 1) / a.group];
    sequence = first.x;
    if (shared) {
      high = min(low + a.prefix_keys, a.prefix);
      mixed = false;
    } else {
      high = min(low + a.own_keys, a.at.before(last) + 1);
      mixed = last.y != first.y;
    }
    sequence = shared ? a.at.tokens[0].x : sequence;
    if (sequence < 0 || sequence >= a.at.sequences) high = low;
  }
  // Rows that stop before the shared ones end are not expected of a plan, but served.
  if (shared && __syncthreads_or(limit < high)) mixed = true;
  if (!shared && low >= high) return;   // no row of the tile reaches this split, nor is it merged

  // Q^T as the B operand: column = row, k = 8 half + j of each 16-wide step.
  s16x8 q[kSteps];
  {
    const uint16_t* from = a.q + (static_cast<int64_t>(token) * a.heads + head) * D + 8 * half;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const s16x8*>(from + 16 * s);
  }

  // Staging: thread t's vector i is row (t + 256 i) / kChunks, chunk t % kChunks of the tile.
  // Chunks are permuted in LDS so that both operands' reads touch every bank once: K's 16
  // rows of one chunk, V's four rows of one 64-byte group. A row outside [low, high), or of no
  // page, comes as zeros (a zero weight times what the page happens to hold could be a NaN).
  const int chunk = threadIdx.x % kChunks;
  u32x4 stage_k[kLoads], stage_v[kLoads];
  auto load_tile = [&](int tile) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int key = tile * kTileKeys + (static_cast<int>(threadIdx.x) + 256 * i) / kChunks;
      const int sixteen = __builtin_amdgcn_readfirstlane(key & ~15);   // of the whole wave
      const int page = sixteen < high ? a.at.page(sequence, sixteen) : -1;
      const int64_t first = ((static_cast<int64_t>(max(page, 0)) * a.kv_heads + kv_head) << a.at.page_shift) +
                            (sixteen & ((1 << a.at.page_shift) - 1));
      const int64_t at = (first + (key & 15)) * D + chunk * 8;
      stage_k[i] = stage_v[i] = u32x4{0, 0, 0, 0};
      if (page >= 0 && key >= low && key < high) {
        stage_k[i] = *reinterpret_cast<const u32x4*>(a.keys + at);
        stage_v[i] = *reinterpret_cast<const u32x4*>(a.values + at);
      }
    }
  };
  // Where rows see different keys, a value that is not finite is taken out and its row marked:
  // a row that does not see it would have zero times it, a NaN.
  auto store_tile = [&](int stage, int mark) {
    uint16_t* tile_k = lds + stage * 2 * kTile;
    uint16_t* tile_v = tile_k + kTile;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = (static_cast<int>(threadIdx.x) + 256 * i) / kChunks;
      const int turn_k = D == 128 ? at & 15 : (at >> 1) & 7;
      const int turn_v = D == 128 ? (at & 3) << 2 : (at & 2) << 1;
      if (mixed) {
        bool found = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t word = stage_v[i][j];
          const bool lo = (word & 0x7f80u) == 0x7f80u, hi = (word & 0x7f800000u) == 0x7f800000u;
          stage_v[i][j] = word & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
          found = found || lo || hi;
        }
        if (found) atomicOr(&odd_rows[mark], 1ull << at);
      }
      *reinterpret_cast<u32x4*>(tile_k + at * D + (chunk ^ turn_k) * 8) = stage_k[i];
      *reinterpret_cast<u32x4*>(tile_v + at * D + (chunk ^ turn_v) * 8) = stage_v[i];
    }
  };

  // Where this lane reads: K row `column`, chunk 2 s + half; V keys 4 half + sub / 4, 4
  // values from 16 (lane / 16 % 2) + 4 (sub % 4) of each 32-wide block.
  const int turn_k = D == 128 ? column & 15 : (column >> 1) & 7;
  const int key_at = column * D + ((half ^ turn_k) * 8);
  const int sub = lane % 16;
  int value_at[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int r = sub / 4;
    const int turn = D == 128 ? r << 2 : (r & 2) << 1;
    const int piece = (b * 4 + 2 * (lane / 16 % 2) + (sub % 4) / 2) ^ turn;
    value_at[b] = (4 * half + r) * D + piece * 8 + (sub % 2) * 4;
  }

  f32x16 out[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) out[b] = f32x16{};
  float top = -INFINITY, total = 0.0f;

  const int tiles = (high + kTileKeys - 1) / kTileKeys;   // past the last
  int tile = low / kTileKeys;
  if (threadIdx.x < 3) odd_rows[threadIdx.x] = 0;
  __syncthreads();
  if (tile < tiles) {
    load_tile(tile);
    store_tile(0, 0);
  }
  lds_barrier();
  int mark = 0;
  for (int turn = 0; tile < tiles; turn ^= 1, ++tile) {
    const bool more = tile + 1 < tiles;
    if (more) load_tile(tile + 1);
    const int next_mark = mark == 2 ? 0 : mark + 1;
    // The mark after the next one was last read a tile ago, behind a barrier.
    if (threadIdx.x == 0) odd_rows[next_mark == 2 ? 0 : next_mark + 1] = 0;
    const int key0 = tile * kTileKeys;
    if (first_row + wave * kWaveRows < end_row) {   // the same for the whole wave
      const uint16_t* tile_k = lds + turn * 2 * kTile;
      const uint16_t* tile_v = tile_k + kTile;
      f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const s16x8 k = *reinterpret_cast<const s16x8*>(tile_k + kb * 32 * D + (key_at ^ (step * 16)));
          s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, k),
                                                          __builtin_bit_cast(bf16x8, q[step]), s[kb], 0, 0, 0);
        }
      }
      // Keys that count: of this piece, seen by the row, on a page that is there.
      uint32_t absent = 0;   // sixteens of the tile without a page
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * i;
        absent |= key < high && a.at.page(sequence, key) < 0 ? 1u << i : 0u;
      }
      if (mixed || key0 < low || key0 + kTileKeys > high || absent != 0) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int in = (e / 16) * 32 + 8 * ((e % 16) / 4) + 4 * half + e % 4;
          const int key = key0 + in;
          const bool keep = key >= low && key < high && key < limit && ((absent >> (in / 16)) & 1u) == 0;
          s[e / 16][e % 16] = keep ? s[e / 16][e % 16] : -INFINITY;
        }
      }
      float best = s[0][0];
#pragma unroll
      for (int e = 1; e < 32; ++e) best = fmaxf(best, s[e / 16][e % 16]);
      uint32_t lower, upper;
      half_pair(__float_as_uint(best), lower, upper);
      best = fmaxf(__uint_as_float(lower), __uint_as_float(upper)) * a.scale_log2;
      const float next = fmaxf(top, best);
      const float base = next == -INFINITY ? 0.0f : next;
      if (__ballot(next > top) != 0) {
        const float shrink = __builtin_amdgcn_exp2f(top - base);
        total *= shrink;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) out[b] *= shrink;
        top = next;
      }
      float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int step = 0; step < 4; ++step) {   // 16 keys each
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = __builtin_amdgcn_exp2f(
              __builtin_fmaf(s[step / 2][(step % 2) * 8 + j], a.scale_log2, -base));
          sums[j % 4] += p[j];
        }
        const u32x4 weights = pack8(p);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          typedef __attribute__((address_space(3))) s16x4_lds* LdsPtr;
          const uint16_t* at = tile_v + step * 16 * D + value_at[b];
          const s16x4_lds v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at));
          const s16x4_lds v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at + 8 * D));
          const s16x8 v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
          out[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v),
                                                           __builtin_bit_cast(bf16x8, weights), out[b], 0, 0, 0);
        }
      }
      total += (sums[0] + sums[1]) + (sums[2] + sums[3]);
      // The values that were taken out, for the rows that see them: the weight once more from
      // its score, times the value as it is.
      if (mixed) {
        unsigned long long marked = odd_rows[mark];
        while (marked != 0) {
          const int key = key0 + __builtin_ctzll(marked);
          marked &= marked - 1;
          if (key >= limit) continue;
          const int page = a.at.page(sequence, key);   // it was read from there
          const int64_t at = ((((static_cast<int64_t>(page) * a.kv_heads + kv_head) << a.at.page_shift) +
                               (key & ((1 << a.at.page_shift) - 1))) * D);
          const uint16_t* mine = a.q + (static_cast<int64_t>(token) * a.heads + head) * D;
          float score = 0.0f;
          for (int d = 0; d < D; ++d) {
            score = __builtin_fmaf(bf16_to_f32(mine[d]), bf16_to_f32(a.keys[at + d]), score);
          }
          const float weight =
              fmaxf(__builtin_amdgcn_exp2f(__builtin_fmaf(score, a.scale_log2, -base)), FLT_MIN);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float v = bf16_to_f32(a.values[at + b * 32 + 8 * (e / 4) + 4 * half + e % 4]);
              out[b][e] += fabsf(v) <= FLT_MAX ? 0.0f : weight * v;
            }
          }
        }
      }
    }
    if (more) store_tile(turn ^ 1, next_mark);
    mark = next_mark;
    lds_barrier();
  }

  uint32_t lower, upper;
  half_pair(__float_as_uint(total), lower, upper);
  total = __uint_as_float(lower) + __uint_as_float(upper);
  if (!live) return;
  const int64_t splits = a.prefix_splits + a.own_splits;
  const int64_t at = (static_cast<int64_t>(token) * a.heads + head) * splits + (shared ? split : a.prefix_splits + split);
  float* to = a.partial + at * D + 4 * half;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<f32x4*>(to + b * 32 + 8 * i) =
          f32x4{out[b][4 * i], out[b][4 * i + 1], out[b][4 * i + 2], out[b][4 * i + 3]};
    }
  }
  if (half == 0) {
    float* state = a.partial + static_cast<int64_t>(a.tokens) * a.heads * splits * D + 2 * at;
    state[0] = top;
    state[1] = total;
  }
}

// Merges a row's pieces: 4 columns a thread. A piece that the row does not reach was not
// written and is not read. A row that attends nothing comes as zeros.
template <int D>
__global__ __launch_bounds__(256) void attention_batch_merge_kernel(BatchArgs a) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = item / (D / 4);   // token * heads + head
  if (row >= static_cast<int64_t>(a.tokens) * a.heads) return;
  const int column = static_cast<int>(item % (D / 4)) * 4;
  const int64_t token = row / a.heads;
  const int own = a.at.before(a.at.tokens[token]) + 1 - a.prefix;
  const int splits = a.prefix_splits + a.own_splits;
  const int count = a.prefix_splits + min(own <= 0 ? 0 : (own + a.own_keys - 1) / a.own_keys, a.own_splits);
  const float2* states =
      reinterpret_cast<const float2*>(a.partial + static_cast<int64_t>(a.tokens) * a.heads * splits * D) + row * splits;
  const float* parts = a.partial + row * splits * D + column;
  const float sink = a.sinks != nullptr ? bf16_to_f32(a.sinks[row - token * a.heads]) : -INFINITY;
  constexpr float kLog2e = 1.4426950408889634f;
  float top = fminf(fmaxf(sink, -FLT_MAX), FLT_MAX) * kLog2e;
  top = sink == -INFINITY ? -INFINITY : fminf(fmaxf(top, -FLT_MAX), FLT_MAX);
  // The sink's own weight: 1, or 0 where it is -inf, or NaN where it is +inf or a NaN. (Its
  // maximum stays finite, so that it compares and cancels.)
  const float sink_top = top;
  const float sink_weight = __builtin_amdgcn_exp2f(sink - fmaxf(sink, -FLT_MAX));
  for (int s = 0; s < count; ++s) top = fmaxf(top, states[s].x);
  const float base = top == -INFINITY ? 0.0f : top;
  float total = a.sinks != nullptr ? sink_weight * __builtin_amdgcn_exp2f(sink_top - base) : 0.0f;
  f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = 0; s < count; ++s) {
    const float2 state = states[s];
    const f32x4 part = *reinterpret_cast<const f32x4*>(parts + static_cast<int64_t>(s) * D);
    const float factor = __builtin_amdgcn_exp2f(state.x - base);
    total = __builtin_fmaf(state.y, factor, total);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(part[i], factor, sum[i]);
  }
  const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
  uint2 packed;
  packed.x = pack_bf16(sum[0] * inverse, sum[1] * inverse);
  packed.y = pack_bf16(sum[2] * inverse, sum[3] * inverse);
  *reinterpret_cast<uint2*>(a.out + row * D + column) = packed;
}

// How the keys are cut: the shared rows and the sequences' own each into pieces of a multiple
// of 64 keys, as many as give every CU a workgroup, each of at least four tiles.
struct Plan {
  int64_t prefix_tiles, prefix_splits, prefix_keys, own_splits, own_keys;
};

constexpr int kTargetBlocks = 256, kMinSplitTiles = 4, kMaxSplits = 64;

int64_t split_count(int64_t blocks, int64_t keys) {
  if (keys <= 0 || blocks <= 0) return 0;
  const int64_t by_blocks = (kTargetBlocks + blocks - 1) / blocks;
  const int64_t by_tiles = (keys + kTileKeys - 1) / kTileKeys / kMinSplitTiles;
  const int64_t splits = by_blocks < by_tiles ? by_blocks : by_tiles;
  return splits < 1 ? 1 : splits > kMaxSplits ? kMaxSplits : splits;
}

// Keys of one of `splits` pieces, and as many pieces as that leaves.
int64_t piece_keys(int64_t keys, int64_t& splits) {
  if (splits == 0) return kTileKeys;
  const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys;
  const int64_t each = (tiles + splits - 1) / splits;
  splits = (tiles + each - 1) / each;
  return each * kTileKeys;
}

Plan plan_for(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t prefix, int64_t own_rows, int64_t own_tiles) {
  Plan p{};
  const int64_t rows = tokens * (heads / kv_heads);
  p.prefix_tiles = prefix > 0 ? (rows + kTileRows - 1) / kTileRows : 0;
  p.prefix_splits = split_count(kv_heads * p.prefix_tiles, prefix);
  p.prefix_keys = piece_keys(prefix, p.prefix_splits);
  p.own_splits = split_count(kv_heads * own_tiles, own_rows);
  p.own_keys = piece_keys(own_rows, p.own_splits);
  return p;
}

bool geometry_served(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t prefix,
                     int64_t own_rows, int64_t own_tiles) {
  constexpr int64_t kMaxRows = int64_t{1} << 30;
  return (head_dim == 64 || head_dim == 128) && kv_heads > 0 && heads > 0 && heads <= 4096 && heads % kv_heads == 0 &&
         tokens >= 0 && tokens * heads < kMaxRows && prefix >= 0 && prefix < kMaxRows && own_rows >= 0 &&
         own_rows < kMaxRows && own_tiles >= 0 && own_tiles < kMaxRows;
}

int page_shift_of(int64_t page_rows) {
  for (int shift = 4; shift <= 8; ++shift) {
    if (page_rows == int64_t{1} << shift) return shift;
  }
  return -1;
}

}  // namespace
}  // namespace omnia

extern "C" int32_t omnia_attention_batch_project(
    const uint16_t* raw_queries, int64_t query_stride, const uint16_t* raw_keys, int64_t key_stride,
    const uint16_t* raw_values, int64_t value_stride, const uint16_t* query_weight, const uint16_t* key_weight,
    const float* cos_rows, const float* sin_rows, int64_t table_stride, int64_t angle_rows, int64_t rotary_pairs,
    float mscale, float eps, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, uint16_t* queries,
    uint16_t* keys, uint16_t* values, int64_t pages, int64_t page_rows, const int32_t* tables, int64_t sequences,
    int64_t width, const int32_t* lengths, const int32_t* token_map, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(geometry_served(tokens, heads, kv_heads, head_dim, 0, 0, 0), "attention_batch_project: bad geometry");
  OMNIA_REQUIRE(rotary_pairs >= 0 && rotary_pairs % 8 == 0 && 2 * rotary_pairs <= head_dim,
                "attention_batch_project: rotary_pairs must be a multiple of 8 within the head");
  const int shift = page_shift_of(page_rows);
  OMNIA_REQUIRE(shift > 0, "attention_batch_project: page_rows must be 16, 32, 64, 128 or 256");
  OMNIA_REQUIRE(pages > 0 && pages < (int64_t{1} << 31) && sequences > 0 && sequences < (int64_t{1} << 31) &&
                    width > 0 && width < (int64_t{1} << 31) / page_rows,
                "attention_batch_project: bad tables");
  if (tokens == 0) return 0;
  OMNIA_REQUIRE(raw_queries && raw_keys && raw_values && queries && keys && values && tables && lengths && token_map,
                "attention_batch_project: null pointer");
  OMNIA_REQUIRE(aligned16(raw_queries) && aligned16(raw_keys) && aligned16(raw_values) && aligned16(queries) &&
                    aligned16(keys) && aligned16(values) && aligned16(query_weight) && aligned16(key_weight),
                "attention_batch_project: pointers must be 16-byte aligned");
  OMNIA_REQUIRE(query_stride % 8 == 0 && key_stride % 8 == 0 && value_stride % 8 == 0 &&
                    query_stride >= heads * head_dim && key_stride >= kv_heads * head_dim &&
                    value_stride >= kv_heads * head_dim,
                "attention_batch_project: row strides must be multiples of 8 covering the heads");
  OMNIA_REQUIRE(rotary_pairs == 0 || (cos_rows && sin_rows && aligned16(cos_rows) && aligned16(sin_rows) &&
                                      table_stride % 4 == 0 && table_stride >= rotary_pairs && angle_rows > 0),
                "attention_batch_project: angle rows must be 16-byte aligned and cover the pairs");
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  const BatchProjectArgs a{{raw_queries, raw_keys, raw_values}, {query_stride, key_stride, value_stride},
                           {query_weight, key_weight}, cos_rows, sin_rows, table_stride, angle_rows, queries,
                           {keys, values},
                           {tables, lengths, reinterpret_cast<const int2*>(token_map), static_cast<int>(sequences),
                            static_cast<int>(width), static_cast<int>(pages), shift},
                           static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(tokens),
                           static_cast<int>(rotary_pairs), mscale, eps};
  const int64_t threads = tokens * (heads + 2 * kv_heads) * (head_dim / 8);
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
  (head_dim == 64 ? attention_batch_project_kernel<64> : attention_batch_project_kernel<128>)<<<grid, 256, 0, stream>>>(a);
  return launched("attention_batch_project");
}

extern "C" int64_t omnia_attention_batch_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads,
                                                         int64_t head_dim, int64_t prefix, int64_t own_rows,
                                                         int64_t own_tiles) {
  using namespace omnia;
  if (!geometry_served(tokens, heads, kv_heads, head_dim, prefix, own_rows, own_tiles)) return -EINVAL;
  const Plan p = plan_for(tokens, heads, kv_heads, prefix, own_rows, own_tiles);
  return (p.prefix_splits + p.own_splits) * tokens * heads * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

extern "C" int32_t omnia_attention_batch(const uint16_t* queries, const uint16_t* keys, const uint16_t* values,
                                         int64_t pages, int64_t page_rows, const int32_t* tables, int64_t sequences,
                                         int64_t width, const int32_t* lengths, const int32_t* token_map,
                                         int64_t tokens, const int32_t* tiles, int64_t own_tiles, int64_t prefix,
                                         int64_t own_rows, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                         const uint16_t* sinks, float scale, void* workspace, int64_t workspace_bytes,
                                         uint16_t* out, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(geometry_served(tokens, heads, kv_heads, head_dim, prefix, own_rows, own_tiles),
                "attention_batch: head_dim 64 or 128, heads a multiple of kv_heads, fewer than 2^30 rows");
  const int shift = page_shift_of(page_rows);
  OMNIA_REQUIRE(shift > 0, "attention_batch: page_rows must be 16, 32, 64, 128 or 256");
  OMNIA_REQUIRE(pages > 0 && pages < (int64_t{1} << 31) && sequences > 0 && sequences < (int64_t{1} << 31) &&
                    width > 0 && width < (int64_t{1} << 31) / page_rows,
                "attention_batch: bad tables");
  OMNIA_REQUIRE(scale > 0.0f && scale < INFINITY, "attention_batch: the scale must be positive");
  if (tokens == 0) return 0;
  OMNIA_REQUIRE(queries && keys && values && tables && lengths && token_map && out && (own_tiles == 0 || tiles),
                "attention_batch: null pointer");
  OMNIA_REQUIRE(aligned16(queries) && aligned16(keys) && aligned16(values) && aligned16(out),
                "attention_batch: pointers must be 16-byte aligned");
  const int64_t need = omnia_attention_batch_workspace_bytes(tokens, heads, kv_heads, head_dim, prefix, own_rows,
                                                             own_tiles);
  OMNIA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
                "attention_batch: workspace too small (omnia_attention_batch_workspace_bytes) or not aligned");
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  const Plan p = plan_for(tokens, heads, kv_heads, prefix, own_rows, own_tiles);
  constexpr float kLog2e = 1.4426950408889634f;
  const BatchArgs a{queries, keys, values, reinterpret_cast<const int2*>(tiles), sinks, out,
                    static_cast<float*>(workspace),
                    {tables, lengths, reinterpret_cast<const int2*>(token_map), static_cast<int>(sequences),
                     static_cast<int>(width), static_cast<int>(pages), shift},
                    static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(heads / kv_heads),
                    static_cast<int>(tokens), static_cast<int>(prefix), static_cast<int>(p.prefix_tiles),
                    static_cast<int>(own_tiles), static_cast<int>(p.prefix_splits), static_cast<int>(p.prefix_keys),
                    static_cast<int>(p.own_splits), static_cast<int>(p.own_keys), scale * kLog2e};
  const int64_t blocks = kv_heads * (p.prefix_tiles * p.prefix_splits + own_tiles * p.own_splits);
  const int64_t merges = (tokens * heads * (head_dim / 4) + 255) / 256;
  OMNIA_REQUIRE(blocks < (int64_t{1} << 31) && merges < (int64_t{1} << 31), "attention_batch: too many tiles");
  if (blocks > 0) {
    const auto kernel = head_dim == 64 ? attention_batch_kernel<64> : attention_batch_kernel<128>;
    kernel<<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(a);
  }
  const auto merge = head_dim == 64 ? attention_batch_merge_kernel<64> : attention_batch_merge_kernel<128>;
  merge<<<dim3(static_cast<unsigned>(merges)), 256, 0, stream>>>(a);
  return launched("attention_batch");
}
