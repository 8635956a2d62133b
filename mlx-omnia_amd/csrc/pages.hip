// Pages of a cache that many sequences share: copying them, and editing the tables that say
// which pages a sequence lies on.
//
// A pool holds [layers, pages, kv_heads, page_rows, D] bf16 for keys and as much for values;
// sequence s's row r is row r % page_rows of page tables[s][r / page_rows], the same in every
// layer. The page ids to copy and the edits come from the host in the kernel's arguments, each
// checked before the launch: no list has to be on the device, or outlive the call, and no id
// that a kernel here follows is one that the host has not seen.
#include "common.hpp"
#include "host.hpp"

namespace omnia {
namespace {

struct Move {
  int32_t from, to, rows;
};

struct CopyArgs {
  uint16_t* pool[2];        // keys, values
  int64_t layer_stride;     // elements from a layer to the next
  int32_t* tables;          // renamed from -> to where they name a moved page, or null
  int64_t entries;          // of the tables
  int heads, page_rows, head_dim, count, layers, pieces, copies;
  Move moves[OMNIA_PAGES_MOVES];
};

constexpr int kPieceVectors = 1024;   // 16-byte vectors a workgroup copies

// One piece (16 KB) of one page of one layer of one pool a workgroup; the workgroups past the
// copies rename table entries, 256 each.
__global__ __launch_bounds__(256) void pages_copy_kernel(CopyArgs a) {
  const int block = blockIdx.x;
  if (block >= a.copies) {
    const int64_t entry = static_cast<int64_t>(block - a.copies) * 256 + threadIdx.x;
    if (entry >= a.entries) return;
    const int32_t page = a.tables[entry];
    int low = 0, high = a.count;   // the moves are sorted by `from`
    while (low < high) {
      const int middle = (low + high) / 2;
      if (a.moves[middle].from < page) {
        low = middle + 1;
      } else {
        high = middle;
      }
    }
    if (low < a.count && a.moves[low].from == page) a.tables[entry] = a.moves[low].to;
    return;
  }
  const int piece = block % a.pieces;
  const int rest = block / a.pieces;
  const int move = rest % a.count;
  const int plane = rest / a.count;   // layer, pool
  const Move m = a.moves[move];
  uint16_t* layer = a.pool[plane & 1] + (plane >> 1) * a.layer_stride;
  const int64_t page_elements = static_cast<int64_t>(a.heads) * a.page_rows * a.head_dim;
  const uint16_t* from = layer + m.from * page_elements;
  uint16_t* to = layer + m.to * page_elements;
  const int head_vectors = m.rows * a.head_dim / 8;   // of a head's rows in use
  const int vectors = a.heads * head_vectors;
  const int head_stride = a.page_rows * a.head_dim;
  u32x4 v[4];
  int at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int vector = piece * kPieceVectors + i * 256 + threadIdx.x;
    const int head = vector / head_vectors;
    at[i] = vector < vectors ? head * head_stride + (vector - head * head_vectors) * 8 : -1;
    if (at[i] >= 0) v[i] = *reinterpret_cast<const u32x4*>(from + at[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (at[i] >= 0) *reinterpret_cast<u32x4*>(to + at[i]) = v[i];
  }
}

struct Edit {
  int32_t kind, sequence, a, b, c;
};

struct EditArgs {
  int32_t* tables;
  int32_t* lengths;
  int64_t width;
  Edit edits[OMNIA_PAGES_EDITS];
};

// One edit a workgroup; the entry point has refused edits that meet in one place (`meet`).
__global__ __launch_bounds__(256) void pages_edit_kernel(EditArgs a) {
  const Edit e = a.edits[blockIdx.x];
  int32_t* row = a.tables + e.sequence * a.width;
  if (e.kind == OMNIA_PAGES_ENTRY) {
    if (threadIdx.x == 0) row[e.a] = e.b;
    return;
  }
  if (e.kind == OMNIA_PAGES_LENGTH) {
    if (threadIdx.x == 0) a.lengths[e.sequence] = e.a;
    return;
  }
  // A fork's row: `b` entries of sequence `a`, then page `c`. A cleared one has none.
  const int32_t* source = a.tables + (e.kind == OMNIA_PAGES_FORK ? e.a : e.sequence) * a.width;
  for (int64_t i = threadIdx.x; i < a.width; i += 256) row[i] = i < e.b ? source[i] : i == e.b ? e.c : -1;
  if (threadIdx.x == 0) a.lengths[e.sequence] = e.kind == OMNIA_PAGES_FORK ? a.lengths[e.a] : 0;
}

// Whether one of two edits writes what the other writes or reads.
bool meet(const Edit& x, const Edit& y) {
  const auto whole = [](const Edit& e) { return e.kind == OMNIA_PAGES_FORK || e.kind == OMNIA_PAGES_CLEAR; };
  if (x.kind == OMNIA_PAGES_FORK && x.a == y.sequence) return true;
  if (y.kind == OMNIA_PAGES_FORK && y.a == x.sequence) return true;
  if (x.sequence != y.sequence) return false;
  return whole(x) || whole(y) || (x.kind == y.kind && (x.kind == OMNIA_PAGES_LENGTH || x.a == y.a));
}

__global__ __launch_bounds__(256) void pages_advance_kernel(int32_t* lengths, const int32_t* sequences,
                                                            const int32_t* rows, int64_t all, int64_t count) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= count) return;
  const int32_t sequence = sequences[i];
  if (sequence >= 0 && sequence < all) lengths[sequence] += rows[i];
}

// A small set of page ids, open addressing: whether two moves meet is asked of at most
// OMNIA_PAGES_MOVES ids, without an allocation that could fail.
struct PageSet {
  static constexpr int kSlots = 4 * OMNIA_PAGES_MOVES;
  int32_t slots[kSlots];
  PageSet() {
    for (int32_t& s : slots) s = -1;
  }
  int find(int32_t page) const {
    int at = static_cast<int>((static_cast<uint32_t>(page) * 2654435761u) >> 16) % kSlots;
    while (slots[at] != -1 && slots[at] != page) at = (at + 1) % kSlots;
    return at;
  }
  bool has(int32_t page) const { return slots[find(page)] == page; }
  void add(int32_t page) { slots[find(page)] = page; }
};

}  // namespace
}  // namespace omnia

extern "C" int32_t omnia_pages_copy(uint16_t* keys, uint16_t* values, int64_t layers, int64_t pages, int64_t kv_heads,
                                    int64_t page_rows, int64_t head_dim, const int32_t* moves, int64_t count,
                                    int32_t* tables, int64_t entries, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(layers > 0 && layers <= 65536 && pages > 0 && pages < (int64_t{1} << 31), "pages_copy: bad pool");
  OMNIA_REQUIRE(kv_heads > 0 && kv_heads <= 4096 && head_dim > 0 && head_dim % 8 == 0 && head_dim <= 1024 &&
                    page_rows > 0 && page_rows <= 4096 && kv_heads * page_rows * head_dim < (int64_t{1} << 30),
                "pages_copy: bad page");
  OMNIA_REQUIRE(count >= 0 && count <= OMNIA_PAGES_MOVES, "pages_copy: more moves than one call takes");
  if (count == 0) return 0;
  OMNIA_REQUIRE(keys && values && moves && aligned16(keys) && aligned16(values),
                "pages_copy: null or unaligned pointer");
  OMNIA_REQUIRE(tables == nullptr || (entries >= 0 && entries < (int64_t{1} << 37)), "pages_copy: bad table");
  CopyArgs a{{keys, values}, pages * kv_heads * page_rows * head_dim, tables, tables ? entries : 0,
             static_cast<int>(kv_heads), static_cast<int>(page_rows), static_cast<int>(head_dim),
             static_cast<int>(count), static_cast<int>(layers), 0, 0, {}};
  PageSet written;
  int64_t most = 0;
  for (int64_t i = 0; i < count; ++i) {
    const Move m{moves[3 * i], moves[3 * i + 1], moves[3 * i + 2]};
    OMNIA_REQUIRE(m.from >= 0 && m.from < pages && m.to >= 0 && m.to < pages, "pages_copy: no such page");
    OMNIA_REQUIRE(m.rows > 0 && m.rows <= page_rows, "pages_copy: rows outside the page");
    OMNIA_REQUIRE(!written.has(m.to), "pages_copy: two moves write one page");
    OMNIA_REQUIRE(tables == nullptr || i == 0 || moves[3 * (i - 1)] < m.from,
                  "pages_copy: moves that rename have to be sorted by the page they leave");
    written.add(m.to);
    most = m.rows > most ? m.rows : most;
    a.moves[i] = m;
  }
  for (int64_t i = 0; i < count; ++i) {
    OMNIA_REQUIRE(!written.has(a.moves[i].from), "pages_copy: a page is both read and written");
  }
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  a.pieces = static_cast<int>((kv_heads * most * head_dim / 8 + kPieceVectors - 1) / kPieceVectors);
  const int64_t copies = a.pieces * count * layers * 2;
  const int64_t blocks = copies + (a.entries + 255) / 256;
  OMNIA_REQUIRE(blocks < (int64_t{1} << 31), "pages_copy: too many pieces for one launch");
  a.copies = static_cast<int>(copies);
  pages_copy_kernel<<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(a);
  return launched("pages_copy");
}

extern "C" int32_t omnia_pages_edit(int32_t* tables, int32_t* lengths, int64_t sequences, int64_t width, int64_t pages,
                                    const int32_t* edits, int64_t count, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(sequences > 0 && sequences < (int64_t{1} << 31) && width > 0 && width < (int64_t{1} << 31) &&
                    pages > 0 && pages < (int64_t{1} << 31),
                "pages_edit: bad tables");
  OMNIA_REQUIRE(count >= 0 && count <= OMNIA_PAGES_EDITS, "pages_edit: more edits than one call takes");
  if (count == 0) return 0;
  OMNIA_REQUIRE(tables && lengths && edits, "pages_edit: null pointer");
  EditArgs a{tables, lengths, width, {}};
  for (int64_t i = 0; i < count; ++i) {
    const Edit e{edits[5 * i], edits[5 * i + 1], edits[5 * i + 2], edits[5 * i + 3], edits[5 * i + 4]};
    OMNIA_REQUIRE(e.sequence >= 0 && e.sequence < sequences, "pages_edit: no such sequence");
    if (e.kind == OMNIA_PAGES_ENTRY) {
      OMNIA_REQUIRE(e.a >= 0 && e.a < width && e.b >= -1 && e.b < pages, "pages_edit: no such entry or page");
    } else if (e.kind == OMNIA_PAGES_LENGTH) {
      OMNIA_REQUIRE(e.a >= 0, "pages_edit: a length below zero");
    } else if (e.kind == OMNIA_PAGES_FORK) {
      OMNIA_REQUIRE(e.a >= 0 && e.a < sequences && e.a != e.sequence, "pages_edit: no such sequence to fork");
      OMNIA_REQUIRE(e.b >= 0 && e.b <= width && e.c >= -1 && e.c < pages, "pages_edit: no such entry or page");
    } else {
      OMNIA_REQUIRE(e.kind == OMNIA_PAGES_CLEAR && e.b == 0 && e.c == -1, "pages_edit: no such edit");
    }
    for (int64_t j = 0; j < i; ++j) OMNIA_REQUIRE(!meet(a.edits[j], e), "pages_edit: two edits of one place");
    a.edits[i] = e;
  }
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  pages_edit_kernel<<<dim3(static_cast<unsigned>(count)), 256, 0, stream>>>(a);
  return launched("pages_edit");
}

extern "C" int32_t omnia_pages_advance(int32_t* lengths, int64_t sequences, const int32_t* chosen, const int32_t* rows,
                                       int64_t count, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(sequences > 0 && count >= 0 && count < (int64_t{1} << 31), "pages_advance: bad counts");
  if (count == 0) return 0;
  OMNIA_REQUIRE(lengths && chosen && rows, "pages_advance: null pointer");
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  pages_advance_kernel<<<dim3(static_cast<unsigned>((count + 255) / 256)), 256, 0, stream>>>(lengths, chosen, rows,
                                                                                             sequences, count);
  return launched("pages_advance");
}
