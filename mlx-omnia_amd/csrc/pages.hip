// Pages of a cache that many sequences share: copying them, and editing the tables that say
// which pages a sequence lies on.
//
// A pool holds [layers, pages, kv_heads, page_rows, D] bf16 for keys and as much for values;
// sequence s's row r is row r % page_rows of page tables[s][r / page_rows], the same in every
// layer. The page ids to copy and the edits come from the host in the kernel's arguments, each
// checked before the launch: no list has to be on the device, or outlive the call, and no id
// that a kernel here follows is one that the host has not seen.
#include <string>

#include "common.hpp"
#include "host.hpp"

namespace omnia {
namespace {

struct Move {
  int32_t from, to, rows;
};

// A pool's pages, as far as a copy needs them.
struct Pool {
  uint16_t* pages[2];       // keys, values
  int64_t layer_stride;     // elements from a layer to the next
  int heads, page_rows, head_dim, planes;   // planes: layers of both

  // Page `page` of plane `plane` (layer, then keys or values).
  __device__ __forceinline__ uint16_t* page(int plane, int32_t page) const {
    return pages[plane & 1] + (plane >> 1) * layer_stride + static_cast<int64_t>(page) * heads * page_rows * head_dim;
  }
};

constexpr int kVectors = 2, kPieceVectors = 256 * kVectors;   // 16-byte vectors a thread and a workgroup copy

// Where thread t's i-th vector of a piece of the first `rows` rows of every head lies in a page,
// or -1 past them.
__device__ __forceinline__ int vector_at(const Pool& pool, int rows, int piece, int i) {
  const int head_vectors = rows * pool.head_dim / 8;
  const int vector = piece * kPieceVectors + i * 256 + threadIdx.x;
  const int head = vector / head_vectors;
  return head < pool.heads ? head * pool.page_rows * pool.head_dim + (vector - head * head_vectors) * 8 : -1;
}

int pieces_of(int64_t kv_heads, int64_t rows, int64_t head_dim) {
  return static_cast<int>((kv_heads * rows * head_dim / 8 + kPieceVectors - 1) / kPieceVectors);
}

struct CopyArgs {
  Pool pool;
  int32_t* tables;          // renamed from -> to where they name a moved page, or null
  int64_t entries;          // of the tables
  int count, pieces, copies;
  Move moves[OMNIA_PAGES_MOVES];
};

// One piece (8 KB) of one page of one plane a workgroup; the workgroups past the copies rename
// table entries, 256 each. Bound by memory: nothing is read or written twice, and what is
// written goes past the caches (69 pages of 16 layers, 579 MB: 88 us, 6.6 TB/s; reads past them
// as well 100 us, both through them 107; 32 KB a workgroup 94).
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
  const Move m = a.moves[rest % a.count];
  const uint16_t* from = a.pool.page(rest / a.count, m.from);
  uint16_t* to = a.pool.page(rest / a.count, m.to);
  u32x4 v[kVectors];
  int at[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    at[i] = vector_at(a.pool, m.rows, piece, i);
    if (at[i] >= 0) v[i] = *reinterpret_cast<const u32x4*>(from + at[i]);
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    if (at[i] >= 0) store_nt(reinterpret_cast<u32x4*>(to + at[i]), v[i]);
  }
}

struct Kid {
  int32_t sequence, page;
};

struct ForkArgs {
  Pool pool;
  int32_t* tables;
  int32_t* lengths;
  int64_t width;
  int parent, full, page, rows, count, pieces, groups, length;
  Kid kids[OMNIA_PAGES_MOVES];
};

constexpr int kKidsAtOnce = 16;

// A piece of the parent's last page, read once and written for 16 children, a workgroup; behind
// those one for each child's row of the table. Bound by the writes, which a step reads soon: into
// the caches (16 children, 33 rows of 36 layers, 83 MB: 13.7 us; past them, four times the bytes
// a workgroup and half the children 16.5).
__global__ __launch_bounds__(256) void pages_fork_kernel(ForkArgs a) {
  const int copies = a.pieces * a.groups * a.pool.planes;
  const int block = blockIdx.x;
  if (block >= copies) {
    const Kid kid = a.kids[block - copies];
    const int32_t* source = a.tables + a.parent * a.width;
    int32_t* row = a.tables + kid.sequence * a.width;
    for (int64_t i = threadIdx.x; i < a.width; i += 256) row[i] = i < a.full ? source[i] : i == a.full ? kid.page : -1;
    if (threadIdx.x == 0) a.lengths[kid.sequence] = a.length;
    return;
  }
  const int piece = block % a.pieces;
  const int rest = block / a.pieces;
  const int first = rest % a.groups * kKidsAtOnce, plane = rest / a.groups;
  const uint16_t* from = a.pool.page(plane, a.page);
  u32x4 v[kVectors];
  int at[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    at[i] = vector_at(a.pool, a.rows, piece, i);
    if (at[i] >= 0) v[i] = *reinterpret_cast<const u32x4*>(from + at[i]);
  }
  for (int kid = first; kid < min(first + kKidsAtOnce, a.count); ++kid) {
    uint16_t* to = a.pool.page(plane, a.kids[kid].page);
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      if (at[i] >= 0) *reinterpret_cast<u32x4*>(to + at[i]) = v[i];
    }
  }
}

struct Edit {
  int32_t kind, sequence, a, b;
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
  for (int64_t i = threadIdx.x; i < a.width; i += 256) row[i] = -1;
  if (threadIdx.x == 0) a.lengths[e.sequence] = 0;
}

// Whether two edits write one place.
bool meet(const Edit& x, const Edit& y) {
  if (x.sequence != y.sequence) return false;
  if (x.kind == OMNIA_PAGES_CLEAR || y.kind == OMNIA_PAGES_CLEAR) return true;
  return x.kind == y.kind && (x.kind == OMNIA_PAGES_LENGTH || x.a == y.a);
}

__global__ __launch_bounds__(256) void pages_advance_kernel(int32_t* lengths, const int32_t* sequences,
                                                            const int32_t* rows, int64_t all, int64_t count) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= count) return;
  const int32_t sequence = sequences[i];
  if (sequence >= 0 && sequence < all) lengths[sequence] += rows[i];
}

// A small set of numbers, open addressing: whether two moves meet is asked of at most
// OMNIA_PAGES_MOVES of them, without an allocation that could fail.
struct SmallSet {
  static constexpr int kSlots = 4 * OMNIA_PAGES_MOVES;
  int32_t slots[kSlots];
  SmallSet() {
    for (int32_t& s : slots) s = -1;
  }
  int find(int32_t number) const {
    int at = static_cast<int>((static_cast<uint32_t>(number) * 2654435761u) >> 16) % kSlots;
    while (slots[at] != -1 && slots[at] != number) at = (at + 1) % kSlots;
    return at;
  }
  bool has(int32_t number) const { return slots[find(number)] == number; }
  void add(int32_t number) { slots[find(number)] = number; }
};

// A pool's checks; an error text, or null.
const char* bad_pool(const uint16_t* keys, const uint16_t* values, int64_t layers, int64_t pages, int64_t kv_heads,
                     int64_t page_rows, int64_t head_dim) {
  if (layers <= 0 || layers > 65536 || pages <= 0 || pages >= (int64_t{1} << 31)) return "bad pool";
  if (kv_heads <= 0 || kv_heads > 4096 || head_dim <= 0 || head_dim % 8 != 0 || head_dim > 2048 || page_rows <= 0 ||
      page_rows > 4096 || kv_heads * page_rows * head_dim >= (int64_t{1} << 30)) {
    return "bad page";
  }
  return keys && values && aligned16(keys) && aligned16(values) ? nullptr : "null or unaligned pointer";
}

Pool make_pool(uint16_t* keys, uint16_t* values, int64_t layers, int64_t pages, int64_t kv_heads, int64_t page_rows,
               int64_t head_dim) {
  return Pool{{keys, values}, pages * kv_heads * page_rows * head_dim, static_cast<int>(kv_heads),
              static_cast<int>(page_rows), static_cast<int>(head_dim), static_cast<int>(2 * layers)};
}

bool bad_cache(const omnia_paged_cache_t* c) {
  constexpr int64_t kMost = int64_t{1} << 31;
  return !c || !c->host_tables || !c->rows || !c->held || !c->refs || !c->generation || !c->open || c->sequences <= 0 ||
         c->sequences >= kMost || c->width <= 0 || c->width >= kMost || c->pages <= 0 || c->pages >= kMost ||
         c->page_rows <= 0;
}

// The lowest number from `from` on below `end` whose count is none, or `end`.
template <typename T>
int64_t next_none(const T* counts, int64_t from, int64_t end) {
  while (from < end && counts[from] != 0) ++from;
  return from;
}

bool bad_tables(int64_t sequences, int64_t width, int64_t pages) {
  constexpr int64_t kMost = int64_t{1} << 31;
  return sequences <= 0 || sequences >= kMost || width <= 0 || width >= kMost || pages <= 0 || pages >= kMost;
}

}  // namespace
}  // namespace omnia

namespace omnia {
namespace {
int32_t too_few(const char* call, int64_t count, const char* what, int64_t found, int64_t all, const char* state) {
  return fail(-EINVAL, std::string(call) + ": " + std::to_string(count) + " more " + what + ", " + std::to_string(found) +
                           " of " + std::to_string(all) + " are " + state);
}
}  // namespace
}  // namespace omnia

extern "C" int32_t omnia_pages_copy(uint16_t* keys, uint16_t* values, int64_t layers, int64_t pages, int64_t kv_heads,
                                    int64_t page_rows, int64_t head_dim, const int32_t* moves, int64_t count,
                                    int32_t* tables, int64_t entries, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(count >= 0 && count <= OMNIA_PAGES_MOVES, "pages_copy: more moves than one call takes");
  const char* bad = bad_pool(keys, values, layers, pages, kv_heads, page_rows, head_dim);
  if (bad != nullptr) return fail(-EINVAL, std::string("pages_copy: ") + bad);
  if (count == 0) return 0;
  OMNIA_REQUIRE(moves, "pages_copy: null pointer");
  OMNIA_REQUIRE(tables == nullptr || (entries >= 0 && entries < (int64_t{1} << 37)), "pages_copy: bad table");
  CopyArgs a{make_pool(keys, values, layers, pages, kv_heads, page_rows, head_dim), tables, tables ? entries : 0,
             static_cast<int>(count), 0, 0, {}};
  SmallSet written;
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
  a.pieces = pieces_of(kv_heads, most, head_dim);
  const int64_t copies = a.pieces * count * layers * 2;
  const int64_t blocks = copies + (a.entries + 255) / 256;
  OMNIA_REQUIRE(blocks < (int64_t{1} << 31), "pages_copy: too many pieces for one launch");
  a.copies = static_cast<int>(copies);
  pages_copy_kernel<<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(a);
  return launched("pages_copy");
}

extern "C" int32_t omnia_pages_fork(uint16_t* keys, uint16_t* values, int64_t layers, int64_t pages, int64_t kv_heads,
                                    int64_t page_rows, int64_t head_dim, int32_t* tables, int32_t* lengths,
                                    int64_t sequences, int64_t width, int64_t parent, int64_t full, int64_t page,
                                    int64_t rows, const int32_t* kids, int64_t count, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(count >= 0 && count <= OMNIA_PAGES_MOVES, "pages_fork: more children than one call takes");
  const char* bad = bad_pool(keys, values, layers, pages, kv_heads, page_rows, head_dim);
  if (bad != nullptr) return fail(-EINVAL, std::string("pages_fork: ") + bad);
  OMNIA_REQUIRE(!bad_tables(sequences, width, pages), "pages_fork: bad tables");
  OMNIA_REQUIRE(parent >= 0 && parent < sequences, "pages_fork: no such sequence");
  OMNIA_REQUIRE(full >= 0 && full <= width && rows >= 0 && rows <= page_rows, "pages_fork: rows outside the table or page");
  OMNIA_REQUIRE(full * page_rows + rows < (int64_t{1} << 31), "pages_fork: rows outside the table or page");
  OMNIA_REQUIRE(rows == 0 || (full < width && page >= 0 && page < pages), "pages_fork: no such page");
  if (count == 0) return 0;
  OMNIA_REQUIRE(tables && lengths && kids, "pages_fork: null pointer");
  ForkArgs a{make_pool(keys, values, layers, pages, kv_heads, page_rows, head_dim), tables, lengths, width,
             static_cast<int>(parent), static_cast<int>(full), static_cast<int>(page), static_cast<int>(rows),
             static_cast<int>(count), 0, static_cast<int>((count + kKidsAtOnce - 1) / kKidsAtOnce),
             static_cast<int>(full * page_rows + rows), {}};
  SmallSet named, written;
  for (int64_t i = 0; i < count; ++i) {
    const Kid kid{kids[2 * i], kids[2 * i + 1]};
    OMNIA_REQUIRE(kid.sequence >= 0 && kid.sequence < sequences && kid.sequence != parent && !named.has(kid.sequence),
                  "pages_fork: a child is no other sequence, or named twice");
    OMNIA_REQUIRE(rows == 0 ? kid.page == -1 : kid.page >= 0 && kid.page < pages && kid.page != page &&
                                                   !written.has(kid.page),
                  "pages_fork: a child's page is no other page, or named twice");
    named.add(kid.sequence);
    if (rows != 0) written.add(kid.page);
    a.kids[i] = kid;
  }
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  a.pieces = pieces_of(kv_heads, rows, head_dim);
  const int64_t blocks = static_cast<int64_t>(a.pieces) * a.groups * a.pool.planes + count;
  OMNIA_REQUIRE(blocks < (int64_t{1} << 31), "pages_fork: too many pieces for one launch");
  pages_fork_kernel<<<dim3(static_cast<unsigned>(blocks)), 256, 0, stream>>>(a);
  return launched("pages_fork");
}

extern "C" int32_t omnia_pages_edit(int32_t* tables, int32_t* lengths, int64_t sequences, int64_t width, int64_t pages,
                                    const int32_t* edits, int64_t count, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(!bad_tables(sequences, width, pages), "pages_edit: bad tables");
  OMNIA_REQUIRE(count >= 0 && count <= OMNIA_PAGES_EDITS, "pages_edit: more edits than one call takes");
  if (count == 0) return 0;
  OMNIA_REQUIRE(tables && lengths && edits, "pages_edit: null pointer");
  EditArgs a{tables, lengths, width, {}};
  for (int64_t i = 0; i < count; ++i) {
    const Edit e{edits[4 * i], edits[4 * i + 1], edits[4 * i + 2], edits[4 * i + 3]};
    OMNIA_REQUIRE(e.sequence >= 0 && e.sequence < sequences, "pages_edit: no such sequence");
    if (e.kind == OMNIA_PAGES_ENTRY) {
      OMNIA_REQUIRE(e.a >= 0 && e.a < width && e.b >= -1 && e.b < pages, "pages_edit: no such entry or page");
    } else if (e.kind == OMNIA_PAGES_LENGTH) {
      OMNIA_REQUIRE(e.a >= 0, "pages_edit: a length below zero");
    } else {
      OMNIA_REQUIRE(e.kind == OMNIA_PAGES_CLEAR, "pages_edit: no such edit");
    }
    for (int64_t j = 0; j < i; ++j) OMNIA_REQUIRE(!meet(a.edits[j], e), "pages_edit: two edits of one place");
    a.edits[i] = e;
  }
  int32_t rc = check_device(stream);
  if (rc != 0) return rc;
  pages_edit_kernel<<<dim3(static_cast<unsigned>(count)), 256, 0, stream>>>(a);
  return launched("pages_edit");
}

// What the host keeps of a cache changes only once the device's part has been launched, so a
// refused or failed call leaves it as it was.
extern "C" int32_t omnia_paged_cache_fork(const omnia_paged_cache_t* c, int64_t parent, int64_t count, int32_t* kids,
                                          hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(!bad_cache(c), "paged_cache_fork: null pointer or bad tables");
  if (parent < 0 || parent >= c->sequences || c->open[parent] == 0) {
    return fail(-EINVAL, "paged_cache_fork: sequence " + std::to_string(parent) + " is not open");
  }
  OMNIA_REQUIRE(count >= 0, "paged_cache_fork: fewer than no forks");
  if (count == 0) return 0;
  OMNIA_REQUIRE(kids, "paged_cache_fork: null pointer");
  const int64_t full = c->rows[parent] / c->page_rows, rest = c->rows[parent] % c->page_rows;
  const int32_t* line = c->host_tables + parent * c->width;
  OMNIA_REQUIRE(full + (rest > 0 ? 1 : 0) <= c->held[parent] && c->held[parent] <= c->width,
                "paged_cache_fork: a sequence holds more rows than pages");
  for (int64_t i = 0; i < full; ++i) {
    OMNIA_REQUIRE(line[i] >= 0 && line[i] < c->pages, "paged_cache_fork: a table names a page outside the pool");
  }
  int64_t found = 0;
  for (int64_t s = next_none(c->open, 0, c->sequences); s < c->sequences && found < count;
       s = next_none(c->open, s + 1, c->sequences)) {
    kids[2 * found++] = static_cast<int32_t>(s);
  }
  if (found < count) return too_few("paged_cache_fork", count, "sequences are asked for", found, c->sequences, "not open");
  found = rest > 0 ? 0 : count;
  for (int64_t p = next_none(c->refs, 0, c->pages); p < c->pages && found < count;
       p = next_none(c->refs, p + 1, c->pages)) {
    kids[2 * found++ + 1] = static_cast<int32_t>(p);
  }
  if (found < count) return too_few("paged_cache_fork", count, "pages are needed", found, c->pages, "free");
  if (rest == 0) {
    for (int64_t i = 0; i < count; ++i) kids[2 * i + 1] = -1;
  }
  for (int64_t first = 0; first < count; first += OMNIA_PAGES_MOVES) {
    const int64_t some = count - first < OMNIA_PAGES_MOVES ? count - first : OMNIA_PAGES_MOVES;
    const int32_t rc = omnia_pages_fork(c->keys, c->values, c->layers, c->pages, c->kv_heads, c->page_rows, c->head_dim,
                                        c->tables, c->lengths, c->sequences, c->width, parent, full,
                                        rest > 0 ? line[full] : -1, rest, kids + 2 * first, some, stream);
    if (rc != 0) return rc;
  }
  for (int64_t i = 0; i < full; ++i) c->refs[line[i]] += count;
  for (int64_t i = 0; i < count; ++i) {
    const int32_t s = kids[2 * i], page = kids[2 * i + 1];
    int32_t* entries = c->host_tables + s * c->width;
    for (int64_t e = 0; e < full; ++e) entries[e] = line[e];
    if (page >= 0) {
      entries[full] = page;
      c->refs[page] = 1;
    }
    c->held[s] = full + (page >= 0 ? 1 : 0);
    c->rows[s] = c->rows[parent];
    c->generation[s] += 1;
    c->open[s] = 1;
  }
  return 0;
}

extern "C" int32_t omnia_paged_cache_free(const omnia_paged_cache_t* c, const int32_t* gone, int64_t count,
                                          hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(!bad_cache(c), "paged_cache_free: null pointer or bad tables");
  OMNIA_REQUIRE(count >= 0, "paged_cache_free: bad count");
  if (count == 0) return 0;
  OMNIA_REQUIRE(gone, "paged_cache_free: null pointer");
  // Those seen are marked in `open` until all are.
  constexpr uint8_t kSeen = 2;
  int64_t seen = 0;
  int32_t rc = 0;
  while (seen < count && rc == 0) {
    const int32_t s = gone[seen];
    if (s < 0 || s >= c->sequences || c->open[s] == 0) {
      rc = fail(-EINVAL, "paged_cache_free: sequence " + std::to_string(s) + " is not open");
    } else if (c->open[s] == kSeen) {
      rc = fail(-EINVAL, "paged_cache_free: a sequence to free is named twice");
    } else if (c->held[s] < 0 || c->held[s] > c->width) {
      rc = fail(-EINVAL, "paged_cache_free: a sequence holds more pages than its table");
    } else {
      c->open[s] = kSeen;
      ++seen;
    }
  }
  for (int64_t i = 0; i < seen; ++i) c->open[gone[i]] = 1;
  for (int64_t first = 0; first < count && rc == 0; first += OMNIA_PAGES_EDITS) {
    const int64_t some = count - first < OMNIA_PAGES_EDITS ? count - first : OMNIA_PAGES_EDITS;
    int32_t edits[4 * OMNIA_PAGES_EDITS];
    for (int64_t i = 0; i < some; ++i) {
      edits[4 * i] = OMNIA_PAGES_CLEAR;
      edits[4 * i + 1] = gone[first + i];
      edits[4 * i + 2] = edits[4 * i + 3] = 0;
    }
    rc = omnia_pages_edit(c->tables, c->lengths, c->sequences, c->width, c->pages, edits, some, stream);
  }
  if (rc != 0) return rc;
  for (int64_t i = 0; i < count; ++i) {
    const int32_t s = gone[i];
    int32_t* entries = c->host_tables + s * c->width;
    for (int64_t e = 0; e < c->held[s]; ++e) {
      if (entries[e] >= 0 && entries[e] < c->pages) c->refs[entries[e]] -= 1;
      entries[e] = -1;
    }
    c->held[s] = c->rows[s] = 0;
    c->generation[s] += 1;
    c->open[s] = 0;
  }
  return 0;
}

extern "C" int32_t omnia_paged_cache_open(const omnia_paged_cache_t* c, int64_t rows, int32_t* sequence,
                                          hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(!bad_cache(c) && sequence, "paged_cache_open: null pointer or bad tables");
  OMNIA_REQUIRE(rows >= 0, "paged_cache_open: a sequence of fewer than no rows");
  const int64_t need = rows / c->page_rows + (rows % c->page_rows > 0 ? 1 : 0);
  if (need > c->width) {
    return fail(-EINVAL, "paged_cache_open: a sequence holds at most " + std::to_string(c->width * c->page_rows) +
                             " rows, not " + std::to_string(rows));
  }
  const int64_t s = next_none(c->open, 0, c->sequences);
  if (s == c->sequences) return too_few("paged_cache_open", 1, "sequences are asked for", 0, c->sequences, "not open");
  int64_t found = 0;
  for (int64_t p = next_none(c->refs, 0, c->pages); p < c->pages && found < need;
       p = next_none(c->refs, p + 1, c->pages)) {
    ++found;
  }
  if (found < need) return too_few("paged_cache_open", need, "pages are needed", found, c->pages, "free");
  int32_t edits[4 * OMNIA_PAGES_EDITS];
  int64_t count = 0, done = 0, page = -1;
  int32_t rc = 0;
  // Its entries, and the length at the end; the line is nobody's until it is open.
  int32_t* line = c->host_tables + s * c->width;
  for (int64_t i = 0; i <= need && rc == 0; ++i) {
    if (i < need) {
      page = next_none(c->refs, page + 1, c->pages);
      line[i] = static_cast<int32_t>(page);
    } else if (rows == 0) {
      break;
    }
    const int32_t edit[4] = {i < need ? OMNIA_PAGES_ENTRY : OMNIA_PAGES_LENGTH, static_cast<int32_t>(s),
                             static_cast<int32_t>(i < need ? i : rows), static_cast<int32_t>(i < need ? page : 0)};
    for (int64_t j = 0; j < 4; ++j) edits[4 * count + j] = edit[j];
    ++count;
    done = i < need ? i + 1 : need;
    if (count == OMNIA_PAGES_EDITS || i == need) {
      rc = omnia_pages_edit(c->tables, c->lengths, c->sequences, c->width, c->pages, edits, count, stream);
      count = 0;
    }
  }
  if (rc != 0) {
    for (int64_t i = 0; i < done; ++i) line[i] = -1;
    return rc;
  }
  for (int64_t i = 0; i < need; ++i) c->refs[line[i]] = 1;
  c->held[s] = need;
  c->rows[s] = rows;
  c->generation[s] += 1;
  c->open[s] = 1;
  *sequence = static_cast<int32_t>(s);
  return 0;
}

extern "C" int32_t omnia_paged_cache_compact(const omnia_paged_cache_t* c, int64_t* live, hipStream_t stream) {
  using namespace omnia;
  OMNIA_REQUIRE(!bad_cache(c) && live, "paged_cache_compact: null pointer or bad tables");
  int64_t used = 0;
  for (int64_t p = 0; p < c->pages; ++p) used += c->refs[p] != 0 ? 1 : 0;
  int64_t target = -1, source = used - 1;
  int32_t rc = 0;
  bool moved = false;
  // As many pages in use lie behind the first `used` as free ones among them. A page that was left
  // says where to until the tables have been renamed: -1 - target.
  while (rc == 0) {
    int32_t moves[3 * OMNIA_PAGES_MOVES];
    int64_t count = 0;
    while (count < OMNIA_PAGES_MOVES) {
      do ++source; while (source < c->pages && c->refs[source] == 0);
      if (source >= c->pages) break;
      target = next_none(c->refs, target + 1, used);
      moves[3 * count] = static_cast<int32_t>(source);
      moves[3 * count + 1] = static_cast<int32_t>(target);
      moves[3 * count + 2] = static_cast<int32_t>(c->page_rows);
      ++count;
    }
    if (count == 0) break;
    rc = omnia_pages_copy(c->keys, c->values, c->layers, c->pages, c->kv_heads, c->page_rows, c->head_dim, moves, count,
                          c->tables, c->sequences * c->width, stream);
    for (int64_t i = 0; i < count && rc == 0; ++i) {
      c->refs[moves[3 * i + 1]] = c->refs[moves[3 * i]];
      c->refs[moves[3 * i]] = -1 - moves[3 * i + 1];
      moved = true;
    }
  }
  if (moved) {
    for (int64_t i = 0; i < c->sequences * c->width; ++i) {
      const int32_t page = c->host_tables[i];
      if (page >= used && page < c->pages && c->refs[page] < 0) c->host_tables[i] = static_cast<int32_t>(-1 - c->refs[page]);
    }
    for (int64_t p = used; p < c->pages; ++p) c->refs[p] = c->refs[p] < 0 ? 0 : c->refs[p];
  }
  if (rc == 0) *live = used;
  return rc;
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
