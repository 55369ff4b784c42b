// Eviction from paged KV by the keys' accumulated weights for gfx950: of a
// sequence's keys the `first` first, the `recent` last and the heaviest of the
// others stay, `keep` together, moved to the front of its pages in their order.
//
// Two launches. A workgroup per (sequence, set of heads) chooses: the weight of
// the last key that stays is found digit by digit (12, 12 and 8 bits of the
// weights as ordered whole numbers, histograms in LDS, the weights read again for
// each: they are in L2), then one pass over the keys in order writes the list of
// those that stay and moves their weights. Then tiles of rows move.
//
// The rows move within their own pages, so a row must not be written before
// what lies there has been read. Row j of the list comes from a place not before
// it, so what lies in a tile's rows is read by the tile itself or by
// tiles before it, of which the choice leaves the bounds: a tile reads all of its
// rows into registers, says so in a flag, waits for the flags of the one or
// two tiles that read from its rows, and writes. Tiles are handed out by a
// counter, a unit's in order: a tile only waits for tiles that were handed out
// before, to workgroups that run, and these read, and raise their flag, before they
// wait for anything; so every wait ends, whatever else the GPU does. (Only reads have to
// be done, nothing is passed on: the flags need no fences, only loads that
// have come back.)
// Bound by HBM: the rows behind the first one that leaves are read and written once.
#include <algorithm>

#include "cbk_common.hpp"

namespace cbk {
namespace {

constexpr int kThreads = 1024;   // of the choice
constexpr int kMove = 256;       // of a move
constexpr int kPieces = 8;       // a thread's pieces of a tile
constexpr uint32_t kMaxRows = 512;

struct EvictArgs {
  char* k_base;
  char* v_base;
  int64_t block_stride, token_stride;  // bytes
  uint32_t num_blocks;
  FastDiv block_div;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lens;
  int32_t* new_lens;
  float* weights;
  int64_t w_batch, w_set;
  const int32_t* keeps;  // NULL: keep
  uint32_t keep, first, recent;
  uint32_t batch, sets, max_len, most;  // most: keys that may stay
  // the move: a set's rows of pieces_row pieces, `rows` of them a tile (tile k:
  // rows [k rows, (k + 1) rows) of the list), split into `chunks` of columns
  uint32_t rows, tiles, chunks, chunk_pieces, pieces_row;
  int64_t set_bytes;
  FastDiv chunk_div;
  // scratch: for each (sequence, set) the rows that move [begin, end), the list [most],
  // the keys below k rows that stay [tiles + 1], and the flags [2 planes][chunks][tiles]
  uint2* moved;
  int32_t* list;
  int32_t* below;
  uint32_t* flags;
  uint32_t* ticket;
};

__device__ __forceinline__ uint32_t ordered(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t bits = __float_as_uint(w + 0.f);  // -0 as 0
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Adds one to a bin for each active lane; the bin of the first such lane, which may be
// that of most (weights of zero), by one of them.
__device__ __forceinline__ void count_bin(uint32_t* bins, uint32_t bin) {
  const uint32_t lead = uint32_t(__builtin_amdgcn_readfirstlane(int(bin)));
  const uint64_t same = __ballot(bin == lead);
  if (bin != lead) atomicAdd(&bins[bin], 1u);
  else if (__builtin_ctzll(same) == int(threadIdx.x & 63)) atomicAdd(&bins[lead], uint32_t(__popcll(same)));
}

// The bin, from the highest down, in which the count reaches `want` (>= 1), and
// what is still wanted of it.
__device__ __forceinline__ uint32_t find_bin(const uint32_t* bins, uint32_t count, uint32_t* want, uint32_t* scratch,
                                             uint32_t* found) {
  const uint32_t per = count / kThreads > 0 ? count / kThreads : 1;
  const bool mine = threadIdx.x * per < count;
  const uint32_t top = count - threadIdx.x * per;  // bins [top - per, top)
  uint32_t sum = 0;
  if (mine)
    for (uint32_t i = 1; i <= per; ++i) sum += bins[top - i];
  uint32_t total;
  uint32_t before = block_exclusive_scan<kThreads>(sum, scratch, &total);
  if (mine && before < *want && before + sum >= *want) {
    for (uint32_t i = 1; i <= per; ++i) {
      const uint32_t n = bins[top - i];
      if (before + n >= *want) {
        found[0] = top - i;
        found[1] = *want - before;
        break;
      }
      before += n;
    }
  }
  __syncthreads();
  const uint32_t bin = found[0];
  *want = found[1];
  __syncthreads();
  return bin;
}

__global__ __launch_bounds__(kThreads) void evict_choose_kernel(const EvictArgs a) {
  __shared__ uint32_t bins[4096];
  __shared__ uint32_t scratch[kThreads / 64], found[2], s_gone;
  const uint32_t unit = blockIdx.x, b = unit / a.sets, set = unit - b * a.sets, tid = threadIdx.x;
  const uint32_t n = uint32_t(min(max(a.lens[b], 0), int32_t(a.max_len)));
  uint32_t keep = a.keeps ? uint32_t(max(a.keeps[b], 0)) : a.keep;
  keep = max(keep, a.first + a.recent);
  if (unit == 0 && tid == 0) *a.ticket = 0;
  if (set == 0 && tid == 0) a.new_lens[b] = int32_t(min(n, keep));
  uint32_t* const flags = a.flags + int64_t(unit) * 2 * a.chunks * a.tiles;
  if (n <= keep) {
    if (tid == 0) a.moved[unit] = make_uint2(0, 0);
    return;
  }
  for (uint32_t i = tid; i < 2 * a.chunks * a.tiles; i += kThreads) flags[i] = 0;
  int32_t* const below = a.below + int64_t(unit) * (a.tiles + 1);
  for (uint32_t i = tid; i <= a.tiles; i += kThreads) below[i] = int32_t(keep);
  float* const w = a.weights + int64_t(b) * a.w_batch + int64_t(set) * a.w_set;
  const uint32_t lo = a.first, hi = n - a.recent;  // the keys to choose from
  uint32_t want = keep - a.first - a.recent;        // of them; fewer than there are

  // the lowest ordered weight that stays, and how many of those that have it
  uint32_t limit = 0xffffffffu, equal = 0;
  const bool some = want != 0;
  if (some) {
    limit = 0;
    int shift = 20, bits = 12;
    for (int digit = 0; digit < 3; ++digit) {
      const uint32_t count = 1u << bits;
      for (uint32_t i = tid; i < count; i += kThreads) bins[i] = 0;
      __syncthreads();
      const uint64_t above = uint64_t(1) << (shift + bits);  // of the digits before
      for (uint32_t i = lo + tid; i < hi; i += kThreads) {
        const uint32_t key = ordered(w[i]);
        if (((uint64_t(key) ^ uint64_t(limit)) & ~(above - 1)) == 0) count_bin(bins, (key >> shift) & (count - 1));
      }
      __syncthreads();
      limit |= find_bin(bins, count, &want, scratch, found) << shift;
      bits = digit == 0 ? 12 : 8;
      shift -= bits;
    }
    equal = want;
  }
  if (tid == 0) s_gone = n;
  __syncthreads();

  // the keys in order: the list, their weights moved down, the counts at tiles' starts
  int32_t* const list = a.list + int64_t(unit) * a.most;
  uint32_t base = 0;
  for (uint32_t i0 = 0; i0 < n; i0 += kThreads) {
    const uint32_t i = i0 + tid;
    const float x = i < n ? w[i] : 0.f;
    const uint32_t key = ordered(x);
    const bool always = i < n && (i < lo || i >= hi), may = i < n && !always && some;
    const bool sure = always || (may && key > limit), tie = may && key == limit;
    // (at most 1024 of each: two sums in one scan)
    uint32_t total;
    const uint32_t before = block_exclusive_scan<kThreads>(uint32_t(sure) | (uint32_t(tie) << 16), scratch, &total);
    const uint32_t ties = before >> 16;
    const bool stays = sure || (tie && ties < equal);
    const uint32_t at = base + (before & 0xffffu) + min(ties, equal);
    if (stays) {
      list[at] = int32_t(i);
      w[at] = x;  // places up to i, which have been read
    } else if (i < n) {
      atomicMin(&s_gone, i);
    }
    if (i < n && i % a.rows == 0 && i / a.rows <= a.tiles) below[i / a.rows] = int32_t(at);
    const uint32_t used = min(total >> 16, equal);
    base += (total & 0xffffu) + used;
    equal -= used;
  }
  __syncthreads();
  for (uint32_t i = keep + tid; i < n; i += kThreads) w[i] = 0.f;
  if (tid == 0) a.moved[unit] = make_uint2(min(s_gone, keep), keep);
}

template <int VB>
__global__ __launch_bounds__(kMove) void evict_move_kernel(const EvictArgs a) {
  typedef typename Vec<VB>::T V;
  typedef typename Vec<(VB < 4 ? 4 : VB)>::T Held;  // of it in registers
  __shared__ int64_t s_from[kMaxRows], s_to[kMaxRows];  // byte offsets; -1: a page out of range
  __shared__ uint32_t s_tile;
  const uint32_t tid = threadIdx.x;
  const uint32_t lanes = 2 * a.chunks;               // (plane, chunk) of a unit
  const uint32_t units = a.batch * a.sets * lanes;
  for (;;) {
    if (tid == 0) s_tile = atomicAdd(a.ticket, 1u);
    __syncthreads();
    const uint32_t t = uint32_t(__builtin_amdgcn_readfirstlane(int(s_tile)));
    const uint32_t tile = t / units;
    if (tile >= a.tiles) return;
    const uint32_t rest = t - tile * units, unit = rest / lanes, lane = rest - unit * lanes;
    const uint32_t plane = lane & 1, chunk = lane >> 1;
    const uint2 moved = a.moved[unit];
    const uint32_t begin = max(moved.x, tile * a.rows), end = min(moved.y, (tile + 1) * a.rows);
    if (begin >= end) {
      __syncthreads();
      continue;
    }
    const uint32_t b = unit / a.sets, set = unit - b * a.sets, rows = end - begin;
    const int32_t* list = a.list + int64_t(unit) * a.most;
    const int32_t* table = a.tables + int64_t(b) * a.table_stride;
    auto offset = [&](uint32_t key) {
      const uint32_t blk = a.block_div.div(key), page = uint32_t(table[blk]);
      if (page >= a.num_blocks) return int64_t(-1);
      return int64_t(page) * a.block_stride + int64_t(key - blk * a.block_div.d) * a.token_stride;
    };
    for (uint32_t r = tid; r < rows; r += kMove) {
      s_from[r] = offset(uint32_t(list[begin + r]));
      s_to[r] = offset(begin + r);
    }
    __syncthreads();
    const uint32_t first_piece = chunk * a.chunk_pieces, width = min(a.chunk_pieces, a.pieces_row - first_piece);
    char* const base = (plane ? a.v_base : a.k_base) + int64_t(set) * a.set_bytes + int64_t(first_piece) * VB;
    Held v[kPieces];
    int64_t to[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const uint32_t f = tid + kMove * u, r = a.chunk_div.div(f), piece = f - r * a.chunk_pieces;
      to[u] = -1;
      v[u] = Held{};
      if (r < rows && piece < width && s_from[r] >= 0 && s_to[r] >= 0) {
        v[u] = __builtin_nontemporal_load(reinterpret_cast<const V*>(base + s_from[r] + int64_t(piece) * VB));
        to[u] = s_to[r] + int64_t(piece) * VB;
      }
    }
    // the loads have come back (their values are used here), then the flag
#pragma unroll
    for (int u = 0; u < kPieces; ++u) asm volatile("" : "+v"(v[u])::"memory");
    __syncthreads();
    uint32_t* const flags = a.flags + (int64_t(unit) * lanes + lane) * a.tiles;
    if (tid == 0) {
      __hip_atomic_store(&flags[tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int32_t* below = a.below + int64_t(unit) * (a.tiles + 1) + tile;
      const int32_t from = below[0], past = below[1];  // of the list: what lies in this tile's rows
      if (past > from) {
        const uint32_t last = min(uint32_t(past - 1) / a.rows + 1, tile);
        for (uint32_t u = uint32_t(from) / a.rows; u < last; ++u)
          while (__hip_atomic_load(&flags[u], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0) __builtin_amdgcn_s_sleep(2);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
      if (to[u] >= 0) __builtin_nontemporal_store(V(v[u]), reinterpret_cast<V*>(base + to[u]));
  }
}

struct Plan {
  uint32_t most, rows, tiles, chunks, chunk_pieces;
  size_t moved, list, below, flags;
  size_t bytes() const { return moved + list + below + flags + 256; }
};

size_t padded(size_t n) { return (n + 255) & ~size_t(255); }

// `keep` < 0: lengths of their own. A piece of a row is at least a byte: the
// counts of tiles and chunks are those of the widest pieces that divide the row.
int plan_of(int64_t batch, int64_t sets, int64_t set_bytes, int64_t vec, int64_t max_len, int64_t keep, Plan* p) {
  CBK_REQUIRE(batch >= 0 && sets > 0 && batch * sets < (int64_t(1) << 31), "batch out of range");
  CBK_REQUIRE(max_len >= 0 && max_len < (int64_t(1) << 31), "context out of range");
  const int64_t pieces = set_bytes / vec, room = kMove * kPieces;
  p->most = uint32_t(keep < 0 ? max_len : std::min(keep, max_len));
  p->chunk_pieces = uint32_t(std::min(pieces, room));
  p->chunks = uint32_t((pieces + p->chunk_pieces - 1) / p->chunk_pieces);
  p->rows = uint32_t(std::min<int64_t>(room / p->chunk_pieces, kMaxRows));
  p->tiles = (p->most + p->rows - 1) / p->rows;
  const size_t units = size_t(batch) * size_t(sets);
  CBK_REQUIRE(units * 2 * p->chunks * (size_t(p->tiles) + 1) < (size_t(1) << 31), "eviction: too many tiles for one launch");
  p->moved = padded(units * sizeof(uint2));
  p->list = padded(units * p->most * sizeof(int32_t));
  p->below = padded(units * (size_t(p->tiles) + 1) * sizeof(int32_t));
  p->flags = padded(units * 2 * p->chunks * p->tiles * sizeof(uint32_t));
  return CBK_OK;
}

int vec_of(const cbk_kv_desc* kv, int64_t set_bytes) {
  const int64_t words[5] = {int64_t(reinterpret_cast<uintptr_t>(kv->k_base)), int64_t(reinterpret_cast<uintptr_t>(kv->v_base)),
                            kv->block_stride, kv->token_stride, set_bytes};
  return common_vec_bytes(words, 5);
}

int check(const cbk_kv_desc* kv, int64_t sets, int64_t first, int64_t recent, int64_t keep) {
  if (int rc = validate_desc(kv)) return rc;
  CBK_REQUIRE(sets > 0 && kv->row_bytes % sets == 0, "%lld sets of heads do not divide rows of %lld bytes", (long long)sets,
              (long long)kv->row_bytes);
  CBK_REQUIRE(kv->num_blocks < (int64_t(1) << 31), "num_blocks out of range");
  CBK_REQUIRE(first >= 0 && recent >= 0 && first + recent < (int64_t(1) << 31), "first and recent out of range");
  CBK_REQUIRE(keep < 0 || keep >= first + recent, "keep %lld is less than first and recent together", (long long)keep);
  return CBK_OK;
}

}  // namespace
}  // namespace cbk

extern "C" {

size_t cbk_paged_evict_workspace_bytes(const cbk_kv_desc* kv, int64_t table_width, int64_t batch, int64_t sets, int64_t keep) {
  using namespace cbk;
  Plan p;
  if (check(kv, sets, 0, 0, keep)) return 0;
  const int64_t set_bytes = kv->row_bytes / sets;
  if (plan_of(batch, sets, set_bytes, vec_of(kv, set_bytes), table_width * kv->block_size, keep, &p)) return 0;
  return p.bytes();
}

int cbk_paged_evict(const cbk_kv_desc* kv, const int32_t* tables_dev, int64_t table_stride, int64_t table_width,
                    const int32_t* lens_dev, int64_t batch, float* weights_dev, int64_t weights_batch_stride,
                    int64_t weights_set_stride, int64_t sets, int64_t keep, const int32_t* keeps_dev, int64_t first,
                    int64_t recent, int32_t* new_lens_dev, void* workspace_dev, size_t workspace_bytes,
                    cbk_stream_t stream) {
  using namespace cbk;
  clear_error();
  CBK_REQUIRE((keep < 0) == (keeps_dev != nullptr), "keep, or a keep for each sequence");
  if (int rc = check(kv, sets, first, recent, keep)) return rc;
  CBK_REQUIRE(table_width >= 0 && table_width < (int64_t(1) << 31) && table_stride >= 0, "block table width out of range");
  const int64_t set_bytes = kv->row_bytes / sets, max_len = table_width * kv->block_size;
  const int vec = vec_of(kv, set_bytes);
  Plan p;
  if (int rc = plan_of(batch, sets, set_bytes, vec, max_len, keep, &p)) return rc;
  if (batch == 0) return CBK_OK;
  CBK_REQUIRE(lens_dev && new_lens_dev && weights_dev && (tables_dev || table_width == 0), "NULL pointer");
  if (workspace_dev == nullptr || workspace_bytes < p.bytes())
    return set_error(CBK_ERR_WORKSPACE, "eviction workspace %zu < %zu bytes", workspace_bytes, p.bytes());
  CBK_REQUIRE((reinterpret_cast<uintptr_t>(workspace_dev) & 255) == 0, "workspace must be 256-byte aligned");
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  EvictArgs a;
  a.k_base = static_cast<char*>(kv->k_base);
  a.v_base = static_cast<char*>(kv->v_base);
  a.block_stride = kv->block_stride;
  a.token_stride = kv->token_stride;
  a.num_blocks = uint32_t(kv->num_blocks);
  a.block_div = FastDiv::make(uint32_t(kv->block_size));
  a.tables = tables_dev;
  a.table_stride = table_stride;
  a.lens = lens_dev;
  a.new_lens = new_lens_dev;
  a.weights = weights_dev;
  a.w_batch = weights_batch_stride;
  a.w_set = weights_set_stride;
  a.keeps = keeps_dev;
  a.keep = uint32_t(std::min(std::max(keep, int64_t(0)), int64_t(0x7fffffff)));
  a.first = uint32_t(first);
  a.recent = uint32_t(recent);
  a.batch = uint32_t(batch);
  a.sets = uint32_t(sets);
  a.max_len = uint32_t(max_len);
  a.most = p.most;
  a.rows = p.rows;
  a.tiles = p.tiles;
  a.chunks = p.chunks;
  a.chunk_pieces = p.chunk_pieces;
  a.pieces_row = uint32_t(set_bytes / vec);
  a.set_bytes = set_bytes;
  a.chunk_div = FastDiv::make(p.chunk_pieces);
  char* at = static_cast<char*>(workspace_dev);
  a.ticket = reinterpret_cast<uint32_t*>(at);
  a.moved = reinterpret_cast<uint2*>(at += 256);
  a.list = reinterpret_cast<int32_t*>(at += p.moved);
  a.below = reinterpret_cast<int32_t*>(at += p.list);
  a.flags = reinterpret_cast<uint32_t*>(at + p.below);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint64_t units = uint64_t(batch) * uint64_t(sets);
  hipLaunchKernelGGL(evict_choose_kernel, dim3(uint32_t(units)), dim3(kThreads), 0, s, a);
  if (int rc = launch_status("eviction's choice")) return rc;
  if (p.tiles == 0) return CBK_OK;
  const dim3 grid(uint32_t(std::min<uint64_t>(units * 2 * p.chunks * p.tiles, uint64_t(cus) * 8)));
  switch (vec) {
    case 16: hipLaunchKernelGGL((evict_move_kernel<16>), grid, dim3(kMove), 0, s, a); break;
    case 8: hipLaunchKernelGGL((evict_move_kernel<8>), grid, dim3(kMove), 0, s, a); break;
    case 4: hipLaunchKernelGGL((evict_move_kernel<4>), grid, dim3(kMove), 0, s, a); break;
    case 2: hipLaunchKernelGGL((evict_move_kernel<2>), grid, dim3(kMove), 0, s, a); break;
    default: hipLaunchKernelGGL((evict_move_kernel<1>), grid, dim3(kMove), 0, s, a); break;
  }
  return launch_status("eviction's move");
}

}  // extern "C"
