// Eviction from paged KV by the keys' accumulated weights for gfx950: of a
// sequence's keys the `first` first, the `recent` last and the heaviest of the
// others stay, `keep` together, moved to the front of its pages in their order.
//
// Two launches. A workgroup per (sequence, set of heads) chooses: the weight of
// the last key that stays is found digit by digit (11, 11 and 10 bits of the
// weights as ordered whole numbers, histograms in LDS; up to 8192 weights stay in
// LDS meanwhile, more are read again from L2), then one pass over the keys in order
// writes the list of those that stay and moves their weights. Then tiles of rows move.
//
// The rows move within their own pages, so a row must not be written before
// what lies there has been read. Row j of the list comes from a place not before
// it, so what lies in a tile's rows is read by the tile itself or by
// tiles before it, of which the choice leaves the bounds: a tile reads all of its
// rows into registers, says so in a flag, waits for the flags of the one or
// two tiles that read from its rows, and writes. A counter for each set's plane
// hands out its tiles in order: a tile only waits for tiles that were handed out
// before, to workgroups that run, and these read, and raise their flag, before they
// wait for anything; so every wait ends, whatever else the GPU does. (Only reads have to
// be done, nothing is passed on: the flags need no fences, only loads that
// have come back.) As many workgroups take a tile as there are tiles that move;
// the others that the tables and `keep` have room for end at once.
// Bound by HBM: the rows behind the first one that leaves are read and written once. A
// workgroup takes one tile and ends: one that went on to the next waited for its stores
// before it had its next loads (32 sequences of 2 K to 8 K to 4 K, 8 x 128, bf16, 0.56 GB: the
// move 217 us, 115 now, 4.85 TB/s, as a plain copy). A set's tiles turn through the XCDs, which a column of
// its own on one leaves unequal work (both kernels there 149 us, 131 turned), and take 68
// registers, so that 7 fit a SIMD (350 us with 254, to which the compiler unrolls the pieces'
// addresses). 32 KB a tile: 16 KB and 64 KB take 33.6 us for 4 sequences of 8 K to 2 K, not
// 31.5, and 47.0 and 45.7 for 32 of 8 K to 7000 for each head by itself, not 42.9.
// The choice is bound by its chain of loads and barriers: 9 us for 1 K keys, 14 for 8 K.
#include <algorithm>
#include <type_traits>

#include "cbk_common.hpp"

namespace cbk {
namespace {

constexpr int kThreads = 1024;   // of the choice
constexpr int kPass = 8192;      // keys in LDS
constexpr int kMove = 256;       // of a move
constexpr int kPieces = 8;       // a thread's pieces of a tile
constexpr uint32_t kMaxRows = 512;
constexpr uint32_t kNoSlot = 0xffffffffu;  // a page out of range
constexpr uint32_t kTicketPitch = 32;    // a counter in each cache line
constexpr uint32_t kGroups = 1u << 22;   // workgroups of a launch, at most (a grid's 2^32 threads are 2^24)

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
  uint32_t group0;  // of this launch
  FastDiv chunk_div, rows_div;
  // scratch: for each (sequence, set) the rows that move [begin, end), the list of slots [most],
  // the keys below k rows that stay [tiles + 1], and by [2 planes][chunks] the flags [tiles] and a counter
  uint2* moved;
  uint32_t* list;
  int32_t* below;
  uint32_t* flags;
  uint32_t* tickets;
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
// what is still wanted of it; by each wave for itself, so that nobody waits.
template <int BINS>
__device__ __forceinline__ uint32_t find_bin(const uint32_t* bins, uint32_t& want) {
  constexpr int PER = BINS / 64;  // lane l: bins [BINS - PER (l + 1), BINS - PER l)
  const uint32_t lane = threadIdx.x & 63;
  uint32_t sum = 0;
#pragma unroll
  for (int i = 0; i < PER; i += 4) {  // (from another place in each lane: neighbours' bins lie in the same banks)
    const Vec<16>::T n = *reinterpret_cast<const Vec<16>::T*>(&bins[BINS - PER * (lane + 1) + ((i + 4 * lane) & (PER - 1))]);
    sum += (n[0] + n[1]) + (n[2] + n[3]);
  }
  const uint32_t upto = wave_inclusive_scan(sum);
  const int at = __builtin_ctzll(__ballot(upto >= want));
  want -= uint32_t(__builtin_amdgcn_readlane(int(upto - sum), at));
  // its bins, a lane each
  static_assert(PER <= 64, "a lane a bin");
  const uint32_t top = BINS - PER * uint32_t(at) - 1;
  const uint32_t n = lane < PER ? bins[top - lane] : 0u;
  const uint32_t past = wave_inclusive_scan(n);
  const int bin = __builtin_ctzll(__ballot(past >= want));
  want -= uint32_t(__builtin_amdgcn_readlane(int(past - n), bin));
  return top - uint32_t(bin);
}

__global__ __launch_bounds__(kThreads) void evict_choose_kernel(const EvictArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t bins[3][2048];
  __shared__ float held[kPass];       // the weights of a pass's keys
  __shared__ uint32_t places[kPass];  // these as ordered numbers; then where the keys go
  __shared__ uint32_t scratch[kThreads / 64], s_gone;
  const uint32_t unit = blockIdx.x, b = unit / a.sets, set = unit - b * a.sets, tid = threadIdx.x;
  const uint32_t n = uint32_t(min(max(a.lens[b], 0), int32_t(a.max_len)));
  uint32_t keep = a.keeps ? uint32_t(max(a.keeps[b], 0)) : a.keep;
  keep = max(keep, a.first + a.recent);
  if (set == 0 && tid == 0) a.new_lens[b] = int32_t(min(n, keep));
  if (n <= keep) {
    if (tid == 0) a.moved[unit] = make_uint2(0, 0);
    return;
  }
  float* const w = a.weights + int64_t(b) * a.w_batch + int64_t(set) * a.w_set;
  const int32_t* const table = a.tables + int64_t(b) * a.table_stride;
  uint32_t page[kPass / kThreads];  // of the keys i0 + tid + k kThreads
  auto fetch = [&](uint32_t i0) {
    float x[kPass / kThreads];
#pragma unroll
    for (uint32_t k = 0; k < kPass / kThreads; ++k) {
      const uint32_t i = min(i0 + tid + k * kThreads, n - 1);
      x[k] = w[i];
      page[k] = uint32_t(table[a.block_div.div(i)]);
    }
#pragma unroll
    for (uint32_t k = 0; k < kPass / kThreads; ++k) {
      held[tid + k * kThreads] = x[k];
      places[tid + k * kThreads] = ordered(x[k]);
    }
  };
  fetch(0);
  uint32_t* const flags = a.flags + int64_t(unit) * 2 * a.chunks * a.tiles;
  for (uint32_t i = tid; i < 2 * a.chunks * a.tiles; i += kThreads) flags[i] = 0;
  for (uint32_t i = tid; i < 2 * a.chunks; i += kThreads) a.tickets[(int64_t(unit) * 2 * a.chunks + i) * kTicketPitch] = 0;
  int32_t* const below = a.below + int64_t(unit) * (a.tiles + 1);
  for (uint32_t i = tid; i <= a.tiles; i += kThreads) below[i] = int32_t(keep);
  const uint32_t lo = a.first, hi = n - a.recent;  // the keys to choose from
  uint32_t want = keep - a.first - a.recent;        // of them; fewer than there are

  // the lowest ordered weight that stays, and how many of those that have it
  uint32_t limit = 0xffffffffu, equal = 0;
  const bool some = want != 0;
  for (uint32_t i = tid; i < 3 * 2048; i += kThreads) bins[0][i] = 0;
  if (tid == 0) s_gone = n;
  __syncthreads();
  if (some) {
    limit = 0;
    auto digit = [&](auto top, auto width, uint32_t* counts) {  // bits [top - width, top) of those alike above
      constexpr int T = decltype(top)::value, W = decltype(width)::value;
      for (uint32_t i0 = 0; i0 < n; i0 += kPass) {
        if (n > kPass) {
          __syncthreads();
          fetch(i0);
          __syncthreads();
        }
        const uint32_t past = min(hi, i0 + uint32_t(kPass));
        for (uint32_t j = tid; i0 + j < past; j += 4 * kThreads) {
          uint32_t key[4];
#pragma unroll
          for (uint32_t u = 0; u < 4; ++u) key[u] = places[(j + u * kThreads) % kPass];
#pragma unroll
          for (uint32_t u = 0; u < 4; ++u) {
            const uint32_t i = i0 + j + u * kThreads;
            const bool alike = T == 32 || ((key[u] ^ limit) >> (T & 31)) == 0;
            if (i >= lo && i < past && alike) count_bin(counts, (key[u] >> (T - W)) & ((1u << W) - 1));
          }
        }
      }
      __syncthreads();
      limit |= find_bin<(1 << W)>(counts, want) << (T - W);
    };
    digit(std::integral_constant<int, 32>(), std::integral_constant<int, 11>(), bins[0]);
    digit(std::integral_constant<int, 21>(), std::integral_constant<int, 11>(), bins[1]);
    digit(std::integral_constant<int, 10>(), std::integral_constant<int, 10>(), bins[2]);
    equal = want;
  }

  // the keys in order: the list of their slots, their weights moved down, the counts at tiles' starts
  uint32_t* const list = a.list + int64_t(unit) * a.most;
  uint32_t base = 0;
  for (uint32_t i0 = 0; i0 < n; i0 += kPass) {
    if (n > kPass) {
      __syncthreads();
      fetch(i0);
      __syncthreads();
    }
    const uint32_t count = min(n - i0, uint32_t(kPass));
    // a thread's neighbours (an odd number: they lie in different banks)
    const uint32_t per = ((count + kThreads - 1) / kThreads) | 1u, from = tid * per, past = min(from + per, count);
    uint32_t kinds = 0, both = 0;  // two bits a key (1: stays, 2: has the lowest weight); counts of the two
    static_assert(kPass / kThreads <= 8, "nine keys at most, two bits each");
    for (uint32_t k = 0; k < per; k += 3) {
#pragma unroll
      for (uint32_t u = 0; u < 3; ++u) {
        const uint32_t j = from + k + u, i = i0 + j, key = places[j % kPass];
        uint32_t is = !some || key < limit ? 0u : key > limit ? 1u : 2u;
        if (i < lo || i >= hi) is = 1u;
        if (k + u >= per || j >= count) is = 0u;
        kinds |= is << (2 * (k + u));
        both += (is & 1u) | (is >> 1 << 16);
      }
    }
    uint32_t total;
    const uint32_t before = block_exclusive_scan<kThreads>(both, scratch, &total);
    uint32_t ties = before >> 16, at = base + (before & 0xffffu) + min(ties, equal), gone = n;
    for (uint32_t k = from; k < past; ++k, kinds >>= 2) {
      const uint32_t i = i0 + k, t = a.rows_div.div(i), is = kinds & 3u;
      if (t * a.rows == i && t <= a.tiles) below[t] = int32_t(at);
      const bool stays = is == 1u || (is == 2u && ties < equal);
      places[k] = stays ? at : kNoSlot;
      if (!stays) gone = min(gone, i);
      at += stays;
      ties += is >> 1;
    }
    // the first lane that has one that leaves has the wave's first
    const uint64_t leave = __ballot(gone < n);
    if (leave && int(tid & 63) == __builtin_ctzll(leave)) atomicMin(&s_gone, gone);
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kPass / kThreads; ++k) {
      const uint32_t j = tid + k * kThreads, i = i0 + j;
      if (j >= count) break;
      const uint32_t to = places[j], blk = a.block_div.div(i);
      if (to != kNoSlot) {
        list[to] = page[k] < a.num_blocks ? page[k] * a.block_div.d + (i - blk * a.block_div.d) : kNoSlot;
        w[to] = held[j];  // places up to i: they are in LDS by now
      }
      if (i >= keep) w[i] = 0.f;
    }
    const uint32_t used = min(total >> 16, equal);
    base += (total & 0xffffu) + used;
    equal -= used;
  }
  if (tid == 0) a.moved[unit] = make_uint2(min(s_gone, keep), keep);
}

template <int VB>
__global__ __launch_bounds__(kMove, 4) void evict_move_kernel(const EvictArgs a) {
  typedef typename Vec<VB>::T V;
  typedef typename Vec<(VB < 4 ? 4 : VB)>::T Held;  // of it in registers
  __shared__ int64_t s_from[kMaxRows], s_to[kMaxRows];  // byte offsets; -1: does not move
  __shared__ uint32_t s_ticket;
  const uint32_t tid = threadIdx.x;
  // all units' first tiles, their second ones, ..
  const uint32_t lanes = 2 * a.chunks;  // (plane, chunk) of a unit
  const uint32_t group = a.group0 + blockIdx.x, columns = a.batch * a.sets * lanes;
  const uint32_t turn = group / columns, column = (group + turn) % columns;  // (its tiles on all XCDs)
  const uint32_t unit = column / lanes, lane = column - unit * lanes;
  const uint2 moved = a.moved[unit];
  if (moved.x >= moved.y) return;
  const uint32_t first_tile = a.rows_div.div(moved.x);
  if (turn > a.rows_div.div(moved.y - 1) - first_tile) return;  // the others are as many as the tiles
  if (tid == 0) s_ticket = atomicAdd(&a.tickets[int64_t(column) * kTicketPitch], 1u);
  __syncthreads();
  const uint32_t tile = first_tile + uint32_t(__builtin_amdgcn_readfirstlane(int(s_ticket)));
  const uint32_t plane = lane & 1, chunk = lane >> 1;
  const uint32_t b = unit / a.sets, set = unit - b * a.sets, row0 = tile * a.rows;
  // (loads that do not wait for each other)
  const int32_t* below = a.below + int64_t(unit) * (a.tiles + 1) + tile;
  const int32_t first_below = below[0], past_below = below[1];  // of the list: what lies in this tile's rows
  const uint32_t* list = a.list + int64_t(unit) * a.most;
  const int32_t* table = a.tables + int64_t(b) * a.table_stride;
  for (uint32_t r = tid; r < a.rows; r += kMove) {
    const uint32_t key = min(row0 + r, a.most - 1), blk = a.block_div.div(key);
    const uint32_t slot = list[key], page = uint32_t(table[blk]);
    const bool moves = row0 + r >= moved.x && row0 + r < moved.y && slot != kNoSlot && page < a.num_blocks;
    const uint32_t from = a.block_div.div(slot);
    s_from[r] = moves ? int64_t(from) * a.block_stride + int64_t(slot - from * a.block_div.d) * a.token_stride : -1;
    s_to[r] = int64_t(page) * a.block_stride + int64_t(key - blk * a.block_div.d) * a.token_stride;
  }
  __syncthreads();
  const uint32_t first_piece = chunk * a.chunk_pieces, width = min(a.chunk_pieces, a.pieces_row - first_piece);
  char* const base = (plane ? a.v_base : a.k_base) + int64_t(set) * a.set_bytes + int64_t(first_piece) * VB;
  Held v[kPieces];
  // piece u of this thread, of row r; whether it moves
  auto place = [&](int u, uint32_t& r, uint32_t& piece) __attribute__((always_inline)) {
    const uint32_t f = tid + kMove * u;
    r = a.chunk_div.div(f);
    piece = f - r * a.chunk_pieces;
    return r < a.rows && piece < width && s_from[r] >= 0;
  };
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    uint32_t r, piece;
    v[u] = Held{};
    if (place(u, r, piece))
      v[u] = __builtin_nontemporal_load(reinterpret_cast<const V*>(base + s_from[r] + int64_t(piece) * VB));
  }
  // the loads have come back (their values are used here), then the flag
#pragma unroll
  for (int u = 0; u < kPieces; ++u) asm volatile("" : "+v"(v[u])::"memory");
  __syncthreads();
  uint32_t* const flags = a.flags + (int64_t(unit) * lanes + lane) * a.tiles;
  if (tid == 0) {
    __hip_atomic_store(&flags[tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (past_below > first_below) {
      const uint32_t last = min(a.rows_div.div(uint32_t(past_below - 1)) + 1, tile);
      for (uint32_t u = a.rows_div.div(uint32_t(first_below)); u < last; ++u)
        while (__hip_atomic_load(&flags[u], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0) __builtin_amdgcn_s_sleep(2);
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    uint32_t r, piece;
    if (place(u, r, piece)) __builtin_nontemporal_store(V(v[u]), reinterpret_cast<V*>(base + s_to[r] + int64_t(piece) * VB));
  }
}

struct Plan {
  uint32_t most, rows, tiles, chunks, chunk_pieces;
  size_t moved, list, below, flags, tickets;
  size_t bytes() const { return moved + list + below + flags + tickets; }
};

size_t padded(size_t n) { return (n + 255) & ~size_t(255); }

// `keep` < 0: lengths of their own. A piece of a row is at least a byte: the
// counts of tiles and chunks are those of the widest pieces that divide the row.
int plan_of(int64_t batch, int64_t sets, int64_t set_bytes, int64_t vec, int64_t max_len, int64_t keep, Plan* p) {
  CBK_REQUIRE(batch >= 0 && sets > 0 && batch < (1 << 22) && batch * sets < (1 << 22), "batch out of range");
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
  p->list = padded(units * p->most * sizeof(uint32_t));
  p->below = padded(units * (size_t(p->tiles) + 1) * sizeof(int32_t));
  p->flags = padded(units * 2 * p->chunks * p->tiles * sizeof(uint32_t));
  p->tickets = units * 2 * p->chunks * kTicketPitch * sizeof(uint32_t);
  return CBK_OK;
}

int vec_of(const cbk_kv_desc* kv, int64_t set_bytes) {
  const int64_t words[5] = {int64_t(reinterpret_cast<uintptr_t>(kv->k_base)), int64_t(reinterpret_cast<uintptr_t>(kv->v_base)),
                            kv->block_stride, kv->token_stride, set_bytes};
  return common_vec_bytes(words, 5);
}

bool apart(const int32_t* x, const int32_t* y, int64_t n) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
  return (a > b ? a - b : b - a) >= uintptr_t(n) * sizeof(int32_t);
}

int check(const cbk_kv_desc* kv, int64_t sets, int64_t first, int64_t recent, int64_t keep) {
  if (int rc = validate_desc(kv)) return rc;
  // (a plane's tiles do not wait for the other's)
  const intptr_t apart = static_cast<const char*>(kv->v_base) - static_cast<const char*>(kv->k_base);
  CBK_REQUIRE((apart < 0 ? -apart : apart) >= kv->row_bytes, "keys and values in the same rows");
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
  // (a sequence's sets read its length and keep by themselves, and the first writes the new length)
  CBK_REQUIRE(apart(new_lens_dev, lens_dev, batch) && (!keeps_dev || apart(new_lens_dev, keeps_dev, batch)),
              "new lengths over the lengths or keeps");
  if (workspace_dev == nullptr || workspace_bytes < p.bytes())
    return set_error(CBK_ERR_WORKSPACE, "eviction workspace %zu < %zu bytes", workspace_bytes, p.bytes());
  CBK_REQUIRE((reinterpret_cast<uintptr_t>(workspace_dev) & 255) == 0, "workspace must be 256-byte aligned");
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
  a.rows_div = FastDiv::make(p.rows);
  char* at = static_cast<char*>(workspace_dev);
  a.tickets = reinterpret_cast<uint32_t*>(at);
  a.moved = reinterpret_cast<uint2*>(at += p.tickets);
  a.list = reinterpret_cast<uint32_t*>(at += p.moved);
  a.below = reinterpret_cast<int32_t*>(at += p.list);
  a.flags = reinterpret_cast<uint32_t*>(at + p.below);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint64_t units = uint64_t(batch) * uint64_t(sets);
  hipLaunchKernelGGL(evict_choose_kernel, dim3(uint32_t(units)), dim3(kThreads), 0, s, a);
  if (int rc = launch_status("eviction's choice")) return rc;
  if (p.tiles == 0) return CBK_OK;
  const uint32_t all = uint32_t(units * 2 * p.chunks * p.tiles);  // < 2^31
  for (a.group0 = 0; a.group0 < all; a.group0 += kGroups) {
    const dim3 grid(std::min(all - a.group0, kGroups));
    switch (vec) {
      case 16: hipLaunchKernelGGL((evict_move_kernel<16>), grid, dim3(kMove), 0, s, a); break;
      case 8: hipLaunchKernelGGL((evict_move_kernel<8>), grid, dim3(kMove), 0, s, a); break;
      case 4: hipLaunchKernelGGL((evict_move_kernel<4>), grid, dim3(kMove), 0, s, a); break;
      case 2: hipLaunchKernelGGL((evict_move_kernel<2>), grid, dim3(kMove), 0, s, a); break;
      default: hipLaunchKernelGGL((evict_move_kernel<1>), grid, dim3(kMove), 0, s, a); break;
    }
    if (int rc = launch_status("eviction's move")) return rc;
  }
  return CBK_OK;
}

}  // extern "C"
