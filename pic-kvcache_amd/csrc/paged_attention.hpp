// Attention of a sequence's latest tokens over its context in pages of the
// queries' type for gfx950, and each key's attention weight summed over the rows:
//
//   p[b, r, h, k] = softmax_k( scale q[b, r, h] . key[k, h / G] )
//   out[b, r, h]  = sum_k p[b, r, h, k] value[k, h / G]
//   weights[b, m, k] += sum over r and the heads h of set m of p[b, r, h, k]
//
// over keys k <= len_b - R + r of sequence b (row r of its R rows is the
// token at that place), G = Hq / Hkv; a set is a KV head's G heads, or all heads.
//
// Bound by HBM: each key and value row is read once for up to 32 rows of a group
// (more are 32-row tiles, each of which reads it, and bound by their dependences).
// Beside that the matrix cores and the VALU have little to do (a 32-key tile of
// a KV head, 16 KB, is 24 MFMAs and some 250 VALU instructions for up to 16
// rows, a tenth of the time its bytes take), so the kernel is laid out for loads
// in flight and nothing else: a wave takes a tile of one KV head at a time straight
// into registers, K and V of the next tile requested before this one's are waited for,
// no LDS and no barrier on the way. 64 sequences of 4 K to 16 K keys, 32 heads over 8 x
// 128, bf16, 2.6 GB: 396 us, 6.6 TB/s (what a 4 GiB copy moves: 4.9).
//  - S^T = K . Q^T: lane (j = lane / 16, c) reads 16 bytes of key c's row, dims
//    32 st + 8 j .., which is an operand of step st as it is.
//  - O = P . V: S^T leaves lane (j, c) with keys 4 j .. 4 j + 3 of each 16-key
//    half for row c, which is the first operand as it is. For the second the lane
//    reads the same keys' rows, dims D / 16 c ..: an operand wants 8 keys of
//    one dim, and which dim is column c of which product is free, so a column takes
//    the lane's own dims one after another and 32 in-lane byte permutes turn the
//    lane's 8 keys x 8 dims. float32: 16-key tiles, four 16x16x4 products where
//    16 bits have one 16x16x32, the same lanes' keys and no permutes.
// 16-bit weights enter the second product in two parts, so they are held to 2^-16
// (bf16) or 2^-22 (float16) of themselves (below 2^-8 of the largest, float16: 2^-30 of
// that); sums and statistics are float32.
// The waits for loads are the compiler's counts of what was requested later, which only
// straight code keeps exact: so a step behind the last loads too (nothing, or a row that
// is there), and pages in whole 16-key pieces (FAST) are addressed by scalars, for
// vector registers that hold an address now and a tile's rows then are waited for
// (64 x 16 K: 451 us; 397 with both, and the caches passed by).
//
// The batch's tiles are cut into equal ranges (paged_ranges.hpp); a workgroup
// takes one, a wave a KV head, or several waves a head's tiles in turns. A
// sequence that one range holds whole is written at once, the others' partial
// results are merged by a second launch. For the keys' weights the waves leave
// the logits in scratch (4 bytes a row and key, beside 4 D or 8 D bytes a key that
// they read), and the second launch turns them into weights with the rows'
// statistics, or, for sets of many rows, a third one does.
#pragma once

#include <type_traits>

#include "paged_ranges.hpp"

namespace cbk {

struct PagedAttnArgs {
  const char* q;
  char* out;
  int64_t q_batch, q_row, q_head;        // bytes
  int64_t out_batch, out_row, out_head;
  const char* k_base;
  const char* v_base;
  int64_t block_stride, token_stride;    // bytes
  const int32_t* tables;
  int64_t table_stride;                  // entries
  const int32_t* lens;
  uint32_t batch, rows, hq, hkv, group;  // rows: of a sequence
  uint32_t num_blocks, max_len, max_tiles;
  uint32_t row_tiles;                    // of (row, head of the group) pairs
  uint32_t ranges;
  uint32_t rt;                           // 16-row tiles of a wave
  bool fast;                             // 16 keys are one piece of a page
  bool stream;                           // the pages are more than the last cache level holds
  bool whole;                            // range r is sequence r, and no partial results
  uint32_t heads, turns;                 // of a workgroup: KV heads, and waves that share one's tiles
  float c;                               // scale log2 e / kUnit
  FastDiv block_div;
  // partial results of range r's unfinished sequence that began before it (0), and
  // of the one that begins in it (1): entry ((2 r + which) hkv + kv head) * rows * group + row * group + head
  float2* ml;
  float* o;
  // for the keys' weights: the rows' statistics, (b hkv + kv head) * rows * group
  // + ..; the logits [b][tile][kv head][row, head][key of the tile]
  float2* stats;
  float* logits;
  float* weights;
  int64_t w_batch, w_set;                // elements
  uint32_t w_sets;
};

// The launches of one type (in a source each), head_dim 64 or 128.
int launch_paged_attention_bf16(const PagedAttnArgs& a, int64_t head_dim, hipStream_t s);
int launch_paged_attention_f16(const PagedAttnArgs& a, int64_t head_dim, hipStream_t s);
int launch_paged_attention_f32(const PagedAttnArgs& a, int64_t head_dim, hipStream_t s);

// Ranges are cut in places: a sequence has one for each tile, and kHead before
// them, for what a workgroup does at a sequence's start and end. (us with 0 / 1 / 2 / 4, bf16,
// 128: 9 sequences of up to 3 K, 4 rows of 40 heads over 8, 26.2 / 24.3 / 24.3 / 24.5; 8 of 4 K, 32
// heads over 8, 25.5 / 23.5 / 23.7 / 23.6; 64 of 16 K 397 / 397 / 397 / 400.)
constexpr uint32_t kHead = 1;

// waves of a workgroup, at most: two a SIMD; one where two row tiles take its registers
constexpr int max_waves(int rt) { return rt == 1 ? 8 : 4; }

namespace {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
// Logits are held in units of 4 log 2: float32's largest logit times log2 e is
// past its range, a quarter of that is not.
constexpr float kUnit = 4.f;
constexpr float kRescale = 8.f / kUnit;  // headroom before the reference maximum is raised

// 16 and 8 bytes at any element's address
template <int ES> struct Piece;
template <> struct Piece<2> {
  typedef u32x4 V16 __attribute__((aligned(2)));
  typedef u32x2 V8 __attribute__((aligned(2)));
};
template <> struct Piece<4> {
  typedef u32x4 V16 __attribute__((aligned(4)));
  typedef u32x2 V8 __attribute__((aligned(4)));
};

typedef const __attribute__((address_space(4))) int32_t* Const32;  // read by scalar loads
constexpr int kBufferWord = 0x00027000;  // of a buffer's descriptor: bytes, 32-bit data

// What differs between the types. KEYS: of a tile; kWeights: log2 of a weight at the
// reference maximum. 2^-18: a weight is 2^-10 at most, so that sums of 1000 of the
// type's largest values stay within float32. float16's values need no such room,
// its weights all the precision that 2^14 at most leaves below.
template <int DT> struct Type;
template <> struct Type<CBK_DTYPE_BF16> {
  static constexpr int ES = 2, KEYS = 32;
  static constexpr float kWeights = -18.f;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(s16x8, a), __builtin_bit_cast(s16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, b2));
  }
  static __device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  static constexpr uint32_t kExponent = 0x7f80u;
};
template <> struct Type<CBK_DTYPE_F16> {
  static constexpr int ES = 2, KEYS = 32;
  static constexpr float kWeights = 6.f;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (h2){_Float16(x), _Float16(y)});
  }
  static __device__ __forceinline__ float low(uint32_t w) { return float(__builtin_bit_cast(_Float16, uint16_t(w))); }
  static __device__ __forceinline__ float high(uint32_t w) { return float(__builtin_bit_cast(_Float16, uint16_t(w >> 16))); }
  static constexpr uint32_t kExponent = 0x7c00u;
};
template <> struct Type<CBK_DTYPE_F32> {
  static constexpr int ES = 4, KEYS = 16;
  static constexpr float kWeights = -18.f;
};

__device__ __forceinline__ uint32_t context_of(const PagedAttnArgs& a, uint32_t b) {
  return uint32_t(min(max(a.lens[b], 0), int32_t(a.max_len)));
}
template <int KEYS> __device__ __forceinline__ uint32_t tiles_of(uint32_t len) { return (len + KEYS - 1) / KEYS; }
template <int KEYS> __device__ __forceinline__ uint32_t places_of(uint32_t len) { return len ? kHead + tiles_of<KEYS>(len) : 0u; }

__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// What turns a row's logits into weights: the reference maximum (0 without one), 1 / sum.
__device__ __forceinline__ float2 statistics(float m, float l) {
  return make_float2(m == kNegInf ? 0.f : m, l == 0.f ? 0.f : 1.f / l);
}

// N values of a row, rounded to the type
template <int DT, int N>
__device__ __forceinline__ void store_row(char* p, const float (&x)[N]) {
  if constexpr (DT == CBK_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < N; e += 4)
      *reinterpret_cast<Piece<4>::V16*>(p + 4 * e) =
          u32x4{__float_as_uint(x[e]), __float_as_uint(x[e + 1]), __float_as_uint(x[e + 2]), __float_as_uint(x[e + 3])};
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int e = 0; e < N / 2; ++e) w[e] = Type<DT>::pack(x[2 * e], x[2 * e + 1]);
    if constexpr (N == 8) *reinterpret_cast<Piece<2>::V16*>(p) = u32x4{w[0], w[1], w[2], w[3]};
    else *reinterpret_cast<Piece<2>::V8*>(p) = u32x2{w[0], w[1]};
  }
}

// K and V of a tile as a lane holds them. K: piece [h][st] is key 16 h + c, bytes
// 64 st + 16 j .. of its row. V: key 4 j + e % 4 + 16 (e / 4), bytes D / 16 ES c ..
// (float32: dims 64 i + 4 c ..).
template <int DT, int D> struct Tile {
  static constexpr int ES = Type<DT>::ES, HALVES = Type<DT>::KEYS / 16;
  static constexpr int KP = D * ES / 64;                // pieces of a K row in a lane
  static constexpr int VK = 4 * HALVES;                 // keys of V in a lane
  static constexpr int VW = D / 16 * ES / 4;            // words of a V row in a lane
  u32x4 k[HALVES][KP];
  uint32_t v[VK][VW];
};

// MODE 0: any pages. 1 and 2 (FAST): blocks of a multiple of 16 tokens, 16-byte aligned:
// 16 keys are one piece of a page, whose address is uniform, the lanes' offsets in it
// the same for every tile. 2: loads that leave nothing in the caches.
template <int DT, int D, int RT, bool LOGITS, int MODE>
__global__ __launch_bounds__(64 * max_waves(RT), 1) void paged_attn_kernel(const PagedAttnArgs a) {
  using T = Type<DT>;
  using Tl = Tile<DT, D>;
  constexpr int KEYS = T::KEYS, H = Tl::HALVES, NT = D / 16;  // NT: 16-column tiles of the output
  constexpr int ROWS = 16 * RT;
  constexpr bool F32 = DT == CBK_DTYPE_F32;
  constexpr bool FAST = MODE != 0;
  constexpr int kOnce = MODE == 2 ? 2 : 0;  // a buffer load's bits: non-temporal
  constexpr uint32_t kAll = KEYS == 32 ? 0xffffffffu : 0xffffu;
  // A wave's: several waves of a head, their results of 16 rows [row][D], then each row's
  // m and l; before that, its tiles' logits on their way to memory.
  constexpr int kLds = LOGITS ? 160 * 1024 / 4 / max_waves(RT) : 16 * D + 32;
  __shared__ __attribute__((aligned(16))) float lds[max_waves(RT)][kLds];

  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t j = lane >> 4, c = lane & 15;
  // a range's workgroups on one XCD, one after another: a token's row is one piece of
  // memory for all heads
  const uint32_t units = a.hkv / a.heads * a.row_tiles;
  const uint32_t place_in = blockIdx.x >> 3;
  const uint32_t range = __builtin_amdgcn_readfirstlane((place_in / units) * 8 + (blockIdx.x & 7));
  if (range >= a.ranges) return;
  const uint32_t unit = __builtin_amdgcn_readfirstlane(place_in % units);
  const uint32_t head0 = unit / a.row_tiles * a.heads, row_tile = unit % a.row_tiles;  // the workgroup's
  const uint32_t turn = __builtin_amdgcn_readfirstlane(wave / a.heads), turns = a.turns;
  const uint32_t kvh = head0 + (wave - turn * a.heads);
  const uint32_t head_rows = a.rows * a.group;

  // the lengths of the first 64 sequences, a lane each
  const uint32_t len0 = a.whole ? context_of(a, range) : lane < a.batch ? context_of(a, lane) : 0u;
  auto length = [&](uint32_t s) __attribute__((always_inline)) {
    return s < 64 ? uint32_t(__builtin_amdgcn_readlane(int(len0), int(s))) : context_of(a, s);
  };
  uint32_t at = 0, end = 0, seq = 0, before = 0;  // the range, the sequence that holds place `at`, the places before it
  if (a.whole) {
    seq = range;
  } else {
    const uint32_t places0 = places_of<KEYS>(len0);
    uint32_t all = places0;
    for (uint32_t b = lane + 64; b < a.batch; b += 64) all += places_of<KEYS>(context_of(a, b));
    const Ranges cut(wave_total(all), a.ranges);
    at = cut.first(range);
    end = cut.first(range + 1);
    if (at == end) return;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
      uint32_t n = places0;
      if (b0 > 0) n = b0 + lane < a.batch ? places_of<KEYS>(context_of(a, b0 + lane)) : 0u;
      const uint32_t upto = before + wave_inclusive_scan(n);
      const uint64_t past = __ballot(upto > at);
      if (past) {
        const int first = __builtin_ctzll(past);
        seq = b0 + uint32_t(first);
        before = uint32_t(__builtin_amdgcn_readlane(int(upto - n), first));
        break;
      }
      before = uint32_t(__builtin_amdgcn_readlane(int(upto), 63));
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
  }

  const uint32_t k_off = FAST ? c * uint32_t(a.token_stride) + 16 * j : 0u;
  const uint32_t v_off = FAST ? 4 * j * uint32_t(a.token_stride) + (F32 ? 16 : D / 16 * T::ES) * c : 0u;
  // row tile t's row of this lane's column c of S^T
  uint32_t q_r[RT], q_h[RT];
  bool live[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const uint32_t n = row_tile * ROWS + 16 * t + c;
    live[t] = n < head_rows;
    q_r[t] = live[t] ? n / a.group : 0;
    q_h[t] = kvh * a.group + (live[t] ? n - q_r[t] * a.group : 0);
  }

  for (;; ++seq) {
    // the sequence's tiles [from, to) in the range
    const uint32_t len = uint32_t(__builtin_amdgcn_readfirstlane(int(a.whole ? len0 : length(seq))));
    uint32_t from = 0, to = tiles_of<KEYS>(len);
    if (!a.whole) {
      const uint32_t start = before + kHead;
      before += places_of<KEYS>(len);
      from = at > start ? at - start : 0u;
      to = min(to, end > start ? end - start : 0u);
      if (from >= to) {  // an empty sequence, or its head alone
        if (before >= end) break;
        continue;
      }
    }
    const bool whole = from == 0 && to == tiles_of<KEYS>(len);
    // of a range's two unfinished sequences at most, the one that began before it, or in it
    const uint32_t which = from > 0 ? 0u : 1u;
    const uint32_t tile0 = from + turn;  // the wave's first tile
    const int32_t count = to > tile0 ? int32_t((to - tile0 + turns - 1) / turns) : 0;
    const int32_t* table = a.tables + int64_t(seq) * a.table_stride;
    int32_t last_key[RT];  // a row sees keys up to it
#pragma unroll
    for (int t = 0; t < RT; ++t) last_key[t] = live[t] ? int32_t(len) - int32_t(a.rows) + int32_t(q_r[t]) : -1;

    // Q, zero in columns without a row
    u32x4 qf[RT][Tl::KP];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const char* p = a.q + int64_t(seq) * a.q_batch + int64_t(q_r[t]) * a.q_row + int64_t(q_h[t]) * a.q_head + 16 * j;
#pragma unroll
      for (int s = 0; s < Tl::KP; ++s) {
        qf[t][s] = u32x4(0u);
        if (live[t]) qf[t][s] = *reinterpret_cast<const typename Piece<T::ES>::V16*>(p + 64 * s);
      }
    }

    // The block table's entries of a step: of its tile's 16-key halves, or of this
    // lane's key (a tile's keys, one a lane).
    struct Pages {
      uint32_t page[FAST ? H : 1];
    };
    auto fetch = [&](int32_t i) __attribute__((always_inline)) {
      Pages g;
      const uint32_t key0 = (tile0 + turns * uint32_t(i)) * KEYS;
      if constexpr (FAST) {
        const Const32 entries = Const32(reinterpret_cast<uintptr_t>(table));
#pragma unroll
        for (int h = 0; h < H; ++h) g.page[h] = uint32_t(entries[a.block_div.div(min(key0 + 16 * h, len - 1))]);
      } else {
        g.page[0] = uint32_t(table[a.block_div.div(min(key0 + (lane & (KEYS - 1)), len - 1))]);
      }
      return g;
    };
    // The tile's rows; bits of the keys that there are. FAST: halves without any
    // load nothing. Otherwise keys past the context or in a page out of range are read
    // from the wave's first row, as is the step behind the last: every step has the
    // same loads after it, and none waits for more than its own. (The first row of
    // the cache instead, for all waves at the same time: 4 us at the end of a call.)
    const char* const k_base = a.k_base + int64_t(kvh) * (D * T::ES);
    const char* const v_base = a.v_base + int64_t(kvh) * (D * T::ES);
    uint64_t spare = 0;
    auto load = [&](int32_t i, const Pages& g, Tl& to) __attribute__((always_inline)) {
      const uint32_t key0 = (tile0 + turns * uint32_t(i)) * KEYS;
      if constexpr (FAST) {
        const uint32_t left = i < count ? len - key0 : 0u;
        uint32_t here = left >= uint32_t(KEYS) ? kAll : (1u << left) - 1u;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const uint32_t key = key0 + 16 * h, blk = a.block_div.div(key);
          const bool held = key0 + 16 * h < key0 + left && g.page[h] < a.num_blocks;
          if (!held) here &= ~(0xffffu << (16 * h));
          const int64_t at = held ? int64_t(g.page[h]) * a.block_stride + int64_t(key - blk * a.block_div.d) * a.token_stride : 0;
          const int span = held ? int(15 * a.token_stride) + D * T::ES : 0;  // 0: the loads return zeros
          const auto kr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(k_base + at), 0, span, kBufferWord);
          const auto vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(v_base + at), 0, span, kBufferWord);
#pragma unroll
          for (int s = 0; s < Tl::KP; ++s) to.k[h][s] = __builtin_amdgcn_raw_buffer_load_b128(kr, int(k_off), 64 * s, kOnce);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            uint32_t(&v)[Tl::VW] = to.v[4 * h + r];
            const int row = r * int(a.token_stride);
            if constexpr (F32) {
#pragma unroll
              for (int i4 = 0; i4 < D / 64; ++i4) {
                const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(vr, int(v_off) + 256 * i4, row, kOnce);
#pragma unroll
                for (int x = 0; x < 4; ++x) v[4 * i4 + x] = w[x];
              }
            } else if constexpr (Tl::VW == 4) {
              const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(vr, int(v_off), row, kOnce);
#pragma unroll
              for (int x = 0; x < 4; ++x) v[x] = w[x];
            } else {
              const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(vr, int(v_off), row, kOnce);
              v[0] = w[0];
              v[1] = w[1];
            }
          }
        }
        return here;
      } else {
        const uint32_t key = key0 + (lane & (KEYS - 1));
        const bool held = i < count && key < len && g.page[0] < a.num_blocks;
        uint64_t row = spare;
        if (held) {
          const uint32_t blk = a.block_div.div(key);
          row = uint64_t(g.page[0]) * uint64_t(a.block_stride) + uint64_t(key - blk * a.block_div.d) * uint64_t(a.token_stride);
        }
        if (i == 0)
          spare = (uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(row >> 32))))) << 32) |
                  uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(row))));
        auto row_of = [&](uint32_t from) __attribute__((always_inline)) {
          return uint64_t(uint32_t(__shfl(int(uint32_t(row)), int(from)))) |
                 (uint64_t(uint32_t(__shfl(int(uint32_t(row >> 32)), int(from)))) << 32);
        };
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const char* p = k_base + 16 * j + row_of(16 * h + c);
#pragma unroll
          for (int s = 0; s < Tl::KP; ++s) to.k[h][s] = *reinterpret_cast<const typename Piece<T::ES>::V16*>(p + 64 * s);
        }
#pragma unroll
        for (int e = 0; e < Tl::VK; ++e) {
          const char* p = v_base + row_of(4 * j + (e & 3) + 16 * (e >> 2));
          if constexpr (F32) {
#pragma unroll
            for (int i4 = 0; i4 < D / 64; ++i4) {
              const u32x4 w = *reinterpret_cast<const Piece<4>::V16*>(p + 256 * i4 + 16 * c);
#pragma unroll
              for (int x = 0; x < 4; ++x) to.v[e][4 * i4 + x] = w[x];
            }
          } else if constexpr (Tl::VW == 4) {
            const u32x4 w = *reinterpret_cast<const Piece<2>::V16*>(p + 16 * c);
#pragma unroll
            for (int x = 0; x < 4; ++x) to.v[e][x] = w[x];
          } else {
            const u32x2 w = *reinterpret_cast<const Piece<2>::V8*>(p + 8 * c);
            to.v[e][0] = w[0];
            to.v[e][1] = w[1];
          }
        }
        return uint32_t(__ballot(held)) & kAll;
      }
    };

    float m[RT], l[RT];  // of the lane's column: reference maximum, sum of the lane's keys
    f32x4 o[RT][NT];     // rows 4 j + i of the row tile, column c of tile n: dim NT c + n (float32: 64 (n / 4) + 4 c + n % 4)
    // 16 bits: an infinite value's products with a weight's two parts, of which the second
    // may be negative or 0, have no sum. So where an output is not finite the wave takes its
    // tiles a second time, such values one by one, by the whole weight. (0.3 us a call for
    // the look at the outputs; at every tile's values it would be over 100 VALU instructions
    // beside 250.)
    bool careful = false;

    // The logits of the wave's tiles wait in LDS and leave it together: written tile by
    // tile they break up the reads of all memory channels (64 sequences of 4 K to 16 K
    // keys, 3% of the bytes: 555 us, 400 without them; the whole call 586, 515 so).
    float* const stage = lds[wave];
    const uint32_t stage_floats = min(head_rows - row_tile * ROWS, uint32_t(ROWS)) * KEYS, stage_room = kLds / stage_floats;
    uint32_t staged = 0;
    auto flush = [&](int32_t i) __attribute__((always_inline)) {  // tiles i - staged .. i - 1 of the wave
      float* const to = a.logits + ((int64_t(seq) * a.max_tiles + tile0) * a.hkv + kvh) * int64_t(head_rows * KEYS) + row_tile * ROWS * KEYS;
      const uint32_t pieces = stage_floats / 4;
      for (uint32_t e = lane; e < staged * pieces; e += 64) {
        const uint32_t s = e / pieces, piece = e - s * pieces;
        const f32x4 w = *reinterpret_cast<const f32x4*>(stage + s * stage_floats + 4 * piece);
        *reinterpret_cast<f32x4*>(to + int64_t(turns * (uint32_t(i) - staged + s)) * a.hkv * int64_t(head_rows * KEYS) + 4 * piece) = w;
      }
      staged = 0;
    };
    auto compute = [&](int32_t i, Tl& tl, uint32_t here) __attribute__((always_inline)) {
      const int32_t key0 = int32_t((tile0 + turns * uint32_t(i)) * KEYS);
      f32x4 x[RT][H];  // logits, then weights, of keys 16 h + 4 j + r and column c's row
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < Tl::KP; ++st) {
            if constexpr (F32) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(tl.k[h][st][e]), __uint_as_float(qf[t][st][e]), s, 0, 0, 0);
            } else {
              s = T::mma(tl.k[h][st], qf[t][st], s);
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) x[t][h][r] = s[r] * a.c;
        }
      // not all keys of the tile, for all rows (uniform)
      const bool masked = careful || here != kAll || key0 + KEYS > int32_t(len - a.rows + 1);
      uint32_t odd = 0;  // keys that some rows see and others do not (careful: any), with an infinity or NaN among their values
      if (masked) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int32_t key = 16 * h + 4 * int32_t(j) + r;
              if (!((here >> key) & 1u) || key0 + key > last_key[t]) x[t][h][r] = kNegInf;
            }
        // values of keys that no row sees are zeros, for 0 times anything else may be NaN
#pragma unroll
        for (int e = 0; e < Tl::VK; ++e) {
          const int32_t key = 4 * int32_t(j) + (e & 3) + 16 * (e >> 2);
          const bool held = (here >> key) & 1u;
          bool bad = false;
#pragma unroll
          for (int w = 0; w < Tl::VW; ++w) {
            if (!held) tl.v[e][w] = 0u;
            if constexpr (F32) bad |= (tl.v[e][w] & 0x7f800000u) == 0x7f800000u;
            else
              bad |= (tl.v[e][w] & T::kExponent) == T::kExponent ||
                     (tl.v[e][w] & (T::kExponent << 16)) == (T::kExponent << 16);
          }
          const uint64_t who = __ballot(bad && (careful || key0 + key > int32_t(len - a.rows)));
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (who & (0xffffull << (16 * g))) odd |= 1u << (4 * g + (e & 3) + 16 * (e >> 2));
        }
      }
      if constexpr (LOGITS) {
        if (staged == stage_room) flush(i);
        float* const to = stage + staged * stage_floats + c * KEYS + 4 * j;
        ++staged;
#pragma unroll
        for (int t = 0; t < RT; ++t)
          if (live[t])
#pragma unroll
            for (int h = 0; h < H; ++h) *reinterpret_cast<f32x4*>(to + 16 * t * KEYS + 16 * h) = x[t][h];
      }
      uint32_t pw[RT][2][4];  // 16 bits: the weights' parts
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float lm = x[t][0][0];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) lm = fmaxf(lm, x[t][h][r]);
        if (__any(lm > m[t] + kRescale)) {  // rare: raise the reference of the columns that need it
          float bm = fmaxf(lm, __shfl_xor(lm, 16));
          bm = fmaxf(bm, __shfl_xor(bm, 32));
          const float mn = fmaxf(m[t], bm);
          const float alpha = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f((m[t] - mn) * kUnit);
          m[t] = mn;
          l[t] *= alpha;
          float ao[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) ao[r] = __shfl(alpha, int(4 * j + r));
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][n][r] *= ao[r];
        }
        const float ms = m[t] == kNegInf ? 0.f : m[t];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[t][h][r] = __builtin_amdgcn_exp2f(fmaf(x[t][h][r] - ms, kUnit, T::kWeights));
            l[t] += x[t][h][r];
          }
        if constexpr (!F32) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float p0 = x[t][w / 2][2 * (w & 1)], p1 = x[t][w / 2][2 * (w & 1) + 1];
            pw[t][0][w] = T::pack(p0, p1);
            pw[t][1][w] = T::pack(p0 - T::low(pw[t][0][w]), p1 - T::high(pw[t][0][w]));
          }
        }
      }
      if (odd) {  // rare: infinities and NaN that not all rows see, or that have no sum, are added one by one
#pragma unroll
        for (int e = 0; e < Tl::VK; ++e) {
          const uint32_t mine = odd >> ((e & 3) + 16 * (e >> 2));
#pragma unroll 1
          for (uint32_t g = 0; g < 4; ++g) {
            if (!((mine >> (4 * g)) & 1u)) continue;
            const int32_t key = key0 + int32_t(4 * g + (e & 3) + 16 * (e >> 2));
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float p = __shfl(x[t][e >> 2][e & 3], int(16 * g + 4 * j + r));
                const bool sees = __shfl(last_key[t], int(4 * j + r)) >= key;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  float value;
                  if constexpr (F32) {
                    value = __uint_as_float(uint32_t(__shfl(int(tl.v[e][n]), int(16 * g + c))));
                  } else {
                    const uint32_t w = uint32_t(__shfl(int(tl.v[e][n / 2]), int(16 * g + c)));
                    value = n & 1 ? T::high(w) : T::low(w);
                  }
                  if (sees && !finite_bits(value)) o[t][n][r] = fmaf(p, value, o[t][n][r]);
                }
              }
          }
          if ((mine >> (4 * j)) & 1u)
#pragma unroll
            for (int w = 0; w < Tl::VW; ++w) {
              uint32_t& word = tl.v[e][w];
              if constexpr (F32) {
                if (!finite_bits(__uint_as_float(word))) word = 0u;
              } else {
                if ((word & T::kExponent) == T::kExponent) word &= 0xffff0000u;
                if ((word & (T::kExponent << 16)) == (T::kExponent << 16)) word &= 0xffffu;
              }
            }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (F32) {
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              o[t][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t][0][r], __uint_as_float(tl.v[r][n]), o[t][n], 0, 0, 0);
        } else {
          u32x4 vf;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            vf[w] = __builtin_amdgcn_perm(tl.v[2 * w + 1][n / 2], tl.v[2 * w][n / 2], n & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int part = 0; part < 2; ++part)
              o[t][n] = T::mma(u32x4{pw[t][part][0], pw[t][part][1], pw[t][part][2], pw[t][part][3]}, vf, o[t][n]);
        }
      }
    };

    for (;; careful = true) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        m[t] = kNegInf;
        l[t] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      if (count > 0) {
        Tl ta, tb;
        // a step's table entries are requested before the rows of the step before it:
        // loads come back in order, and behind the rows they would wait for them
        Pages pages = fetch(0), more = fetch(1);
        uint32_t held_a = load(0, pages, ta), held_b;
        for (int32_t i = 0;;) {
          pages = more;
          more = fetch(i + 2);
          held_b = load(i + 1, pages, tb);
          if constexpr (FAST) __builtin_amdgcn_sched_barrier(0);
          compute(i, ta, held_a);
          if (++i >= count) break;
          pages = more;
          more = fetch(i + 2);
          held_a = load(i + 1, pages, ta);
          if constexpr (FAST) __builtin_amdgcn_sched_barrier(0);
          compute(i, tb, held_b);
          if (++i >= count) break;
        }
      }
      if constexpr (LOGITS) flush(count);
      if (F32 || careful) break;
      float none = 0.f;  // NaN if an output is infinite or NaN
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) none = fmaf(o[t][n][r], 0.f, none);
      if (!__any(none != none)) break;
    }

    // The lane's dims of output row r, in their order: (its tiles n one after
    // another, or four by four)
    auto dim_of = [&](int n) __attribute__((always_inline)) { return F32 ? 64 * (n / 4) + 4 * int(c) : NT * int(c) + n; };
    constexpr int STEP = F32 ? 4 : NT;  // neighbouring dims
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float lt = l[t];
      lt += __shfl_xor(lt, 16);
      lt += __shfl_xor(lt, 32);
      const uint32_t row0 = row_tile * ROWS + 16 * t;
      auto out_of = [&](uint32_t n) __attribute__((always_inline)) {
        const uint32_t r = n / a.group;
        return a.out + int64_t(seq) * a.out_batch + int64_t(r) * a.out_row +
               int64_t(kvh * a.group + (n - r * a.group)) * a.out_head;
      };
      if (turns == 1) {  // uniform in the workgroup
        const int64_t first_id = whole ? (int64_t(seq) * a.hkv + kvh) * head_rows
                                       : (int64_t(2 * range + which) * a.hkv + kvh) * head_rows;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t n = row0 + 4 * j + r;
          const float sum = __shfl(lt, int(4 * j + r));
          if (n >= head_rows) continue;
          const float inverse = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
          char* to = whole ? out_of(n) : nullptr;
#pragma unroll
          for (int d = 0; d < NT; d += STEP) {
            float y[STEP];
#pragma unroll
            for (int e = 0; e < STEP; ++e) y[e] = o[t][d + e][r] * inverse;
            if (whole) {
              store_row<DT, STEP>(to + dim_of(d) * T::ES, y);
            } else {
              float* part = a.o + (first_id + n) * D + dim_of(d);
#pragma unroll
              for (int e = 0; e < STEP; e += 4) *reinterpret_cast<f32x4*>(part + e) = f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]};
            }
          }
        }
        if (j == 0 && live[t]) {
          if (!whole) a.ml[first_id + row0 + c] = make_float2(m[t], lt);
          else if (a.stats) a.stats[first_id + row0 + c] = statistics(m[t], lt);
        }
      } else {
        float* mine = lds[wave];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int n = 0; n < NT; n += 4)
            *reinterpret_cast<f32x4*>(mine + (4 * j + r) * D + dim_of(n)) =
                f32x4{o[t][n][r], o[t][n + 1][r], o[t][n + 2][r], o[t][n + 3][r]};
        if (j == 0) {
          mine[16 * D + 2 * c] = m[t];
          mine[16 * D + 2 * c + 1] = lt;
        }
        __syncthreads();
        // the waves' results of 4 dims of a row, a thread
        for (uint32_t e = threadIdx.x; e < a.heads * uint32_t(16 * D / 4); e += blockDim.x) {
          const uint32_t line = e / (D / 4), dim = 4 * (e - line * (D / 4)), head = line / 16, row = line - head * 16;
          const uint32_t n = row0 + row;
          if (n >= head_rows) continue;
          float top = kNegInf, sum = 0.f;
          f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
          for (uint32_t w = head; w < a.heads * turns; w += a.heads) top = fmaxf(top, lds[w][16 * D + 2 * row]);
          const float ts = top == kNegInf ? 0.f : top;
          for (uint32_t w = head; w < a.heads * turns; w += a.heads) {
            const float f = __builtin_amdgcn_exp2f((lds[w][16 * D + 2 * row] - ts) * kUnit);
            sum = fmaf(f, lds[w][16 * D + 2 * row + 1], sum);
            const f32x4 part = *reinterpret_cast<const f32x4*>(&lds[w][row * D + dim]);
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[x] = fmaf(f, part[x], acc[x]);
          }
          const uint32_t h = head0 + head;
          if (whole) {
            const uint32_t r = n / a.group;
            char* to = a.out + int64_t(seq) * a.out_batch + int64_t(r) * a.out_row +
                       int64_t(h * a.group + (n - r * a.group)) * a.out_head + dim * T::ES;
            const float inverse = sum == 0.f ? 0.f : 1.f / sum;
            const float y[4] = {acc[0] * inverse, acc[1] * inverse, acc[2] * inverse, acc[3] * inverse};
            store_row<DT, 4>(to, y);
            if (a.stats && dim == 0) a.stats[(int64_t(seq) * a.hkv + h) * head_rows + n] = statistics(top, sum);
          } else {
            const int64_t id = (int64_t(2 * range + which) * a.hkv + h) * head_rows + n;
            *reinterpret_cast<f32x4*>(a.o + id * D + dim) = acc;
            if (dim == 0) a.ml[id] = make_float2(top, sum);
          }
        }
        __syncthreads();  // the buffers are free again
      }
    }
    if (a.whole || before >= end) break;
  }
}

// The ranges that hold a sequence (wave-uniform): r0 .. r1, one alone if it is written whole.
struct Held {
  uint32_t r0, r1;
};
template <int KEYS>
__device__ __forceinline__ Held ranges_of(const PagedAttnArgs& a, uint32_t seq, uint32_t len) {
  if (a.whole || len == 0) return Held{0, 0};
  // places before the sequence, and of all
  uint32_t before = 0, total = 0;
  for (uint32_t b = threadIdx.x & 63; b < a.batch; b += 64) {
    const uint32_t t = places_of<KEYS>(context_of(a, b));
    total += t;
    before += b < seq ? t : 0u;
  }
  total = wave_total(total);
  before = wave_total(before);
  const Ranges cut(total, a.ranges);
  return Held{cut.of(before + kHead), cut.of(before + kHead + tiles_of<KEYS>(len) - 1)};
}

// A row of a sequence that more than one range holds, or that has no keys: every 32
// lanes each SUBS-th range, each lane D / 32 dims.
template <int DT, int D, int SUBS>
__device__ __forceinline__ void merge_row(const PagedAttnArgs& a, uint32_t seq, uint32_t row) {
  constexpr int N = D / 32, KEYS = Type<DT>::KEYS;
  typedef float VecN __attribute__((ext_vector_type(N)));
  __shared__ float s_o[SUBS][D], s_l[SUBS], s_m[SUBS];
  const uint32_t dim = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const uint32_t len = context_of(a, seq);
  const uint32_t head_rows = a.rows * a.group;
  const uint32_t kvh = row / head_rows, n = row - kvh * head_rows;
  float top = kNegInf, sum = 0.f;
  VecN acc = VecN(0.f);
  if (len != 0) {
    const Held held = ranges_of<KEYS>(a, seq, len);
    if (held.r0 == held.r1) return;  // written by its range
#pragma unroll 4
    for (uint32_t r = held.r0 + sub; r <= held.r1; r += SUBS) {
      const int64_t id = (int64_t(2 * r + (r == held.r0 ? 1u : 0u)) * a.hkv + kvh) * head_rows + n;
      const float2 ml = a.ml[id];
      const VecN part = *reinterpret_cast<const VecN*>(a.o + id * D + N * dim);
      const float mn = fmaxf(top, ml.x), ms = mn == kNegInf ? 0.f : mn;
      const float f = __builtin_amdgcn_exp2f((top - ms) * kUnit), w = __builtin_amdgcn_exp2f((ml.x - ms) * kUnit);
      sum = f * sum + w * ml.y;
      acc = f * acc + w * part;
      top = mn;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) s_o[sub][N * dim + e] = acc[e];
  if (dim == 0) {
    s_m[sub] = top;
    s_l[sub] = sum;
  }
  __syncthreads();
  if (threadIdx.x >= uint32_t(D)) return;
  float all = kNegInf, l = 0.f, o = 0.f;
#pragma unroll
  for (int i = 0; i < SUBS; ++i) all = fmaxf(all, s_m[i]);
  const float ms = all == kNegInf ? 0.f : all;
#pragma unroll
  for (int i = 0; i < SUBS; ++i) {
    const float w = __builtin_amdgcn_exp2f((s_m[i] - ms) * kUnit);
    l = fmaf(w, s_l[i], l);
    o = fmaf(w, s_o[i][threadIdx.x], o);
  }
  const uint32_t r = n / a.group, h = kvh * a.group + n - r * a.group;
  char* to = a.out + int64_t(seq) * a.out_batch + int64_t(r) * a.out_row + int64_t(h) * a.out_head;
  const float y = l == 0.f ? 0.f : o / l;
  if constexpr (DT == CBK_DTYPE_F32) reinterpret_cast<float*>(to)[threadIdx.x] = y;
  else reinterpret_cast<uint16_t*>(to)[threadIdx.x] = uint16_t(Type<DT>::pack(y, 0.f));
  if (a.stats && threadIdx.x == 0) a.stats[(int64_t(seq) * a.hkv + kvh) * head_rows + n] = statistics(all, l);
}

template <int DT, int D, int SUBS>
__global__ __launch_bounds__(32 * SUBS) void paged_attn_merge_kernel(const PagedAttnArgs a) {
  merge_row<DT, D, SUBS>(a, blockIdx.y, blockIdx.x);
}

// weights[b, set, k] += the sum of key k's softmax weights over the set's rows. A
// thread takes 4 keys and every SUBS-th row; the SUBS sums are added in their order. Bound by
// reading the logits, most of them from the last cache level.
template <int DT, int SUBS>
__device__ __forceinline__ void key_weights(const PagedAttnArgs& a, uint32_t seq, uint32_t len, uint32_t set, uint32_t chunk,
                                            const float2* stats) {
  constexpr int KEYS = Type<DT>::KEYS, KT = 256 / SUBS;  // threads beside each other
  constexpr float kWeights = Type<DT>::kWeights;
  typedef Piece<4>::V16 V;
  __shared__ f32x4 s_sum[SUBS == 1 ? 1 : 256];
  const uint32_t sub = threadIdx.x / KT, key = 4 * (chunk * KT + threadIdx.x % KT);
  const uint32_t heads = a.hkv / a.w_sets, rows = heads * a.rows * a.group;
  const float* x = a.logits + ((int64_t(seq) * a.max_tiles + key / KEYS) * a.hkv + set * heads) * int64_t(a.rows * a.group * KEYS) + key % KEYS;
  float* const to = a.weights + int64_t(seq) * a.w_batch + int64_t(set) * a.w_set + key;
  f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
  if (key < len) {
    auto add = [](float sum, float y, const float2& st) __attribute__((always_inline)) {
      return fmaf(__builtin_amdgcn_exp2f(fmaf(y - st.x, kUnit, kWeights)), st.y, sum);
    };
#pragma unroll 4
    for (uint32_t n = sub; n < rows; n += SUBS) {
      const float2 st = stats[n];
      const f32x4 y = *reinterpret_cast<const f32x4*>(x + int64_t(n) * KEYS);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = add(sum[e], y[e], st);
    }
    const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    if (all != all) {
      // rare: a row without a number gives NaN to the keys that it sees, and nothing to others
      // (above 0 times NaN), which their logits of -inf do not tell. (Marks for hidden keys among the
      // logits made the waves that write them slower: 24 sequences of 8 K 99.8 us, 107 to 110 with.)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        sum[e] = 0.f;
        const uint32_t at = min(key + e, len - 1);
        const bool held = uint32_t(a.tables[int64_t(seq) * a.table_stride + a.block_div.div(at)]) < a.num_blocks;
        if (!held) continue;
#pragma unroll 1
        for (uint32_t n = sub; n < rows; n += SUBS) {
          const uint32_t r = n % (a.rows * a.group) / a.group;
          if (int32_t(at) <= int32_t(len) - int32_t(a.rows) + int32_t(r)) sum[e] = add(sum[e], x[int64_t(n) * KEYS + e], stats[n]);
        }
      }
    }
  }
  if constexpr (SUBS > 1) {
    s_sum[threadIdx.x] = sum;
    __syncthreads();
    if (sub != 0) return;
    for (int i = 1; i < SUBS; ++i) sum += s_sum[i * KT + threadIdx.x];
  }
  if (key + 4 <= len) {
    const f32x4 old = __builtin_bit_cast(f32x4, *reinterpret_cast<const V*>(to));
    *reinterpret_cast<V*>(to) = __builtin_bit_cast(u32x4, old + sum);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
      if (key + e < len) to[e] += sum[e];
  }
}

template <int DT, int SUBS>
__global__ __launch_bounds__(256) void key_weights_kernel(const PagedAttnArgs a) {
  const uint32_t seq = blockIdx.z, set = blockIdx.y, len = context_of(a, seq);
  if (blockIdx.x * (1024 / SUBS) >= len) return;
  key_weights<DT, SUBS>(a, seq, len, set, blockIdx.x,
                        a.stats + (int64_t(seq) * a.hkv + set * (a.hkv / a.w_sets)) * (a.rows * a.group));
}

// Both, for sets of few rows: the first workgroups merge a row each, the others take
// keys, and the statistics of their rows from the partial results once more. One
// launch less: 3 to 5 us.
constexpr uint32_t kJoinRows = 64;
template <int DT, int D, int SUBS>
__global__ __launch_bounds__(256) void join_kernel(const PagedAttnArgs a) {
  constexpr int KEYS = Type<DT>::KEYS;
  const uint32_t seq = blockIdx.y, all_rows = a.rows * a.hq;
  if (blockIdx.x < all_rows) {
    merge_row<DT, D, 8>(a, seq, blockIdx.x);
    return;
  }
  const uint32_t chunk = (blockIdx.x - all_rows) / a.w_sets, set = blockIdx.x - all_rows - chunk * a.w_sets;
  const uint32_t len = context_of(a, seq);
  if (chunk * (1024 / SUBS) >= len) return;
  const uint32_t head_rows = a.rows * a.group, head0 = set * (a.hkv / a.w_sets), rows = a.hkv / a.w_sets * head_rows;
  const Held held = ranges_of<KEYS>(a, seq, len);
  const float2* stats = a.stats + (int64_t(seq) * a.hkv + head0) * head_rows;
  if (held.r0 != held.r1) {
    // 16 lanes a row
    __shared__ float2 s_stats[kJoinRows];
    const uint32_t lane = threadIdx.x & 15;
    for (uint32_t n = threadIdx.x >> 4; n < rows; n += 16) {
      float top = kNegInf, sum = 0.f;
#pragma unroll 4
      for (uint32_t r = held.r0 + lane; r <= held.r1; r += 16) {
        const float2 ml = a.ml[(int64_t(2 * r + (r == held.r0 ? 1u : 0u)) * a.hkv + head0) * head_rows + n];
        const float mn = fmaxf(top, ml.x), ms = mn == kNegInf ? 0.f : mn;
        sum = __builtin_amdgcn_exp2f((top - ms) * kUnit) * sum + __builtin_amdgcn_exp2f((ml.x - ms) * kUnit) * ml.y;
        top = mn;
      }
      const float most = row16_reduce(top, [](float x, float y) { return fmaxf(x, y); }), ms = most == kNegInf ? 0.f : most;
      sum = row16_reduce(__builtin_amdgcn_exp2f((top - ms) * kUnit) * sum, [](float x, float y) { return x + y; });
      if (lane == 0) s_stats[n] = statistics(most, sum);
    }
    __syncthreads();
    stats = s_stats;
  }
  key_weights<DT, SUBS>(a, seq, len, set, chunk, stats);
}

// The same for sets and KV heads of many rows, without logits: a second product of the keys with
// the queries, by the rows' statistics. The waves of a workgroup take its 64 keys and each a
// part of the set's 16-row tiles, head by head; their sums are added in their order. Bound by
// dependences at two waves a SIMD (VALU 34% busy, matrix cores 10%): 17 us for 2 prompts of 8 K,
// 32 rows of 32 heads over 4. With 32 keys a wave 25; rows requested a tile or two ahead 17 and
// 18.5; four waves a SIMD spill, 28.
constexpr uint32_t kWindowKeys = 64, kWindowWaves = 8;
template <int DT, int D>
__global__ __launch_bounds__(64 * kWindowWaves, 2) void window_weights_kernel(const PagedAttnArgs a) {
  using T = Type<DT>;
  constexpr int KP = D * T::ES / 64, G = kWindowKeys / 16;
  typedef typename Piece<T::ES>::V16 V;
  __shared__ float s_sum[kWindowWaves][kWindowKeys];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane >> 4, c = lane & 15;
  const uint32_t seq = blockIdx.z, set = blockIdx.y, key0 = blockIdx.x * kWindowKeys, len = context_of(a, seq);
  if (key0 >= len) return;
  const uint32_t head_rows = a.rows * a.group, heads = a.hkv / a.w_sets, head0 = set * heads;
  const uint32_t tiles = (head_rows + 15) / 16, units = heads * tiles;
  const uint32_t begin = units / kWindowWaves * wave + min(wave, units % kWindowWaves);
  const uint32_t end = begin + units / kWindowWaves + (wave < units % kWindowWaves);
  // the lane's keys, as it reads them: key0 + 16 g + c
  const int32_t* const table = a.tables + int64_t(seq) * a.table_stride;
  int64_t row[G];
  bool held[G];
  uint64_t here = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const uint32_t key = key0 + 16 * g + c, blk = a.block_div.div(min(key, len - 1)), page = uint32_t(table[blk]);
    held[g] = key < len && page < a.num_blocks;
    row[g] = held[g] ? int64_t(page) * a.block_stride + int64_t(key - blk * a.block_div.d) * a.token_stride : 0;
    here |= (__ballot(held[g]) & 0xffffull) << (16 * g);
  }
  const bool masked = here != ~0ull >> (64 - kWindowKeys) || int32_t(key0 + kWindowKeys) > int32_t(len) - int32_t(a.rows) + 1;
  struct Rows {
    u32x4 q[KP];
    float2 st;
    int32_t last;  // a row sees keys up to it
  };
  f32x4 sum[G];  // keys 16 g + 4 j + i, column c's rows
#pragma unroll
  for (int g = 0; g < G; ++g) sum[g] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t u = begin; u < end;) {
    const uint32_t head = u / tiles, kvh = head0 + head, first = u - head * tiles, past = min(tiles, end - head * tiles);
    u = head * tiles + past;
    u32x4 k[G][KP];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const char* p = a.k_base + row[g] + int64_t(kvh) * (D * T::ES) + 16 * j;
#pragma unroll
      for (int s = 0; s < KP; ++s) {
        k[g][s] = u32x4(0u);
        if (held[g]) k[g][s] = *reinterpret_cast<const V*>(p + 64 * s);
      }
    }
    // row tile t; a lane without a row has the last row's
    auto rows_of = [&](uint32_t t) __attribute__((always_inline)) {
      Rows x;
      const uint32_t n = 16 * t + c, row = min(n, head_rows - 1);
      const uint32_t r = row / a.group, h = kvh * a.group + (row - r * a.group);
      const char* p = a.q + int64_t(seq) * a.q_batch + int64_t(r) * a.q_row + int64_t(h) * a.q_head + 16 * j;
#pragma unroll
      for (int s = 0; s < KP; ++s) x.q[s] = *reinterpret_cast<const V*>(p + 64 * s);
      x.st = a.stats[(int64_t(seq) * a.hkv + kvh) * head_rows + row];
      x.last = n < head_rows ? int32_t(len) - int32_t(a.rows) + int32_t(r) : -1;
      return x;
    };
    auto add = [&](uint32_t t, const Rows& now) __attribute__((always_inline)) {
      const bool some = masked || 16 * t + 16 > head_rows;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KP; ++s) x = T::mma(k[g][s], now.q[s], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] *= a.c;
        f32x4 y = f32x4{now.st.y, now.st.y, now.st.y, now.st.y};
        if (some) {  // 0, not 0 times what may be no number
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t key = 16 * g + 4 * int32_t(j) + i;
            if (!((here >> key) & 1u) || int32_t(key0) + key > now.last) {
              x[i] = kNegInf;
              y[i] = 0.f;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sum[g][i] = fmaf(__builtin_amdgcn_exp2f(fmaf(x[i] - now.st.x, kUnit, T::kWeights)), y[i], sum[g][i]);
      }
    };
    for (uint32_t t = first; t < past; ++t) add(t, rows_of(t));
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float all = row16_reduce(sum[g][i], [](float x, float y) { return x + y; });
      if (c == 0) s_sum[wave][16 * g + 4 * j + i] = all;
    }
  __syncthreads();
  if (threadIdx.x >= min(kWindowKeys, len - key0)) return;
  float all = s_sum[0][threadIdx.x];
#pragma unroll
  for (uint32_t w = 1; w < kWindowWaves; ++w) all += s_sum[w][threadIdx.x];
  a.weights[int64_t(seq) * a.w_batch + int64_t(set) * a.w_set + key0 + threadIdx.x] += all;
}

template <int DT, int D, int RT, int MODE>
int launch_attn(const PagedAttnArgs& a, hipStream_t s) {
  const uint64_t groups = uint64_t(a.hkv / a.heads) * a.row_tiles * ((a.ranges + 7) / 8 * 8);
  const uint32_t threads = 64 * a.heads * a.turns;
  CBK_REQUIRE(groups * threads < (uint64_t(1) << 32), "paged attention: %llu workgroups exceed one launch",
              (unsigned long long)groups);
  const dim3 grid(uint32_t(groups), 1, 1), block(threads);
  if (a.logits) hipLaunchKernelGGL((paged_attn_kernel<DT, D, RT, true, MODE>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((paged_attn_kernel<DT, D, RT, false, MODE>), grid, block, 0, s, a);
  return launch_status("paged attention");
}

template <int DT, int D, int RT>
int launch_mode(const PagedAttnArgs& a, hipStream_t s) {
  if (!a.fast) return launch_attn<DT, D, RT, 0>(a, s);
  return a.stream ? launch_attn<DT, D, RT, 2>(a, s) : launch_attn<DT, D, RT, 1>(a, s);
}

template <int DT, int D>
int launch(const PagedAttnArgs& a, hipStream_t s) {
  const bool weigh = a.weights != nullptr && a.max_len != 0;
  const uint32_t all_rows = a.rows * a.hq, set_rows = weigh ? all_rows / a.w_sets : 0;
  const bool window = weigh && a.logits == nullptr, join = weigh && !window && !a.whole && set_rows <= kJoinRows;
  // a workgroup's keys: few rows by a thread each, many by several beside each other (us of
  // the weights alone, bf16: 2 prompts of 8 K, 32 rows of 32 heads together 286 / 11.4 with 1
  // / 32; 24 sequences of 8 K, one row of 4 heads, 11.7 with one key a thread, 7.1 with 4)
  const uint32_t keys = window ? kWindowKeys : set_rows <= 8 ? 1024 : set_rows <= 64 ? 256 : 32;
  const uint64_t chunks = weigh ? (uint64_t(a.max_len) + keys - 1) / keys : 0;
  const uint64_t widest = join ? all_rows + chunks * a.w_sets : chunks;
  CBK_REQUIRE(widest < (1 << 23) && all_rows < (1 << 22), "paged attention: %u rows, key weights of %llu workgroups exceed one launch",
              all_rows, (unsigned long long)widest);
  if (int rc = a.rt == 1 ? launch_mode<DT, D, 1>(a, s) : launch_mode<DT, D, 2>(a, s)) return rc;
  if (join) {
    const dim3 grid(uint32_t(widest), a.batch);
    if (set_rows <= 8) hipLaunchKernelGGL((join_kernel<DT, D, 1>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((join_kernel<DT, D, 4>), grid, dim3(256), 0, s, a);
    return launch_status("paged attention merge and key weights");
  }
  if (!a.whole) {
    const dim3 grid(all_rows, a.batch);
    if (a.ranges > 16 * a.batch) hipLaunchKernelGGL((paged_attn_merge_kernel<DT, D, 32>), grid, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((paged_attn_merge_kernel<DT, D, 8>), grid, dim3(256), 0, s, a);
    if (int rc = launch_status("paged attention merge")) return rc;
  }
  if (!weigh) return CBK_OK;
  const dim3 grid(uint32_t(chunks), a.w_sets, a.batch);
  if (window) {
    if constexpr (DT != CBK_DTYPE_F32)
      hipLaunchKernelGGL((window_weights_kernel<DT, D>), grid, dim3(64 * kWindowWaves), 0, s, a);
  }
  else if (set_rows <= 8) hipLaunchKernelGGL((key_weights_kernel<DT, 1>), grid, dim3(256), 0, s, a);
  else if (set_rows <= 64) hipLaunchKernelGGL((key_weights_kernel<DT, 4>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((key_weights_kernel<DT, 32>), grid, dim3(256), 0, s, a);
  return launch_status("key weights");
}

template <int DT>
int launch_type(const PagedAttnArgs& a, int64_t head_dim, hipStream_t s) {
  return head_dim == 128 ? launch<DT, 128>(a, s) : launch<DT, 64>(a, s);
}

}  // namespace
}  // namespace cbk
