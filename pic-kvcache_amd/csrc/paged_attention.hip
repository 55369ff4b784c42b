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
// Bound by HBM: each key and value row is read once for all rows of a group.
// Beside that the matrix cores and the VALU have little to do (a 32-key tile of
// a KV head, 16 KB, is 16 MFMAs and some 300 VALU instructions for up to 16
// rows), so the kernel is laid out for loads in flight and nothing else: a wave
// takes a tile of one KV head at a time straight into registers, K and V of
// the next tile requested before this one's are waited for, no LDS and no
// barrier on the way.
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
// (bf16) or 2^-22 (float16) of themselves (below that, float16: 2^-30 of the
// largest); sums and statistics are float32.
//
// The batch's tiles are cut into equal ranges (paged_ranges.hpp); a workgroup
// takes one, a wave a KV head, or several waves a head's tiles in turns. A
// sequence that one range holds whole is written at once, the others' partial
// results are merged by a second launch. For the keys' weights the waves leave
// the logits in scratch (4 bytes a row and key, beside 4 D or 8 D bytes a key that
// they read), and a third launch turns them into weights with the rows' statistics.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_ranges.hpp"

namespace cbk {
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
  bool whole;                            // range r is sequence r, and no partial results
  uint32_t heads, turns;                 // of a workgroup: KV heads, and waves that share one's tiles
  float c;                               // scale log2 e / kUnit
  FastDiv block_div;
  // partial results of range r's first (0) and last (1) unfinished sequence:
  // entry ((2 r + which) hkv + kv head) * rows * group + row * group + head
  float2* ml;
  float* o;
  // for the keys' weights: the rows' statistics, (b hkv + kv head) * rows * group
  // + ..; the logits [b][tile][kv head][row, head][key of the tile]
  float2* stats;
  float* logits;
};

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

// waves of a workgroup, at most: two a SIMD; one where two row tiles take its registers
constexpr int max_waves(int rt) { return rt == 1 ? 8 : 4; }

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

template <int DT, int D, int RT, bool LOGITS>
__global__ __launch_bounds__(64 * max_waves(RT), 1) void paged_attn_kernel(const PagedAttnArgs a) {
  using T = Type<DT>;
  using Tl = Tile<DT, D>;
  constexpr int KEYS = T::KEYS, H = Tl::HALVES, NT = D / 16;  // NT: 16-column tiles of the output
  constexpr int ROWS = 16 * RT;
  constexpr bool F32 = DT == CBK_DTYPE_F32;
  // several waves of a head: their results of 16 rows [row][D], then each row's m and l
  __shared__ __attribute__((aligned(16))) float lds[max_waves(RT)][16 * D + 32];

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
  uint32_t at = 0, end, seq = 0, before = 0;  // the range, the sequence that holds tile `at`, the tiles before it
  if (a.whole) {
    seq = range;
    end = tiles_of<KEYS>(uint32_t(__builtin_amdgcn_readfirstlane(int(len0))));
  } else {
    const uint32_t tiles0 = tiles_of<KEYS>(len0);
    uint32_t all = tiles0;
    for (uint32_t b = lane + 64; b < a.batch; b += 64) all += tiles_of<KEYS>(context_of(a, b));
    const Ranges cut(wave_total(all), a.ranges);
    at = cut.first(range);
    end = cut.first(range + 1);
    if (at == end) return;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
      uint32_t n = tiles0;
      if (b0 > 0) n = b0 + lane < a.batch ? tiles_of<KEYS>(context_of(a, b0 + lane)) : 0u;
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

  for (bool first_seq = true;; first_seq = false) {
    uint32_t len = a.whole ? uint32_t(__builtin_amdgcn_readfirstlane(int(len0))) : length(seq);
    while (!a.whole && before + tiles_of<KEYS>(len) <= at) {  // empty sequences, and on to the next
      before += tiles_of<KEYS>(len);
      len = length(++seq);
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    len = __builtin_amdgcn_readfirstlane(len);
    before = __builtin_amdgcn_readfirstlane(before);
    const uint32_t seq_end = before + tiles_of<KEYS>(len);
    const uint32_t stop = min(end, seq_end);
    const bool whole = at == before && stop == seq_end;  // (a.whole: an empty one, too)
    const uint32_t tile0 = at - before + turn;  // the wave's first tile of the sequence
    const int32_t count = stop - at > turn ? int32_t((stop - at - turn + turns - 1) / turns) : 0;
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

    // The block table's entry of this lane's key of step i (a tile's keys, one
    // a lane; behind the last step, the last key's), and, from it, the tile's rows.
    // Keys past the context or in a page out of range are read from the
    // wave's first row and masked: their bits of the result are clear. A step behind
    // the last reads that row alone, so that every step has the same loads after
    // it and none waits for more than its own. (The first row of the cache
    // instead, for all waves at the same time: 4 us at the end of a call.)
    auto entry = [&](int32_t i) __attribute__((always_inline)) {
      const uint32_t key = min((tile0 + turns * uint32_t(i)) * KEYS + (lane & (KEYS - 1)), len - 1);
      return uint32_t(table[a.block_div.div(key)]);
    };
    uint64_t spare = 0;
    const char* const k_base = a.k_base + int64_t(kvh) * (D * T::ES) + 16 * j;
    const char* const v_base = a.v_base + int64_t(kvh) * (D * T::ES);
    auto load = [&](int32_t i, uint32_t page, Tl& to) __attribute__((always_inline)) {
      const uint32_t key = (tile0 + turns * uint32_t(i)) * KEYS + (lane & (KEYS - 1));
      const bool held = i < count && key < len && page < a.num_blocks;
      uint64_t row = spare;
      if (held) {
        const uint32_t blk = a.block_div.div(key);
        row = uint64_t(page) * uint64_t(a.block_stride) + uint64_t(key - blk * a.block_div.d) * uint64_t(a.token_stride);
      }
      if (i == 0) spare = (uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(row >> 32))))) << 32) |
                          uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(row))));
      auto row_of = [&](uint32_t from) __attribute__((always_inline)) {
        return uint64_t(uint32_t(__shfl(int(uint32_t(row)), int(from)))) |
               (uint64_t(uint32_t(__shfl(int(uint32_t(row >> 32)), int(from)))) << 32);
      };
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const char* p = k_base + row_of(16 * h + c);
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
      return uint32_t(__ballot(held)) & (KEYS == 32 ? 0xffffffffu : 0xffffu);
    };

    float m[RT], l[RT];  // of the lane's column: reference maximum, sum of the lane's keys
    f32x4 o[RT][NT];     // rows 4 j + i of the row tile, column c of tile n: dim NT c + n (float32: 64 (n / 4) + 4 c + n % 4)
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      m[t] = kNegInf;
      l[t] = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) o[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

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
      const bool masked = here != (KEYS == 32 ? 0xffffffffu : 0xffffu) || key0 + KEYS > int32_t(len - a.rows + 1);
      uint32_t odd = 0;  // keys that some rows see and others do not, with an infinity or NaN among their values
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
          const uint64_t who = __ballot(bad && key0 + key > int32_t(len - a.rows));
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (who & (0xffffull << (16 * g))) odd |= 1u << (4 * g + (e & 3) + 16 * (e >> 2));
        }
      }
      if constexpr (LOGITS) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const uint32_t n = row_tile * ROWS + 16 * t + c;
          float* to = a.logits + ((int64_t(seq) * a.max_tiles + (tile0 + turns * uint32_t(i))) * a.hkv + kvh) * int64_t(head_rows * KEYS) +
                      n * KEYS + 4 * j;
          if (live[t])
#pragma unroll
            for (int h = 0; h < H; ++h) *reinterpret_cast<f32x4*>(to + 16 * h) = x[t][h];
        }
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
      if (odd) {  // rare: infinities and NaN that only some rows see are added one by one
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

    if (count > 0) {
      Tl ta, tb;
      // a step's table entries are requested before the rows of the step before it:
      // loads come back in order, and behind the rows they would wait for them
      uint32_t page = entry(0), next = entry(1);
      uint32_t held_a = load(0, page, ta), held_b;
      for (int32_t i = 0;;) {
        page = next;
        next = entry(i + 2);
        held_b = load(i + 1, page, tb);
        compute(i, ta, held_a);
        if (++i >= count) break;
        page = next;
        next = entry(i + 2);
        held_a = load(i + 1, page, ta);
        compute(i, tb, held_b);
        if (++i >= count) break;
      }
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
                                       : (int64_t(2 * range + (first_seq ? 0 : 1)) * a.hkv + kvh) * head_rows;
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
          else if (LOGITS) a.stats[first_id + row0 + c] = statistics(m[t], lt);
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
            if (LOGITS && dim == 0) a.stats[(int64_t(seq) * a.hkv + h) * head_rows + n] = statistics(top, sum);
          } else {
            const int64_t id = (int64_t(2 * range + (first_seq ? 0 : 1)) * a.hkv + h) * head_rows + n;
            *reinterpret_cast<f32x4*>(a.o + id * D + dim) = acc;
            if (dim == 0) a.ml[id] = make_float2(top, sum);
          }
        }
        __syncthreads();  // the buffers are free again
      }
    }
    at = stop;
    if (at >= end) break;
  }
}

// The sequences that more than one range holds, and those without keys: a
// workgroup per row, every 32 lanes each SUBS-th range of it, each lane D / 32
// dims.
template <int DT, int D, int SUBS>
__global__ __launch_bounds__(32 * SUBS) void paged_attn_merge_kernel(const PagedAttnArgs a) {
  constexpr int N = D / 32, KEYS = Type<DT>::KEYS;
  typedef float VecN __attribute__((ext_vector_type(N)));
  __shared__ float s_o[SUBS][D], s_l[SUBS], s_m[SUBS];
  const uint32_t seq = blockIdx.y;
  const uint32_t lane = threadIdx.x & 63, dim = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const uint32_t tiles = tiles_of<KEYS>(context_of(a, seq));
  const uint32_t head_rows = a.rows * a.group;
  const uint32_t kvh = blockIdx.x / head_rows, n = blockIdx.x - kvh * head_rows;
  float top = kNegInf, sum = 0.f;
  VecN acc = VecN(0.f);
  if (tiles != 0) {
    // tiles before the sequence, and of all
    uint32_t before = 0, total = 0;
    for (uint32_t b = lane; b < a.batch; b += 64) {
      const uint32_t t = tiles_of<KEYS>(context_of(a, b));
      total += t;
      before += b < seq ? t : 0u;
    }
    total = wave_total(total);
    before = wave_total(before);
    const Ranges cut(total, a.ranges);
    const uint32_t r0 = cut.of(before), r1 = cut.of(before + tiles - 1);
    if (r0 == r1) return;  // written by its range
    // range r0 may end with this sequence after others; the rest begin in it
    const uint32_t which0 = cut.first(r0) < before ? 1u : 0u;
#pragma unroll 4
    for (uint32_t r = r0 + sub; r <= r1; r += SUBS) {
      const int64_t id = (int64_t(2 * r + (r == r0 ? which0 : 0u)) * a.hkv + kvh) * head_rows + n;
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

// weights[b, set, k] += the sum of key k's softmax weights over the set's rows. A
// thread takes 4 keys and every SUBS-th row; the SUBS sums are added in their order.
template <int DT, int SUBS>
__global__ __launch_bounds__(256) void key_weights_kernel(const PagedAttnArgs a, float* weights, int64_t batch_stride,
                                                          int64_t set_stride, uint32_t sets) {
  constexpr int KEYS = Type<DT>::KEYS, KT = 256 / SUBS;  // threads beside each other
  constexpr float kWeights = Type<DT>::kWeights;
  typedef Piece<4>::V16 V;
  __shared__ f32x4 s_sum[SUBS == 1 ? 1 : 256];
  const uint32_t seq = blockIdx.z, set = blockIdx.y, sub = threadIdx.x / KT;
  const uint32_t key = 4 * (blockIdx.x * KT + threadIdx.x % KT);
  const uint32_t len = context_of(a, seq);
  if (4 * blockIdx.x * KT >= len) return;
  const uint32_t heads = a.hkv / sets, rows = heads * a.rows * a.group;
  const float* x = a.logits + ((int64_t(seq) * a.max_tiles + key / KEYS) * a.hkv + set * heads) * int64_t(a.rows * a.group * KEYS) + key % KEYS;
  const float2* stats = a.stats + (int64_t(seq) * a.hkv + set * heads) * (a.rows * a.group);
  float* const to = weights + int64_t(seq) * batch_stride + int64_t(set) * set_stride + key;
  f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
  if (key < len) {
#pragma unroll 4
    for (uint32_t n = sub; n < rows; n += SUBS) {
      const float2 st = stats[n];
      const f32x4 y = *reinterpret_cast<const f32x4*>(x + int64_t(n) * KEYS);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(__builtin_amdgcn_exp2f(fmaf(y[e] - st.x, kUnit, kWeights)), st.y, sum[e]);
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

// Sequences stay whole where that gives a wave few more tiles than equal ranges (a merge
// is as long as two or three), and few altogether (they may differ in length, and the
// longest counts). us a call, ranges / whole, bf16, 32 heads over 8 x 128: 1 sequence of
// 600 12.6 / 12.0, of 1000 (weights summed, 4 tiles instead of 1) 15.6 / 21.0; 64 of 256 to 1024
// 38.5 / 35.9; 256 of 128 to 512 88 / 77; 64 of 4 K to 16 K (512 tiles both) 451 / 534.
constexpr int64_t kMergeTiles = 2, kWholeTiles = 16;

struct Plan {
  uint32_t rt, row_tiles, ranges, heads, turns, max_tiles;
  bool whole;
  size_t ml, o, stats, logits;  // bytes of the scratch's parts
  size_t bytes() const { return ml + o + stats + logits; }
};

size_t padded(size_t n) { return (n + 255) & ~size_t(255); }

int plan_of(int64_t batch, int64_t rows, int64_t hq, int64_t hkv, int64_t d, int64_t max_len, int32_t dtype, bool weights,
            Plan* p) {
  CBK_REQUIRE(batch >= 0 && batch < (1 << 16), "batch out of range");
  CBK_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "query heads must be divisible by KV heads");
  CBK_REQUIRE(rows > 0 && hq < (1 << 16) && rows < (1 << 16) && rows * hq < (int64_t(1) << 31), "rows or heads out of range");
  CBK_REQUIRE(max_len >= 0 && max_len < (int64_t(1) << 31) - 32, "context out of range");
  const int64_t n = rows * (hq / hkv), keys = dtype == CBK_DTYPE_F32 ? 16 : 32;
  p->rt = n <= 16 ? 1 : 2;
  p->row_tiles = uint32_t((n + 16 * p->rt - 1) / (16 * p->rt));
  const uint32_t waves = uint32_t(max_waves(int(p->rt)));
  for (p->heads = waves; hkv % p->heads != 0;) --p->heads;
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  p->max_tiles = uint32_t((max_len + keys - 1) / keys);
  const int64_t most = batch * int64_t(p->max_tiles);
  CBK_REQUIRE(most < (int64_t(1) << 31), "context tiles out of range");
  // Short sequences: a range each, no second launch, the waves of a workgroup
  // taking a head's tiles in turns while that leaves no CU two workgroups.
  uint32_t heads = p->heads;
  for (uint32_t h = p->heads; h > 0; --h)
    if (hkv % h == 0 && batch * (hkv / h) * int64_t(p->row_tiles) <= cus) heads = h;
  const int64_t groups = batch * (hkv / heads) * int64_t(p->row_tiles), turns = waves / heads;
  const int64_t alone = (p->max_tiles + turns - 1) / turns * ((groups + cus - 1) / cus);  // a wave's tiles
  const int64_t cut = (most * hkv * p->row_tiles + int64_t(cus) * waves - 1) / (int64_t(cus) * waves);
  p->whole = alone <= std::min(cut + kMergeTiles, kWholeTiles);
  if (p->whole) {
    p->heads = heads;
    p->turns = uint32_t(turns);
    p->ranges = uint32_t(std::max<int64_t>(batch, 1));
  } else {
    // a workgroup of each CU (registers); fewer where its waves would have less
    // than a tile each
    p->turns = waves / p->heads;
    const int64_t units = hkv / p->heads * int64_t(p->row_tiles);
    int64_t ranges = (int64_t(cus) + units - 1) / units;
    ranges = std::min(ranges, (most + p->turns - 1) / p->turns);
    p->ranges = uint32_t(ranges > 1 ? ranges : 1);
  }
  const size_t all_rows = size_t(rows) * size_t(hq);
  const size_t parts = p->whole ? 0 : size_t(2) * p->ranges * all_rows;
  p->ml = padded(parts * sizeof(float2));
  p->o = padded(parts * size_t(d) * sizeof(float));
  p->stats = weights ? padded(size_t(batch) * all_rows * sizeof(float2)) : 0;
  p->logits = weights ? padded(size_t(most) * size_t(keys) * all_rows * sizeof(float)) : 0;
  return CBK_OK;
}

template <int DT, int D, int RT>
int launch_attn(const PagedAttnArgs& a, hipStream_t s) {
  const uint64_t groups = uint64_t(a.hkv / a.heads) * a.row_tiles * ((a.ranges + 7) / 8 * 8);
  const uint32_t threads = 64 * a.heads * a.turns;
  CBK_REQUIRE(groups * threads < (uint64_t(1) << 32), "paged attention: %llu workgroups exceed one launch",
              (unsigned long long)groups);
  const dim3 grid(uint32_t(groups), 1, 1), block(threads);
  if (a.logits) hipLaunchKernelGGL((paged_attn_kernel<DT, D, RT, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((paged_attn_kernel<DT, D, RT, false>), grid, block, 0, s, a);
  return launch_status("paged attention");
}

template <int DT, int D>
int launch(const PagedAttnArgs& a, const Plan& p, float* weights, int64_t batch_stride, int64_t set_stride, uint32_t sets,
           hipStream_t s) {
  if (int rc = p.rt == 1 ? launch_attn<DT, D, 1>(a, s) : launch_attn<DT, D, 2>(a, s)) return rc;
  if (!a.whole) {
    const dim3 grid(a.rows * a.hq, a.batch);
    if (a.ranges > 16 * a.batch) hipLaunchKernelGGL((paged_attn_merge_kernel<DT, D, 32>), grid, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((paged_attn_merge_kernel<DT, D, 8>), grid, dim3(256), 0, s, a);
    if (int rc = launch_status("paged attention merge")) return rc;
  }
  if (weights == nullptr || a.max_len == 0) return CBK_OK;
  const uint32_t set_rows = a.rows * a.hq / sets;
  auto run = [&](auto kernel, uint32_t keys) {
    hipLaunchKernelGGL(kernel, dim3((a.max_len + keys - 1) / keys, sets, a.batch), dim3(256), 0, s, a, weights, batch_stride,
                       set_stride, sets);
  };
  if (set_rows <= 8) run(key_weights_kernel<DT, 1>, 1024);
  else if (set_rows <= 64) run(key_weights_kernel<DT, 4>, 256);
  else run(key_weights_kernel<DT, 32>, 32);
  return launch_status("key weights");
}

}  // namespace
}  // namespace cbk

extern "C" {

size_t cbk_paged_attention_workspace_bytes(int64_t batch, int64_t rows, int64_t hq, int64_t hkv, int64_t head_dim,
                                           int64_t max_len, int32_t dtype, int32_t key_weights) {
  using namespace cbk;
  Plan p;
  if (batch <= 0 || head_dim <= 0 || plan_of(batch, rows, hq, hkv, head_dim, max_len, dtype, key_weights != 0, &p)) return 0;
  return p.bytes();
}

int cbk_paged_attention(const void* q_dev, int64_t q_batch_stride, int64_t q_row_stride, int64_t q_head_stride,
                        int64_t batch, int64_t rows, int64_t hq, const cbk_kv_desc* kv, int64_t hkv, int64_t head_dim,
                        const int32_t* tables_dev, int64_t table_stride, int64_t table_width, const int32_t* lens_dev,
                        float scale, int32_t dtype, void* out_dev, int64_t out_batch_stride, int64_t out_row_stride,
                        int64_t out_head_stride, float* key_weights_dev, int64_t weights_batch_stride,
                        int64_t weights_set_stride, int64_t weight_sets, void* workspace_dev, size_t workspace_bytes,
                        cbk_stream_t stream) {
  using namespace cbk;
  clear_error();
  if (int rc = validate_desc(kv)) return rc;
  CBK_REQUIRE(dtype == CBK_DTYPE_F32 || dtype == CBK_DTYPE_BF16 || dtype == CBK_DTYPE_F16, "dtype %d", int(dtype));
  CBK_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim %lld: 64 or 128 supported", (long long)head_dim);
  const int64_t es = dtype == CBK_DTYPE_F32 ? 4 : 2;
  CBK_REQUIRE(hkv > 0 && kv->row_bytes == hkv * head_dim * es, "a row of %lld x %lld is not %lld bytes", (long long)hkv,
              (long long)head_dim, (long long)kv->row_bytes);
  CBK_REQUIRE(std::isfinite(scale), "scale must be finite");
  CBK_REQUIRE(table_width >= 0 && table_width < (int64_t(1) << 31) && table_stride >= 0,
              "block table width out of range");
  CBK_REQUIRE(kv->num_blocks < (int64_t(1) << 31), "num_blocks out of range");
  CBK_REQUIRE(key_weights_dev == nullptr || weight_sets == 1 || weight_sets == hkv, "%lld sets of weights for %lld KV heads",
              (long long)weight_sets, (long long)hkv);
  const int64_t max_len = table_width * kv->block_size;
  Plan p;
  if (int rc = plan_of(batch, rows, hq, hkv, head_dim, max_len, dtype, key_weights_dev != nullptr, &p)) return rc;
  if (batch == 0) return CBK_OK;
  CBK_REQUIRE(q_dev && out_dev && lens_dev && (tables_dev || table_width == 0), "NULL pointer");
  const int64_t words[6] = {int64_t(reinterpret_cast<uintptr_t>(kv->k_base)),
                            int64_t(reinterpret_cast<uintptr_t>(kv->v_base)), kv->block_stride, kv->token_stride,
                            int64_t(reinterpret_cast<uintptr_t>(q_dev)), int64_t(reinterpret_cast<uintptr_t>(out_dev))};
  CBK_REQUIRE(common_vec_bytes(words, 6) >= es, "tensors must be aligned to their elements");
  if (workspace_dev == nullptr || workspace_bytes < p.bytes())
    return set_error(CBK_ERR_WORKSPACE, "paged attention workspace %zu < %zu bytes", workspace_bytes, p.bytes());
  CBK_REQUIRE((reinterpret_cast<uintptr_t>(workspace_dev) & 255) == 0, "workspace must be 256-byte aligned");
  PagedAttnArgs a;
  a.q = static_cast<const char*>(q_dev);
  a.out = static_cast<char*>(out_dev);
  a.q_batch = q_batch_stride * es;
  a.q_row = q_row_stride * es;
  a.q_head = q_head_stride * es;
  a.out_batch = out_batch_stride * es;
  a.out_row = out_row_stride * es;
  a.out_head = out_head_stride * es;
  a.k_base = static_cast<const char*>(kv->k_base);
  a.v_base = static_cast<const char*>(kv->v_base);
  a.block_stride = kv->block_stride;
  a.token_stride = kv->token_stride;
  a.tables = tables_dev;
  a.table_stride = table_stride;
  a.lens = lens_dev;
  a.batch = uint32_t(batch);
  a.rows = uint32_t(rows);
  a.hq = uint32_t(hq);
  a.hkv = uint32_t(hkv);
  a.group = uint32_t(hq / hkv);
  a.num_blocks = uint32_t(kv->num_blocks);
  a.max_len = uint32_t(max_len);
  a.max_tiles = p.max_tiles;
  a.row_tiles = p.row_tiles;
  a.ranges = p.ranges;
  a.whole = p.whole;
  a.heads = p.heads;
  a.turns = p.turns;
  a.c = scale * (kLog2e / kUnit);
  a.block_div = FastDiv::make(uint32_t(kv->block_size));
  char* at = static_cast<char*>(workspace_dev);
  a.ml = reinterpret_cast<float2*>(at);
  a.o = reinterpret_cast<float*>(at += p.ml);
  a.stats = p.stats ? reinterpret_cast<float2*>(at + p.o) : nullptr;
  a.logits = p.logits ? reinterpret_cast<float*>(at + p.o + p.stats) : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define CBK_PAGED_ATTN(DT)                                                                                            \
  return head_dim == 128                                                                                              \
             ? launch<DT, 128>(a, p, key_weights_dev, weights_batch_stride, weights_set_stride, uint32_t(weight_sets), s) \
             : launch<DT, 64>(a, p, key_weights_dev, weights_batch_stride, weights_set_stride, uint32_t(weight_sets), s);
  switch (dtype) {
    case CBK_DTYPE_F32: CBK_PAGED_ATTN(CBK_DTYPE_F32)
    case CBK_DTYPE_BF16: CBK_PAGED_ATTN(CBK_DTYPE_BF16)
    default: CBK_PAGED_ATTN(CBK_DTYPE_F16)
  }
#undef CBK_PAGED_ATTN
}

}  // extern "C"
