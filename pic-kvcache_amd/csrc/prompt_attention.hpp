// Packed prompts: the arguments of their attention, and which sequence and row
// tile a workgroup has.
#pragma once

#include "attention_split.hpp"

namespace cbk {

struct PromptArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  // elements
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;
  const int32_t* ends_q;  // [batch + 1]: sequence s has the queries ends_q[s] .. ends_q[s + 1]
  const int32_t* ends_k;
  uint32_t batch, total_q, total_k;
  uint32_t element;  // bytes
  uint32_t hq, hkv, group;
  FastDiv group_div;
  float scale;
  bool zero_outside;  // rows of no sequence become zero, instead of staying as they are
  AttnParts parts;
};

// Row tiles of `rows` (query, group head) rows that any lengths can need, and
// one more: past the last tile workgroups have the rows of no sequence.
inline uint64_t prompt_tiles(const PromptArgs& a, uint32_t rows) {
  return uint64_t(a.total_q) * a.group / rows + a.batch + 1;
}

// Rows of a workgroup of the float32 kernel, for rows of (query, group head): 128,
// which share each K/V block's cutting and LDS reads, from two rounds of 64-row
// workgroups (three a CU) on; below that more and shorter workgroups fill the
// GPU better. us with 64 / 128: 8000 tokens of 32 / 8 heads x 128 2824 / 2506,
// 3000 469 / 404, 2200 237 / 245; 4 of 1000, 16 / 8 heads, 112 / 142.
inline uint32_t prompt_f32_rows(uint64_t rows, uint64_t hkv) { return rows * hkv >= 1536 * 64 ? 128 : 64; }
int launch_prompt_f32(const PromptArgs& a, uint32_t d, hipStream_t stream);

struct PromptTile {
  uint32_t q0, nq, k0, nk;  // of the sequence
  uint32_t tile;            // of its rows
  uint32_t beyond;          // > 0: no tile, the beyond-th such rank of `without`
  uint32_t without;
  bool none;                // no tile, and nothing to do
};

#ifdef __HIPCC__

struct PromptSeq {
  uint32_t q0, nq, k0, nk;
};

// Sequence s; ends past the tensors are taken as their end, and a sequence whose
// end lies before its start is empty. (After ends that fall sequences may overlap,
// and tiles be more than workgroups: rows are then written twice, in either order, or
// not at all, but always within the tensors.)
__device__ __forceinline__ PromptSeq prompt_seq(const PromptArgs& a, uint32_t s) {
  auto at = [](int32_t x, uint32_t total) { return min(uint32_t(max(x, 0)), total); };
  PromptSeq r;
  r.q0 = at(a.ends_q[s], a.total_q);
  r.nq = max(at(a.ends_q[s + 1], a.total_q), r.q0) - r.q0;
  r.k0 = at(a.ends_k[s], a.total_k);
  r.nk = max(at(a.ends_k[s + 1], a.total_k), r.k0) - r.k0;
  return r;
}

// Which sequence and tile workgroup `rank` has. By a whole wave, every wave of a
// workgroup the same.
//
// In general sequence after sequence, each one's highest tile, which has the most
// keys, first. Sequence s has the ranks from ends_q[s] G / ROWS + s on (rounded
// down), as many as it can need or one more, so that its place is found without
// the lengths before it.
//
// A launch of few workgroups (kLeveled) whose sequences' lengths a wave holds:
// the rank-th tile in the order of the tiles' levels, highest first. A tile's
// level counts the tiles of rows up to its last key, so that tiles with about as
// many keys share one, whatever their sequences. The long ones start together,
// and the launch ends with short ones: 32 / 8 heads, head_dim 128, 1416
// workgroups of 8 float32 prompts 70 us and 86 us sequence after sequence, 744
// of them in bf16 29.1 and 31.7; beyond about 2300 workgroups the order costs
// more in keys that leave the L2 (4352 of 64 bf16 prompts 163 us and 150).
constexpr uint32_t kLeveled = 2048;
template <uint32_t ROWS>
__device__ PromptTile prompt_tile(const PromptArgs& a, uint32_t rank, uint32_t lane) {
  PromptTile t;
  t.q0 = t.nq = t.k0 = t.nk = t.tile = t.beyond = t.without = 0;
  t.none = false;
  auto take = [&](uint32_t seq) __attribute__((always_inline)) {
    const PromptSeq q = prompt_seq(a, seq);
    t.q0 = __builtin_amdgcn_readfirstlane(q.q0);
    t.nq = __builtin_amdgcn_readfirstlane(q.nq);
    t.k0 = __builtin_amdgcn_readfirstlane(q.k0);
    t.nk = __builtin_amdgcn_readfirstlane(q.nk);
  };
  const uint32_t ranks = gridDim.x / (a.hkv * a.parts.splits);
  if (a.batch > 1 && a.batch <= 64 && gridDim.x <= kLeveled) {
    // of a lane's sequence (none: no tiles): its lowest level, and one past its highest
    uint32_t lo = 0, hi = 0;
    if (lane < a.batch) {
      const PromptSeq q = prompt_seq(a, lane);
      lo = q.nk > q.nq ? uint32_t(min(uint64_t(q.nk - q.nq) * a.group / ROWS, uint64_t(1) << 30)) : 0u;
      hi = lo + (q.nq * a.group + ROWS - 1) / ROWS;
    }
    auto at_least = [&](uint32_t level) __attribute__((always_inline)) {  // tiles of this level or above
      return uint32_t(__builtin_amdgcn_readlane(int(wave_inclusive_scan(hi - min(max(level, lo), hi))), 63));
    };
    const uint32_t all = at_least(0);
    if (rank >= all) {
      t.beyond = rank - all + 1;
      t.without = ranks - all;
      return t;
    }
    uint32_t low = 0, high = hi;  // the highest level with more than `rank` tiles from it on
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) high = max(high, uint32_t(__shfl_xor(int(high), off)));
    high = __builtin_amdgcn_readfirstlane(high);
    while (high - low > 1) {  // at_least(low) > rank >= at_least(high)
      const uint32_t mid = (low + high) / 2;
      if (at_least(mid) > rank) low = mid;
      else high = mid;
    }
    const uint32_t index = rank - at_least(low + 1);  // within the level, in the sequences' order
    const bool has = lo <= low && low < hi;
    const uint64_t mask = __ballot(has);
    const int seq = __builtin_ctzll(__ballot(has && uint32_t(__popcll(mask & ((uint64_t(1) << lane) - 1))) == index));
    t.tile = low - uint32_t(__builtin_amdgcn_readlane(int(lo), seq));
    take(uint32_t(seq));
    return t;
  }
  auto first_rank = [&](uint32_t s) __attribute__((always_inline)) {
    const uint32_t q0 = min(uint32_t(max(a.ends_q[s], 0)), a.total_q);
    return uint32_t(uint64_t(q0) * a.group / ROWS) + s;
  };
  const uint32_t before = __builtin_amdgcn_readfirstlane(first_rank(0));
  const uint32_t behind = __builtin_amdgcn_readfirstlane(first_rank(a.batch));
  if (rank < before || rank >= behind) {
    t.beyond = (rank < before ? rank : before + rank - behind) + 1;
    t.without = before + ranks - behind;
    return t;
  }
  // the last sequence whose first rank is not past this one, 64 steps at once
  uint32_t seq = 0, n = a.batch;
  while (n > 1) {
    const uint32_t step = (n + 63) / 64, at = lane * step;
    const uint64_t mask = __ballot(at < n && first_rank(seq + min(at, n - 1)) <= rank);
    const uint32_t hit = mask == 0 ? 0 : 63 - uint32_t(__builtin_clzll(mask));
    seq += hit * step;
    n = min(step, n - hit * step);
  }
  take(seq);
  const uint32_t tiles = (t.nq * a.group + ROWS - 1) / ROWS;
  const uint32_t nth = rank - __builtin_amdgcn_readfirstlane(first_rank(seq));
  t.none = nth >= tiles;
  t.tile = tiles - 1 - nth;
  return t;
}

// Zeroes the rows of no sequence, before the first and behind the last: the
// workgroups without a tile share them, each the heads of its KV head. `row`:
// bytes of a head's row, whole 16-byte pieces.
__device__ __forceinline__ void prompt_outside(const PromptArgs& a, const PromptTile& t, uint32_t kvh, uint32_t row) {
  if (!a.zero_outside) return;
  const uint32_t first = min(uint32_t(max(a.ends_q[0], 0)), a.total_q);
  const uint32_t behind = max(min(uint32_t(max(a.ends_q[a.batch], 0)), a.total_q), first);
  const uint32_t per = row / 16, es = a.element;
  const uint64_t n = uint64_t(first + (a.total_q - behind)) * a.group * per;
  for (uint64_t i = uint64_t(t.beyond - 1) * blockDim.x + threadIdx.x; i < n; i += uint64_t(t.without) * blockDim.x) {
    const uint64_t r = i / per;
    const uint32_t piece = uint32_t(i - r * per), at = uint32_t(r / a.group), h = uint32_t(r - uint64_t(at) * a.group);
    const uint32_t token = at < first ? at : behind + (at - first);
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    char* dst = static_cast<char*>(a.out) + (int64_t(token) * a.out_token + int64_t(kvh * a.group + h) * a.out_head) * es;
    reinterpret_cast<u32x4*>(dst)[piece] = u32x4(0u);
  }
}

#endif

}  // namespace cbk
