// Equal ranges of the key tiles of a batch's sequences: the tiles of all
// sequences, one after another, cut into as many pieces as fill the GPU, whatever
// sequences they belong to.
#pragma once

#include "cbk_common.hpp"

namespace cbk {
namespace {

// The tiles [first, end) of range r of `total` tiles.
struct Ranges {
  uint32_t each, more;  // tiles of a range; ranges that have one more
  __device__ __forceinline__ Ranges(uint32_t total, uint32_t ranges) : each(total / ranges), more(total % ranges) {}
  __device__ __forceinline__ uint32_t first(uint32_t r) const { return r * each + min(r, more); }
  __device__ __forceinline__ uint32_t of(uint32_t tile) const {
    const uint32_t big = more * (each + 1);
    return tile < big ? tile / (each + 1) : more + (tile - big) / each;
  }
};

__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
  return uint32_t(__builtin_amdgcn_readlane(int(wave_inclusive_scan(v)), 63));
}

}  // namespace
}  // namespace cbk
