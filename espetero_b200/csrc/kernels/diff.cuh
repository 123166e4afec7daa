// What the kernels of differential attention share: where a record lies and how a row is finished.
//
//   D = O_1 / l_1 - lam O_2 / l_2,   O = out_scale * w * D / sqrt(mean(D^2) + eps)      (w NULL: out_scale * D)
//
// O_c, l_c are the unnormalised sums of map c against its own maximum m_c. Both maps see the same keys, so a row either has two
// sums or none; a row without keys has l = 0 and gets zeros (and 0 * rsqrt(0) must not become NaN with eps = 0).
#pragma once

#include "common.cuh"
#include "../launch.h"

namespace esp {

// First float of the record of (part, kv head, row of the tile, head of the group, map); a record is [O(HD) | m | l].
__device__ __forceinline__ size_t diff_record(const KernelArgs& k, int part, int kvh, int r, int hg, int map) {
  return ((((size_t(part) * k.p.Hkv + kvh) * k.tile_rows + r) * k.G + hg) * 2 + map) * (k.HD + 2);
}

// A row's mask record (segment start, -, ancestors, -), brought into its tree of M rows: records that say "none" or "all" by numbers outside
// it mean the same, and sums with them stay in range.
__device__ __forceinline__ int4 row_record(const KernelArgs& a, int row, int M) {
  int4 d = reinterpret_cast<const int4*>(a.desc)[row];
  d.x = min(max(d.x, 0), M), d.z = min(max(d.z, 0), M);
  return d;
}

// log2 of a (positive) page scale, rounded down, within what references and their differences can hold.
__device__ __forceinline__ float log2_floor(float v) { return fminf(fmaxf(float(int((__float_as_uint(v) >> 23) & 0xFFu) - 127), -100.0f), 100.0f); }

__device__ __forceinline__ float diff_lam(const DiffArgs& a, int row, int h) { return a.lam[size_t(row) * a.lam_ld + h]; }

// The factor that turns D into the normalised row (before the weight), from the sum of D^2 over the head.
__device__ __forceinline__ float diff_row_factor(const DiffArgs& a, float sum_sq, int HD) {
  if (!a.norm_w) return a.out_scale;
  return sum_sq > 0.0f ? a.out_scale * rsqrtf(fmaf(sum_sq, 1.0f / float(HD), a.eps)) : (sum_sq == 0.0f ? 0.0f : sum_sq);  // NaN stays NaN
}

}  // namespace esp
