// Work units of the paged-attention kernels (16-bit, f32 and 4-bit pools): the record a CTA starts from, its
// columns' causal limits, and the merge of its warps' softmax states into final or partial rows.
#pragma once

#include "attn_args.cuh"

namespace mlb {

constexpr float kNegInf = -__builtin_huge_valf();

struct UnitInfo {
  int seq, q0, n_new, L, t0, ncols, pb, pe, part_row;
};

__device__ __forceinline__ UnitInfo unit_info(const AttnArgs& a, int unit_idx) {
  const int4* rec = reinterpret_cast<const int4*>(a.units + unit_idx);  // one 32-byte record, two loads
  const int4 x = __ldg(rec), y = __ldg(rec + 1);
  UnitInfo r;
  r.seq = x.x;
  r.t0 = x.y * a.tile_tokens;
  r.pb = x.z;
  r.pe = x.w;
  r.part_row = y.x;
  r.q0 = y.y;
  r.n_new = y.z;
  r.L = y.w;
  r.ncols = min(a.tile_tokens, r.n_new - r.t0) * a.group;
  return r;
}

// Exclusive key limit of column j: its query token sits at position L - n_new + qi and sees keys up to
// and including itself (causal, aligned to the end of the context; a decode row sees all L keys).
__device__ __forceinline__ int column_limit(const AttnArgs& a, const UnitInfo& ui, int j) {
  if (j >= ui.ncols) return 0;
  return ui.L - ui.n_new + ui.t0 + j / a.group + 1;
}

// Merge the warps' (m, l, O[col][dim]) states and write the unit's result: the final row when the unit
// covers the whole context, else a normalised fp32 partial row plus its log2-sum-exp.
// KEEP_NAN: a NaN sum (a NaN query) gives NaN rows instead of zeros.
template <int DH, int OUT_DT, int NW, bool KEEP_NAN = false>
__device__ __forceinline__ void merge_and_store(const AttnArgs& a, const UnitInfo& ui, int kvh,
                                                const float* const* so, const float* const* sm,
                                                const float* const* sl) {
  constexpr int V = 4, DV = DH / V;  // each thread takes 4 consecutive dims of one column (16-byte reads)
  for (int idx = threadIdx.x; idx < ui.ncols * DV; idx += blockDim.x) {
    const int j = idx / DV, d = (idx % DV) * V;
    float M = kNegInf;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w][j]);
    float lsum = 0.f, acc[V] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = sm[w][j];
      const float e = mw == kNegInf ? 0.f : fast_exp2(mw - M);
      lsum += e * sl[w][j];
      const float4 x = *reinterpret_cast<const float4*>(so[w] + j * DH + d);
      acc[0] += e * x.x;
      acc[1] += e * x.y;
      acc[2] += e * x.z;
      acc[3] += e * x.w;
    }
    const bool some = KEEP_NAN ? lsum != 0.f : lsum > 0.f;
    float val[V];
#pragma unroll
    for (int k = 0; k < V; ++k) val[k] = some ? acc[k] / lsum : 0.f;
    const int qi = ui.t0 + j / a.group;
    const int head = kvh * a.group + j % a.group;
    if (ui.part_row < 0) {
      store_out_n<OUT_DT, V>(a.out, a.out_vec, ui.q0 + qi, head, d, val);
    } else {
      const int64_t row = ui.part_row + j / a.group;
      *reinterpret_cast<float4*>(a.part_o + (row * a.h + head) * DH + d) = make_float4(val[0], val[1], val[2], val[3]);
      if (d == 0) a.part_lse[row * a.h + head] = some ? M + log2f(lsum) : kNegInf;
    }
  }
}

// Opt in to > 48 KB of dynamic shared memory once per kernel instance and device (`done` is the
// caller's per-instance bit set of device ordinals < 64).
template <typename K>
cudaError_t set_smem(K kernel, int bytes, unsigned long long& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (done >> dev) & 1ull) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) __atomic_fetch_or(&done, 1ull << dev, __ATOMIC_RELAXED);
  return e;
}

}  // namespace mlb
