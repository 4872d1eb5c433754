// Paged attention over 4-bit pools (fp4.cuh): the per-sequence kernel and the warp-level shared-unit kernel.
//
// Same units, partial rows and reduction as the 16-bit kernel (paged_attention.cu): one CTA = one work unit x one
// KV head, up to 8 query columns, the CTA's warps taking the unit's pages round robin, each through a private ring
// of shared-memory slots.  A page of one head is 8.5 Dh contiguous bytes (a quarter of the 16-bit page), so a slot
// is one run of K and one of V; the codes are widened in registers (one cvt for two values, one packed multiply for
// their scale; code * scale is exact in fp16) and never written back.
//   S^T[16 tok x 8 col] = K . Q^T: lane (g = lane / 4, t = lane % 4) of an m16n8k16 fragment holds tokens g and
//   g + 8.  The order of the dims inside the products is free as long as Q has the same one, so lane t takes the
//   contiguous dims [t Dh / 4, (t + 1) Dh / 4) of both tokens: one or two 16-byte loads a token, a run of 32 dims
//   is one lane's (Dh 128), and the two tokens' scale bytes are neighbours.
//   O^T[Dh x 8] += V^T . P^T: lane g takes dims [g Dh / 8, (g + 1) Dh / 8) of tokens 2t, 2t + 1, 2t + 8, 2t + 9; a
//   exchange of nibbles between two tokens' words makes bytes of one dim and two tokens, so that a cvt gives the
//   (token, token + 1) pairs of the fragment, which are then multiplied by the tokens' pair of scales.
// All products are fp16 x fp16 with fp32 sums, also for bf16 queries: a query row is first divided by a power of two
// that brings its largest element to [2^14, 2^15) (exact: bf16 has 8 significant bits, fp16 11; only elements 2^-31
// below the row's largest and less lose bits) and the exponent goes into the row's softmax scale (fp4.cuh).
// P is rounded to fp16: 2^-11 relative, 8 times finer than a bf16 output, for weights down to 2^-24 of the largest, on a
// grid of 2^-34 of it below (kFp4Lift).  The running maximum moves only when a page's scores exceed the one it was taken
// from by more than 4 (kFp4Rise), so most pages need one vote instead of the maximum over the lanes and no rescaling of
// O; only pages on an edge (the row's end, a causal limit) test their keys.
// What bounds it: bytes for long rows, the conversions' instructions and a CTA's start and end for short ones.  32 + 8
// heads of 128 dims: 16 rows of 131072 tokens 386 us, 5.9 TB/s (90% of a copy; repeated for seconds 450, the SM clock
// then lowered from 1965 to 1690 MHz by the power limit, so it is the instructions that count there too); 64 rows of
// 512..4096 tokens 40.5 us, 3.9 TB/s, issue slots 60% busy (16-bit pools 97 us); one row of 32001 tokens 17 us.
// 4 warps a CTA and 4 CTAs an SM: 5 or 6 CTAs spill, and 2 or 8 warps a CTA were slower.
#include <climits>

#include "attn_units.cuh"
#include "fp4.cuh"

namespace mlb {

namespace {

constexpr int kFp4Warps = 4;        // warps per CTA of the per-sequence kernel
constexpr int kFp4SharedWarps = 8;  // warps per CTA of the shared-unit kernel

// Shared-memory ring of a warp: two slots of two pages of one head; a page is its K record, then its V record.  Two
// pages a step halve what a step costs beside its conversions (the softmax's vote, the copies' waits, the loop): 370
// instructions a page with one page a step, 259 with two (and 870 a warp for its start and the merge).
template <int DH>
struct Ring {
  static constexpr int kPageBytes = 2 * Fp4<DH>::kRecord;
  static constexpr int kSlotBytes = 2 * kPageBytes;
  static constexpr int kBytes = 2 * kSlotBytes;
  static_assert(8 * DH * 4 <= kBytes, "the merge state takes the ring's place");
};

// W words from shared memory
template <int W>
__device__ __forceinline__ void lds_words(uint32_t p, uint32_t* w) {
  if constexpr (W == 1) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(p));
  } else if constexpr (W == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(p));
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                   : "r"(p + 16 * i));
  }
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t p) {
  uint16_t x;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(p));
  return x;
}

__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// D = A . B + C (fp16, fp32 sums); not volatile, so that the compiler may mix products and conversions
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Lane-constant offsets into a page.
template <int DH>
struct LaneOffsets {
  uint32_t k, v, ks, vs;
  __device__ __forceinline__ explicit LaneOffsets(int lane) {
    const int g = lane >> 2, t = lane & 3;
    k = static_cast<uint32_t>(g * Fp4<DH>::kRow + t * (DH / 8));
    v = static_cast<uint32_t>(Fp4<DH>::kRecord + 2 * t * Fp4<DH>::kRow + g * (DH / 16));
    ks = static_cast<uint32_t>(Fp4<DH>::kScales + fp4_scale_at(t * (DH / 4) / kFp4Run, g));
    vs = static_cast<uint32_t>(Fp4<DH>::kRecord + Fp4<DH>::kScales + fp4_scale_at(g * (DH / 8) / kFp4Run, 2 * t));
  }
};

// The softmax state of a warp's 8 columns; a lane keeps columns 2t and 2t + 1.
template <int DH>
struct Columns {
  uint32_t qb[DH / 16][2];
  float o[DH / 16][4];
  float sl2[2];  // softmax scale * log2(e) * the power of two taken out of the column's query
  float nb[2];   // minus the exponent taken off every score (exp2 domain; the maximum in use less kFp4Lift), or kUnset
  float l[2];
  int lim[2];  // exclusive key limits
  int all;     // the smallest limit of the warp's live columns: pages below it are seen whole
  // before a column has seen a key: any finite score lies above it, so the first page sets it
  static constexpr float kUnset = 1e30f;
  __device__ __forceinline__ float m(int i) const { return nb[i] == kUnset ? kNegInf : -nb[i]; }
};

// Load up to 8 query columns as B fragments: column n = lane / 4, this lane's dims [t Dh / 4, (t + 1) Dh / 4).
template <int DT, int DH>
__device__ __forceinline__ void load_queries(Columns<DH>& c, const AttnArgs& a, const uint16_t* qrow, bool live, int lane) {
  constexpr int N = DH / 4;
  float s = a.sl2;
  if (live) {
    const uint16_t* src = qrow + (lane & 3) * N;
    uint32_t w[N / 2];
    if (a.q_vec) {
#pragma unroll
      for (int i = 0; i < N / 8; ++i) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(src) + i);
        w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        w[i] = static_cast<uint32_t>(__ldg(src + 2 * i)) | (static_cast<uint32_t>(__ldg(src + 2 * i + 1)) << 16);
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) c.qb[i >> 1][i & 1] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) c.qb[i >> 1][i & 1] = 0u;
  }
  if constexpr (DT == MLB_BF16) {
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint32_t w = c.qb[i >> 1][i & 1];
      mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    float up, down;
    fp4_query_scale(mx, up, down);
    s = fp4_softmax_scale(s, up);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint32_t w = c.qb[i >> 1][i & 1];
      c.qb[i >> 1][i & 1] = pack2<MLB_F16>(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
    }
  }
  c.sl2[0] = __shfl_sync(0xffffffffu, s, (lane & 3) * 8);
  c.sl2[1] = __shfl_sync(0xffffffffu, s, (lane & 3) * 8 + 4);
}

template <int DH>
__device__ __forceinline__ void reset_columns(Columns<DH>& c, int lim0, int lim1) {
#pragma unroll
  for (int mt = 0; mt < DH / 16; ++mt) c.o[mt][0] = c.o[mt][1] = c.o[mt][2] = c.o[mt][3] = 0.f;
  c.lim[0] = lim0;
  c.lim[1] = lim1;
  c.all = INT_MAX;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c.nb[i] = c.lim[i] > 0 ? c.kUnset : 0.f;  // an absent column (zero query) never asks for a new maximum
    c.l[i] = 0.f;
    if (c.lim[i] > 0) c.all = min(c.all, c.lim[i]);
  }
  c.all = __reduce_min_sync(0xffffffffu, c.all);
}

// S^T of two pages: rows = tokens g, g + 8, columns 2t, 2t + 1.  The pages take turns, so that a product's latency
// passes under the other page's conversions.
template <int DH>
__device__ __forceinline__ void page_scores(const Columns<DH>& c, uint32_t slot, const LaneOffsets<DH>& lo, float (&s)[2][4]) {
  constexpr int KW = DH / 32;
  uint32_t kw[2][2][KW], ks[2] = {0u, 0u};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t page = slot + h * Ring<DH>::kPageBytes;
    lds_words<KW>(page + lo.k, kw[h][0]);
    lds_words<KW>(page + lo.k + 8 * Fp4<DH>::kRow, kw[h][1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[h][i] = 0.f;
  }
#pragma unroll
  for (int w = 0; w < KW; ++w) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (w % 4 == 0) ks[h] = lds_u16(slot + h * Ring<DH>::kPageBytes + lo.ks + w / 4 * kBlockSize);
      const uint32_t s0 = __byte_perm(ks[h], 0u, 0x4040) << 7, s1 = __byte_perm(ks[h], 0u, 0x4141) << 7;  // scale pairs
      uint32_t x[4], y[4];
      fp4_unpack8(kw[h][0][w], x[0], x[1], x[2], x[3]);
      fp4_unpack8(kw[h][1][w], y[0], y[1], y[2], y[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = hmul2_u32(x[i], s0), y[i] = hmul2_u32(y[i], s1);
      mma_f16(s[h], x[0], y[0], x[1], y[1], c.qb[2 * w][0], c.qb[2 * w][1]);
      mma_f16(s[h], x[2], y[2], x[3], y[3], c.qb[2 * w + 1][0], c.qb[2 * w + 1][1]);
    }
  }
}

// the low nibbles of a and the high nibbles of b, in one logic operation
__device__ __forceinline__ uint32_t low_nibbles_or_high(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, 0x0f0f0f0f, 0xe4;" : "=r"(d) : "r"(a), "r"(b));  // (a & mask) | (b & ~mask)
  return d;
}

// O^T += V^T . P^T of one page; its scale bytes are those of tokens 2t, 2t + 8, 2t + 1, 2t + 9.
template <int DH>
struct PageV {
  uint32_t w[4][DH / 64];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
  uint32_t scales;
  __device__ __forceinline__ void load(uint32_t page, const LaneOffsets<DH>& lo) {
    constexpr int VW = DH / 64, ROW = Fp4<DH>::kRow;
    lds_words<VW>(page + lo.v, w[0]);
    lds_words<VW>(page + lo.v + ROW, w[1]);
    lds_words<VW>(page + lo.v + 8 * ROW, w[2]);
    lds_words<VW>(page + lo.v + 9 * ROW, w[3]);
    lds_words<1>(page + lo.vs, &scales);
  }
};

template <int DH>
__device__ __forceinline__ void page_output(Columns<DH>& c, const PageV<DH>& v, uint32_t pb0, uint32_t pb1) {
  constexpr int VW = DH / 64;
  const uint32_t(&vw)[4][VW] = v.w;
  // pairs of scales: tokens (2t, 2t + 1), (2t + 8, 2t + 9)
  const uint32_t v01 = (v.scales & 0x00ff00ffu) << 7, v89 = (v.scales & 0xff00ff00u) >> 1;
#pragma unroll
  for (int w = 0; w < VW; ++w) {
    // a byte of a token holds two dims of it; the fragment wants one dim of two tokens: exchange the nibbles of the
    // two tokens' words first (4 logic operations for 16 values), then every cvt gives a pair as it is used
    uint32_t e01[4], d01[4], e89[4], d89[4];
    const uint32_t even01 = low_nibbles_or_high(vw[0][w], vw[1][w] << 4);
    const uint32_t odd01 = low_nibbles_or_high(vw[0][w] >> 4, vw[1][w]);
    const uint32_t even89 = low_nibbles_or_high(vw[2][w], vw[3][w] << 4);
    const uint32_t odd89 = low_nibbles_or_high(vw[2][w] >> 4, vw[3][w]);
    fp4_unpack8(even01, e01[0], e01[1], e01[2], e01[3]);
    fp4_unpack8(odd01, d01[0], d01[1], d01[2], d01[3]);
    fp4_unpack8(even89, e89[0], e89[1], e89[2], e89[3]);
    fp4_unpack8(odd89, d89[0], d89[1], d89[2], d89[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      mma_f16(c.o[4 * w + i], hmul2_u32(e01[i], v01), hmul2_u32(d01[i], v01), hmul2_u32(e89[i], v89),
              hmul2_u32(d89[i], v89), pb0, pb1);
  }
}

// Two neighbouring pages (a ring slot) against the warp's columns.  key0: position of the first page's first token;
// rows: tokens from there that the sequence has (the others' V must not reach the product: 0 x NaN); ok: bit h set
// when page h exists and its block id is good.
template <int DH>
__device__ __forceinline__ void attend_fp4_pages(Columns<DH>& c, uint32_t slot, const LaneOffsets<DH>& lo, int key0, int rows,
                                                 uint32_t ok, int lane) {
  constexpr int PAGE = Ring<DH>::kPageBytes;
  const bool edge = ok != 3u || key0 + 2 * kBlockSize > c.all || rows < 2 * kBlockSize;  // uniform
  float s[2][4];
  page_scores<DH>(c, slot, lo, s);
  PageV<DH> v[2];
  v[0].load(slot, lo);
  v[1].load(slot + PAGE, lo);
  if (edge) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool good = (ok >> h) & 1u;
      const int l0 = good ? c.lim[0] : 0, l1 = good ? c.lim[1] : 0, live = good ? rows - h * kBlockSize : 0;
      const int k0 = key0 + h * kBlockSize + (lane >> 2), k1 = k0 + 8, t0 = 2 * (lane & 3);
      if (k0 >= l0) s[h][0] = kNegInf;
      if (k0 >= l1) s[h][1] = kNegInf;
      if (k1 >= l0) s[h][2] = kNegInf;
      if (k1 >= l1) s[h][3] = kNegInf;
      // a zero scale makes a token's values zero whatever its codes are
      v[h].scales &= (t0 < live ? 0xffu : 0u) | (t0 + 8 < live ? 0xff00u : 0u) | (t0 + 1 < live ? 0xff0000u : 0u) |
                     (t0 + 9 < live ? 0xff000000u : 0u);
    }
  }
  // scores less the columns' exponents, exp2 domain
  float y[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[h][i] = fmaf(s[h][i], c.sl2[i & 1], c.nb[i & 1]);
  const float top = fmaxf(fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[0][2], y[0][3])),
                          fmaxf(fmaxf(y[1][0], y[1][1]), fmaxf(y[1][2], y[1][3])));
  if (__any_sync(0xffffffffu, top > kFp4Lift + kFp4Rise)) {
    float mx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(fmaxf(s[0][i], s[0][i + 2]), fmaxf(s[1][i], s[1][i + 2])) * c.sl2[i];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], off));
    }
    float al[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float m = c.m(i), mn = fmaxf(m, mx[i] - kFp4Lift);
      al[i] = m == kNegInf ? 0.f : fast_exp2(m - mn);
      c.l[i] *= al[i];
      c.nb[i] = mn == kNegInf ? c.kUnset : -mn;
    }
#pragma unroll
    for (int mt = 0; mt < DH / 16; ++mt) {
      c.o[mt][0] *= al[0];
      c.o[mt][1] *= al[1];
      c.o[mt][2] *= al[0];
      c.o[mt][3] *= al[1];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) y[h][i] = fmaf(s[h][i], c.sl2[i & 1], c.nb[i & 1]);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float p0 = fast_exp2(y[h][0]), p1 = fast_exp2(y[h][1]), p2 = fast_exp2(y[h][2]), p3 = fast_exp2(y[h][3]);
    c.l[0] += p0 + p2;
    c.l[1] += p1 + p3;
    // P (rows = tokens, column pairs) -> P^T as the B operand (token = k, column = n)
    page_output<DH>(c, v[h], movm_t(pack2<MLB_F16>(p0, p1)), movm_t(pack2<MLB_F16>(p2, p3)));
  }
}

// Pairs of neighbouring pages of a table run, the first at `first`, one every `stride` pages up to page `end`, each
// copied into the warp's ring while the pair before it is attended (16-byte cp.async, one commit group a pair).
// Block ids come 32 (16 pairs) at a time, one window ahead.
template <int DH>
__device__ __forceinline__ void walk_pages(Columns<DH>& c, const AttnArgs& a, const int32_t* table, int first, int end,
                                           int stride, int kvh, int seq_len, const uint8_t* ring_ptr, int lane) {
  constexpr int CH = Fp4<DH>::kRecord / 16;
  const LaneOffsets<DH> lo(lane);
  const int n = first < end ? (end - first + stride - 1) / stride : 0;
  const uint32_t block_units = static_cast<uint32_t>(a.hkv) * CH;  // a block in 16-byte units (the host checks the range)
  // a page's chunks of 16 bytes: K's, then V's; V's source is at a fixed distance from K's
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.k_cache) + kvh * Fp4<DH>::kRecord + lane * 16;
  const int64_t to_v = a.v_cache - a.k_cache - Fp4<DH>::kRecord;
  const int64_t to_mixed = lane < CH % 32 ? 0 : to_v;  // the 32 chunks that hold K's end and V's start
  const uint32_t ring = smem_u32(ring_ptr);
  // lane 2j + h holds the block id of page h of the window's pair j; -1: no such page
  auto load_window = [&](int w) -> int {
    const int page = first + (w * 16 + (lane >> 1)) * stride + (lane & 1);
    return page < end ? __ldg(table + page) : -1;
  };
  uint32_t good = 0;  // ballot of the window's usable ids
  uint32_t offs = 0;  // this lane's page of the window, as an offset in 16-byte units
  auto take_window = [&](int w, int raw) {
    const bool use = raw >= 0 && raw < a.num_blocks;
    if (!use && first + (w * 16 + (lane >> 1)) * stride + (lane & 1) < end) flag_error(a.err, MLB_DEV_BLOCK_RANGE);
    good = __ballot_sync(0xffffffffu, use);
    offs = use ? static_cast<uint32_t>(raw) * block_units : 0u;  // an unusable page's copy reads block 0, unseen
  };
  int ids_next = load_window(0);
  take_window(0, ids_next);
  ids_next = load_window(1);
  auto issue = [&](int j, uint32_t slot) -> uint32_t {
    uint32_t ok = 0;
    if (j < n) {
      if (j > 0 && (j & 15) == 0) {
        take_window(j >> 4, ids_next);
        ids_next = load_window((j >> 4) + 1);
      }
      ok = (good >> (2 * (j & 15))) & 3u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* src = kb + static_cast<uint64_t>(__shfl_sync(0xffffffffu, offs, 2 * (j & 15) + h)) * 16u;
        const uint8_t *src_mixed = src + to_mixed, *src_v = src + to_v;
        const uint32_t dst = slot + h * Ring<DH>::kPageBytes + lane * 16;
#pragma unroll
        for (int i = 0; i < (2 * CH + 31) / 32; ++i) {
          const uint8_t* from = i < CH / 32 ? src : i == CH / 32 && CH % 32 ? src_mixed : src_v;
          if (2 * CH >= 32 * (i + 1) || lane < 2 * CH - 32 * i) cp_async16_at(dst + i * 512, from + i * 512);
        }
      }
    }
    cp_async_commit();
    return ok;
  };
  int key0 = first * kBlockSize;
  uint32_t ok = issue(0, ring);
  // one pair: refill the other slot (pair j - 1 used it), wait for this lane's copies of pair j and every other
  // lane's, attend, and hold the warp until every lane is done with the slot
  auto step = [&](int j, uint32_t slot, uint32_t other) {
    const uint32_t ok_next = issue(j + 1, other);
    cp_async_wait<1>();
    __syncwarp();
    if (ok) attend_fp4_pages<DH>(c, slot, lo, key0, seq_len - key0, ok, lane);
    __syncwarp();
    ok = ok_next;
    key0 += stride * kBlockSize;
  };
  for (int j = 0; j < n; j += 2) {
    step(j, ring, ring + Ring<DH>::kSlotBytes);
    if (j + 1 < n) step(j + 1, ring + Ring<DH>::kSlotBytes, ring);
  }
  cp_async_wait<0>();
  __syncwarp();
}

template <int DT, int DH, int NW, int MINB>
__global__ void __launch_bounds__(NW * 32, MINB) paged_attn_fp4_kernel(AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm[NW][8], sl[NW][8];
  griddep_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x % a.hkv;
  const UnitInfo ui = unit_info(a, blockIdx.x / a.hkv);
  Columns<DH> c;
  {
    const int n = lane >> 2;
    const bool live = n < ui.ncols;
    const int tok = ui.q0 + ui.t0 + (live ? n / a.group : 0);
    const int head = kvh * a.group + (live ? n % a.group : 0);
    load_queries<DT, DH>(c, a, reinterpret_cast<const uint16_t*>(a.q) + static_cast<int64_t>(tok) * a.q_st +
                                   static_cast<int64_t>(head) * a.q_sh, live, lane);
  }
  const int j0 = (lane & 3) * 2, j1 = j0 + 1;
  reset_columns<DH>(c, column_limit(a, ui, j0), column_limit(a, ui, j1));
  uint8_t* ring = smem + warp * Ring<DH>::kBytes;
  walk_pages<DH>(c, a, a.bt + static_cast<int64_t>(ui.seq) * a.bt_stride, ui.pb + 2 * warp, ui.pe, 2 * NW, kvh, ui.L, ring, lane);
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    c.l[0] += __shfl_xor_sync(0xffffffffu, c.l[0], off);
    c.l[1] += __shfl_xor_sync(0xffffffffu, c.l[1], off);
  }
  // lane g holds dims [g Dh / 8, (g + 1) Dh / 8) of its two columns
  const int d0 = (lane >> 2) * (DH / 8);
  float* so = reinterpret_cast<float*>(ring);  // the warp's own ring: every copy into it has been consumed
#pragma unroll
  for (int mt = 0; mt < DH / 16; ++mt) {
    *reinterpret_cast<float2*>(&so[j0 * DH + d0 + 2 * mt]) = make_float2(c.o[mt][0], c.o[mt][2]);
    *reinterpret_cast<float2*>(&so[j1 * DH + d0 + 2 * mt]) = make_float2(c.o[mt][1], c.o[mt][3]);
  }
  if (lane < 4) {
    sm[warp][j0] = c.m(0);
    sm[warp][j1] = c.m(1);
    sl[warp][j0] = c.l[0];
    sl[warp][j1] = c.l[1];
  }
  __syncthreads();
  const float *so_w[NW], *sm_w[NW], *sl_w[NW];
#pragma unroll
  for (int w = 0; w < NW; ++w) so_w[w] = reinterpret_cast<const float*>(smem + w * Ring<DH>::kBytes), sm_w[w] = sm[w], sl_w[w] = sl[w];
  merge_and_store<DH, DT, NW, true>(a, ui, kvh, so_w, sm_w, sl_w);
}

// Shared units (mlb_shared_unit: a shared prefix's member rows, or a query tile of a multi-token row) without the
// tensor-core kernel's layout requirements: each warp takes 8 columns of the unit and walks all of its pages (L2
// holds them for the CTA's other warps).
template <int DT, int DH>
__global__ void __launch_bounds__(kFp4SharedWarps * 32) shared_fp4_kernel(AttnArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  griddep_begin();
  constexpr int NW = kFp4SharedWarps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x % a.hkv;
  const int4* rec = reinterpret_cast<const int4*>(a.shared_units + blockIdx.x / a.hkv);
  const int4 x = __ldg(rec), y = __ldg(rec + 1);
  const int mb = x.x, mc = x.y, pb = x.z, pe = x.w, piece = y.x, tseq = y.y;
  const bool tile_unit = (y.z & 0xff) == 1;  // kind 1: tokens mb .. mb + mc - 1 of sequence tseq, causal keys
  const int tile_pieces = y.z >> 8, tile_part_base = y.w;
  const int seq_len = tile_unit ? __ldg(a.seq_lens + tseq) : INT_MAX;
  const int first_pos = tile_unit ? seq_len - (__ldg(a.qo + tseq + 1) - __ldg(a.qo + tseq)) + (mb - __ldg(a.qo + tseq))
                                  : 0;
  const bool final_rows = tile_unit && piece < 0;
  const int mpw = a.group >= 8 ? 1 : 8 / a.group;  // member rows per warp
  for (int wm = warp * mpw; wm < mc; wm += NW * mpw) {
    const int ncols = min(mpw, mc - wm) * a.group;
    Columns<DH> c;
    {
      const int n = lane >> 2;
      const bool live = n < ncols;
      const int tok = !live ? 0 : tile_unit ? mb + wm + n / a.group : __ldg(&a.members[mb + wm + n / a.group].q0);
      const int head = kvh * a.group + (live ? n % a.group : 0);
      load_queries<DT, DH>(c, a, reinterpret_cast<const uint16_t*>(a.q) + static_cast<int64_t>(tok) * a.q_st +
                                     static_cast<int64_t>(head) * a.q_sh, live, lane);
    }
    const int j0 = (lane & 3) * 2;
    const int l0 = j0 >= ncols ? 0 : tile_unit ? first_pos + wm + j0 / a.group + 1 : INT_MAX;
    const int l1 = j0 + 1 >= ncols ? 0 : tile_unit ? first_pos + wm + (j0 + 1) / a.group + 1 : INT_MAX;
    reset_columns<DH>(c, l0, l1);
    walk_pages<DH>(c, a, a.bt + static_cast<int64_t>(tseq) * a.bt_stride, pb, pe, 2, kvh, seq_len,
                   smem + warp * Ring<DH>::kBytes, lane);
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      c.l[0] += __shfl_xor_sync(0xffffffffu, c.l[0], off);
      c.l[1] += __shfl_xor_sync(0xffffffffu, c.l[1], off);
    }
    const int d0 = (lane >> 2) * (DH / 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = j0 + i;
      if (j >= ncols) continue;
      const float inv = c.l[i] == 0.f ? 0.f : 1.f / c.l[i];  // a NaN sum stays one
      const int m = wm + j / a.group, head = kvh * a.group + j % a.group;
      if (final_rows) {
#pragma unroll
        for (int mt = 0; mt < DH / 16; ++mt) {
          store_out1<DT>(a.out, mb + m, head, d0 + 2 * mt, c.o[mt][i] * inv);
          store_out1<DT>(a.out, mb + m, head, d0 + 2 * mt + 1, c.o[mt][2 + i] * inv);
        }
      } else {
        const int64_t row = tile_unit ? tile_part_base + (static_cast<int64_t>(m) * tile_pieces + piece) * a.tile_tokens
                                      : __ldg(&a.members[mb + m].part_base) + static_cast<int64_t>(piece) * a.tile_tokens;
        if (row < 0 || row >= a.part_rows) {  // a plan inconsistent with the workspace
          flag_error(a.err, MLB_DEV_BLOCK_RANGE);
          continue;
        }
        float* dst = a.part_o + (row * a.h + head) * DH + d0;
#pragma unroll
        for (int mt = 0; mt < DH / 16; ++mt)
          *reinterpret_cast<float2*>(dst + 2 * mt) = make_float2(c.o[mt][i] * inv, c.o[mt][2 + i] * inv);
        if (lane < 4) a.part_lse[row * a.h + head] = c.l[i] == 0.f ? kNegInf : c.m(i) + log2f(c.l[i]);
      }
    }
  }
}

template <int DT, int DH>
cudaError_t launch_rows(const AttnArgs& a, int64_t num_units, cudaStream_t s) {
  constexpr int bytes = kFp4Warps * Ring<DH>::kBytes;
  static unsigned long long done = 0;
  auto k = paged_attn_fp4_kernel<DT, DH, kFp4Warps, DH == 256 ? 2 : 4>;
  const cudaError_t e = set_smem(k, bytes, done);
  if (e != cudaSuccess) return e;
  return launch_k(k, dim3(static_cast<unsigned>(num_units * a.hkv)), dim3(kFp4Warps * 32), bytes, s, a);
}

template <int DT, int DH>
cudaError_t launch_shared(const AttnArgs& a, int64_t num_units, cudaStream_t s) {
  constexpr int bytes = kFp4SharedWarps * Ring<DH>::kBytes;
  static unsigned long long done = 0;
  auto k = shared_fp4_kernel<DT, DH>;
  const cudaError_t e = set_smem(k, bytes, done);
  if (e != cudaSuccess) return e;
  return launch_k(k, dim3(static_cast<unsigned>(num_units * a.hkv)), dim3(kFp4SharedWarps * 32), bytes, s, a);
}

}  // namespace

cudaError_t launch_fp4_attention(const AttnArgs& a, int dtype, int dh, int64_t num_units, cudaStream_t s) {
  if (dtype == MLB_BF16) {
    if (dh == 64) return launch_rows<MLB_BF16, 64>(a, num_units, s);
    if (dh == 128) return launch_rows<MLB_BF16, 128>(a, num_units, s);
    if (dh == 256) return launch_rows<MLB_BF16, 256>(a, num_units, s);
  } else if (dtype == MLB_F16) {
    if (dh == 64) return launch_rows<MLB_F16, 64>(a, num_units, s);
    if (dh == 128) return launch_rows<MLB_F16, 128>(a, num_units, s);
    if (dh == 256) return launch_rows<MLB_F16, 256>(a, num_units, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_fp4_shared(const AttnArgs& a, int dtype, int dh, int64_t num_units, cudaStream_t s) {
  if (dtype == MLB_BF16) {
    if (dh == 64) return launch_shared<MLB_BF16, 64>(a, num_units, s);
    if (dh == 128) return launch_shared<MLB_BF16, 128>(a, num_units, s);
    if (dh == 256) return launch_shared<MLB_BF16, 256>(a, num_units, s);
  } else if (dtype == MLB_F16) {
    if (dh == 64) return launch_shared<MLB_F16, 64>(a, num_units, s);
    if (dh == 128) return launch_shared<MLB_F16, 128>(a, num_units, s);
    if (dh == 256) return launch_shared<MLB_F16, 256>(a, num_units, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace mlb
