// Paged attention over 4-bit pools (fp4.cuh): the per-sequence kernel and the warp-level shared-unit kernel.
//
// Same units, partial rows and reduction as the 16-bit kernel (paged_attention.cu): one CTA = one work unit x one
// KV head, up to 8 query columns, the CTA's warps taking the unit's pages round robin.  What differs is how a page
// reaches the tensor core.  A page of one head is 8.5 Dh contiguous bytes, a quarter of the 16-bit page, and the
// codes are widened in registers, so nothing is staged in shared memory: every lane loads straight from global
// memory the bytes that become its own fragments, NBUF pages ahead, and converts them (one cvt for two values, one
// packed multiply for their scale; code * scale is exact in fp16).
//   S^T[16 tok x 8 col] = K . Q^T: lane (g = lane / 4, t = lane % 4) of an m16n8k16 fragment holds tokens g and
//   g + 8.  The order of the dims inside the products is free as long as Q has the same one, so lane t takes the
//   contiguous dims [t Dh / 4, (t + 1) Dh / 4) of both tokens: one or two 16-byte loads a token, a run of 32 dims
//   is one lane's (Dh 128), and the two tokens' scale bytes are neighbours.
//   O^T[Dh x 8] += V^T . P^T: lane g takes dims [g Dh / 8, (g + 1) Dh / 8) of tokens 2t, 2t + 1, 2t + 8, 2t + 9; a
//   cvt gives two dims of one token, two byte permutes turn two tokens' pairs into the (token, token + 1) pairs of
//   the fragment, which are then multiplied by the tokens' pair of scales.
// All products are fp16 x fp16 with fp32 sums, also for bf16 queries: a query row is first divided by the power of
// two of its largest element (exact: bf16 has 8 significant bits, fp16 11; elements 2^-14 below the row's largest
// and less lose bits that are 2^-25 of it) and the exponent goes into the row's softmax scale.
// P is rounded to fp16 (2^-12 relative), 8 times finer than a bf16 output.
// The running maximum moves only when a page's scores exceed it by more than 8 (a factor 256, far inside fp16), so
// most pages need one vote instead of the maximum over the lanes and no rescaling of O.
#include <climits>

#include "attn_units.cuh"
#include "fp4.cuh"

namespace mlb {

namespace {

constexpr int kFp4Warps = 4;        // warps per CTA of the per-sequence kernel
constexpr int kFp4SharedWarps = 8;  // warps per CTA of the shared-unit kernel

// What one lane holds of a page: its K codes (tokens g, g + 8) and V codes (4 tokens), and their scales.
template <int DH>
struct PageRegs {
  static constexpr int KW = DH / 32, VW = DH / 64 > 0 ? DH / 64 : 1, NKS = DH / 128 > 0 ? DH / 128 : 1;
  uint32_t k[2][KW];
  uint32_t v[4][VW];
  uint32_t ks[NKS];  // scale bytes of tokens g (low) and g + 8
  uint32_t vs;       // scale bytes of tokens 2t, 2t + 8, 2t + 1, 2t + 9
};

template <int W, bool KEEP>
__device__ __forceinline__ void ldg_words(const uint8_t* p, uint32_t* w) {
  if constexpr (W == 1) {
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
  } else if constexpr (W == 2) {
    if constexpr (KEEP)
      asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    else
      asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      if constexpr (KEEP)
        asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                     : "l"(p + 16 * i));
      else
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                     : "l"(p + 16 * i));
    }
  }
}

// Lane-constant offsets into a page record.
template <int DH>
struct LaneOffsets {
  uint32_t k, v, ks, vs;
  __device__ __forceinline__ explicit LaneOffsets(int lane) {
    const int g = lane >> 2, t = lane & 3;
    k = static_cast<uint32_t>(g * Fp4<DH>::kRow + t * (DH / 8));
    v = static_cast<uint32_t>(2 * t * Fp4<DH>::kRow + g * (DH / 16));
    ks = static_cast<uint32_t>(Fp4<DH>::kScales + fp4_scale_at(t * (DH / 4) / kFp4Run, g));
    vs = static_cast<uint32_t>(Fp4<DH>::kScales + fp4_scale_at(g * (DH / 8) / kFp4Run, 2 * t));
  }
};

template <int DH, bool KEEP>
__device__ __forceinline__ void load_page(PageRegs<DH>& p, const uint8_t* krec, const uint8_t* vrec,
                                          const LaneOffsets<DH>& lo) {
  constexpr int ROW = Fp4<DH>::kRow;
  using P = PageRegs<DH>;
  ldg_words<P::KW, KEEP>(krec + lo.k, p.k[0]);
  ldg_words<P::KW, KEEP>(krec + lo.k + 8 * ROW, p.k[1]);
#pragma unroll
  for (int i = 0; i < P::NKS; ++i)
    p.ks[i] = __ldg(reinterpret_cast<const unsigned short*>(krec + lo.ks + i * kBlockSize));
  ldg_words<P::VW, KEEP>(vrec + lo.v, p.v[0]);
  ldg_words<P::VW, KEEP>(vrec + lo.v + ROW, p.v[1]);
  ldg_words<P::VW, KEEP>(vrec + lo.v + 8 * ROW, p.v[2]);
  ldg_words<P::VW, KEEP>(vrec + lo.v + 9 * ROW, p.v[3]);
  p.vs = __ldg(reinterpret_cast<const uint32_t*>(vrec + lo.vs));
}

// The softmax state of a warp's 8 columns; a lane keeps columns 2t and 2t + 1.
template <int DH>
struct Columns {
  uint32_t qb[DH / 16][2];
  float o[DH / 16][4];
  float sl2[2];  // softmax scale * log2(e) * the power of two taken out of the column's query
  float m[2];    // the maximum in use (exp2 domain); -inf: no key seen yet
  float nb[2];   // -m, or 0 while m is -inf
  float l[2];
  int lim[2];    // exclusive key limits
};

// Load up to 8 query columns as B fragments: column n = lane / 4, this lane's dims [t Dh / 4, (t + 1) Dh / 4).
template <int DT, int DH>
__device__ __forceinline__ void load_queries(Columns<DH>& c, const AttnArgs& a, const uint16_t* qrow, bool live, int lane) {
  constexpr int N = DH / 4;
  float f = 1.f;
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
    // biased exponent of the row's largest element, kept where both powers of two are normal numbers
    const int e = max(1, min(static_cast<int>(__float_as_uint(mx) >> 23), 253));
    const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);  // 2^(127 - e)
    f = __uint_as_float(static_cast<uint32_t>(e) << 23);                       // 2^(e - 127)
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint32_t w = c.qb[i >> 1][i & 1];
      c.qb[i >> 1][i & 1] = pack2<MLB_F16>(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
    }
  }
  const float s = a.sl2 * f;
  c.sl2[0] = __shfl_sync(0xffffffffu, s, (lane & 3) * 8);
  c.sl2[1] = __shfl_sync(0xffffffffu, s, (lane & 3) * 8 + 4);
}

template <int DH>
__device__ __forceinline__ void reset_columns(Columns<DH>& c, int lim0, int lim1) {
#pragma unroll
  for (int mt = 0; mt < DH / 16; ++mt) c.o[mt][0] = c.o[mt][1] = c.o[mt][2] = c.o[mt][3] = 0.f;
  c.lim[0] = lim0;
  c.lim[1] = lim1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c.m[i] = c.lim[i] > 0 ? kNegInf : 0.f;  // an absent column never asks for a new maximum
    c.nb[i] = 0.f;
    c.l[i] = 0.f;
  }
}

// One page against the warp's columns.  key0: position of the page's first token; live_rows: tokens of the page
// that the sequence has (the others' V must not reach the product: 0 x NaN).
template <int DH>
__device__ __forceinline__ void attend_fp4_page(Columns<DH>& c, PageRegs<DH>& p, int key0, int live_rows, int lane) {
  constexpr int KW = DH / 32;
  const int t = lane & 3, r0 = lane >> 2;
  float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < KW; ++w) {
    const uint32_t ks = p.ks[w / 4];
    const uint32_t s0 = __byte_perm(ks, 0u, 0x4040) << 7, s1 = __byte_perm(ks, 0u, 0x4141) << 7;  // scale pairs
    uint32_t x[4], y[4];
    fp4_unpack8(p.k[0][w], x[0], x[1], x[2], x[3]);
    fp4_unpack8(p.k[1][w], y[0], y[1], y[2], y[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = hmul2_u32(x[i], s0), y[i] = hmul2_u32(y[i], s1);
    mma16816<MLB_F16>(sa, x[0], y[0], x[1], y[1], c.qb[2 * w][0], c.qb[2 * w][1]);
    mma16816<MLB_F16>(sb, x[2], y[2], x[3], y[3], c.qb[2 * w + 1][0], c.qb[2 * w + 1][1]);
  }
  const int k0 = key0 + r0, k1 = k0 + 8;
  // scores relative to the maximum in use, exp2 domain
  float s00 = sa[0] + sb[0], s01 = sa[1] + sb[1], s10 = sa[2] + sb[2], s11 = sa[3] + sb[3];
  if (k0 >= c.lim[0]) s00 = kNegInf;
  if (k0 >= c.lim[1]) s01 = kNegInf;
  if (k1 >= c.lim[0]) s10 = kNegInf;
  if (k1 >= c.lim[1]) s11 = kNegInf;
  float y00 = fmaf(s00, c.sl2[0], c.nb[0]), y10 = fmaf(s10, c.sl2[0], c.nb[0]);
  float y01 = fmaf(s01, c.sl2[1], c.nb[1]), y11 = fmaf(s11, c.sl2[1], c.nb[1]);
  const float my0 = fmaxf(y00, y10), my1 = fmaxf(y01, y11);
  const bool grow = my0 > 8.f || my1 > 8.f || (c.m[0] == kNegInf && my0 > kNegInf) || (c.m[1] == kNegInf && my1 > kNegInf);
  if (__any_sync(0xffffffffu, grow)) {
    float mx[2] = {my0, my1};
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
      mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
    }
    float al[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float mn = fmaxf(c.m[i], mx[i] - c.nb[i]);  // nb is 0 while m is -inf
      al[i] = c.m[i] == kNegInf ? 0.f : fast_exp2(c.m[i] - mn);
      c.l[i] *= al[i];
      c.m[i] = mn;
      c.nb[i] = mn == kNegInf ? 0.f : -mn;
    }
#pragma unroll
    for (int mt = 0; mt < DH / 16; ++mt) {
      c.o[mt][0] *= al[0];
      c.o[mt][1] *= al[1];
      c.o[mt][2] *= al[0];
      c.o[mt][3] *= al[1];
    }
    y00 = fmaf(s00, c.sl2[0], c.nb[0]), y10 = fmaf(s10, c.sl2[0], c.nb[0]);
    y01 = fmaf(s01, c.sl2[1], c.nb[1]), y11 = fmaf(s11, c.sl2[1], c.nb[1]);
  }
  const float p00 = fast_exp2(y00), p10 = fast_exp2(y10), p01 = fast_exp2(y01), p11 = fast_exp2(y11);
  c.l[0] += p00 + p10;
  c.l[1] += p01 + p11;
  // P (rows = tokens, column pairs) -> P^T as the B operand (token = k, column = n)
  const uint32_t pb0 = movm_t(pack2<MLB_F16>(p00, p01)), pb1 = movm_t(pack2<MLB_F16>(p10, p11));
  uint32_t vs = p.vs;
  if (live_rows < kBlockSize) {  // a zero scale makes a token's values zero whatever its codes are
    const int t0 = 2 * t;
    vs &= (t0 < live_rows ? 0xffu : 0u) | (t0 + 8 < live_rows ? 0xff00u : 0u) | (t0 + 1 < live_rows ? 0xff0000u : 0u) |
          (t0 + 9 < live_rows ? 0xff000000u : 0u);
  }
  const uint32_t v01 = (vs & 0x00ff00ffu) << 7, v89 = (vs & 0xff00ff00u) >> 1;  // pairs (2t, 2t + 1), (2t + 8, 2t + 9)
  constexpr int WORDS = PageRegs<DH>::VW;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    uint32_t x[4], y[4], z[4], u[4];
    fp4_unpack8(p.v[0][w], x[0], x[1], x[2], x[3]);
    fp4_unpack8(p.v[1][w], y[0], y[1], y[2], y[3]);
    fp4_unpack8(p.v[2][w], z[0], z[1], z[2], z[3]);
    fp4_unpack8(p.v[3][w], u[0], u[1], u[2], u[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a0 = hmul2_u32(__byte_perm(x[i], y[i], 0x5410), v01);  // even dim, tokens 2t, 2t + 1
      const uint32_t a1 = hmul2_u32(__byte_perm(x[i], y[i], 0x7632), v01);  // odd dim
      const uint32_t a2 = hmul2_u32(__byte_perm(z[i], u[i], 0x5410), v89);
      const uint32_t a3 = hmul2_u32(__byte_perm(z[i], u[i], 0x7632), v89);
      mma16816<MLB_F16>(c.o[4 * w + i], a0, a1, a2, a3, pb0, pb1);
    }
  }
}

// The warp's pages [0, n) of a table run, one every `stride` entries, loaded NBUF - 1 pages ahead of their use.
// Block ids come 32 at a time, one window ahead.
template <int DH, int NBUF, bool KEEP>
__device__ __forceinline__ void walk_pages(Columns<DH>& c, const AttnArgs& a, const int32_t* table, int first, int n,
                                           int stride, int kvh, int seq_len, int lane) {
  const LaneOffsets<DH> lo(lane);
  const int64_t block_bytes = static_cast<int64_t>(a.hkv) * Fp4<DH>::kRecord;
  const uint8_t* kb = reinterpret_cast<const uint8_t*>(a.k_cache) + kvh * Fp4<DH>::kRecord;
  const uint8_t* vb = reinterpret_cast<const uint8_t*>(a.v_cache) + kvh * Fp4<DH>::kRecord;
  auto load_window = [&](int w) -> int {
    const int i = w * 32 + lane;
    return i < n ? __ldg(table + first + i * stride) : 0;
  };
  int ids = load_window(0), ids_next = load_window(1), win = 0;
  PageRegs<DH> buf[NBUF];
  bool ok[NBUF];
  auto fetch = [&](int j, PageRegs<DH>& p, bool& good) {
    good = false;
    if (j >= n) return;
    if ((j >> 5) != win) {
      ++win;
      ids = ids_next;
      ids_next = load_window(win + 1);
    }
    const int bid = __shfl_sync(0xffffffffu, ids, j & 31);
    good = bid >= 0 && bid < a.num_blocks;
    if (!good) {
      if (lane == 0) flag_error(a.err, MLB_DEV_BLOCK_RANGE);
      return;
    }
    const int64_t off = static_cast<int64_t>(bid) * block_bytes;
    load_page<DH, KEEP>(p, kb + off, vb + off, lo);
  };
#pragma unroll
  for (int b = 0; b < NBUF - 1; ++b) fetch(b, buf[b], ok[b]);
  for (int i = 0; i < n; i += NBUF) {
#pragma unroll
    for (int b = 0; b < NBUF; ++b) {
      fetch(i + b + NBUF - 1, buf[(b + NBUF - 1) % NBUF], ok[(b + NBUF - 1) % NBUF]);
      if (i + b < n && ok[b]) {
        const int key0 = (first + (i + b) * stride) * kBlockSize;
        attend_fp4_page<DH>(c, buf[b], key0, seq_len - key0, lane);
      }
    }
  }
}

template <int DT, int DH, int NBUF, int NW, int MINB>
__global__ void __launch_bounds__(NW * 32, MINB) paged_attn_fp4_kernel(AttnArgs a) {
  __shared__ __align__(16) float so[NW][8 * DH];
  __shared__ float sm[NW][8], sl[NW][8];
  griddep_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x % a.hkv;
  const UnitInfo ui = unit_info(a, blockIdx.x / a.hkv);
  const int first = ui.pb + warp;
  const int npages = first < ui.pe ? (ui.pe - first + NW - 1) / NW : 0;
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
  walk_pages<DH, NBUF, false>(c, a, a.bt + static_cast<int64_t>(ui.seq) * a.bt_stride, first, npages, NW, kvh, ui.L, lane);
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    c.l[0] += __shfl_xor_sync(0xffffffffu, c.l[0], off);
    c.l[1] += __shfl_xor_sync(0xffffffffu, c.l[1], off);
  }
  // lane g holds dims [g Dh / 8, (g + 1) Dh / 8) of its two columns
  const int d0 = (lane >> 2) * (DH / 8);
#pragma unroll
  for (int mt = 0; mt < DH / 16; ++mt) {
    *reinterpret_cast<float2*>(&so[warp][j0 * DH + d0 + 2 * mt]) = make_float2(c.o[mt][0], c.o[mt][2]);
    *reinterpret_cast<float2*>(&so[warp][j1 * DH + d0 + 2 * mt]) = make_float2(c.o[mt][1], c.o[mt][3]);
  }
  if (lane < 4) {
    sm[warp][j0] = c.m[0];
    sm[warp][j1] = c.m[1];
    sl[warp][j0] = c.l[0];
    sl[warp][j1] = c.l[1];
  }
  __syncthreads();
  const float *so_w[NW], *sm_w[NW], *sl_w[NW];
#pragma unroll
  for (int w = 0; w < NW; ++w) so_w[w] = so[w], sm_w[w] = sm[w], sl_w[w] = sl[w];
  merge_and_store<DH, DT, NW, true>(a, ui, kvh, so_w, sm_w, sl_w);
}

// Shared units (mlb_shared_unit: a shared prefix's member rows, or a query tile of a multi-token row) without the
// tensor-core kernel's layout requirements: each warp takes 8 columns of the unit and walks all of its pages, which
// the CTA's warps find in L1 / L2 after the first of them.
template <int DT, int DH>
__global__ void __launch_bounds__(kFp4SharedWarps * 32) shared_fp4_kernel(AttnArgs a) {
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
    walk_pages<DH, 2, true>(c, a, a.bt + static_cast<int64_t>(tseq) * a.bt_stride, pb, pe - pb, 1, kvh, seq_len, lane);
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
        if (lane < 4) a.part_lse[row * a.h + head] = c.l[i] == 0.f ? kNegInf : c.m[i] + log2f(c.l[i]);
      }
    }
  }
}

}  // namespace

cudaError_t launch_fp4_attention(const AttnArgs& a, int dtype, int dh, int64_t num_units, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(num_units * a.hkv)), block(kFp4Warps * 32);
  if (dtype == MLB_BF16) {
    if (dh == 64) return launch_k(paged_attn_fp4_kernel<MLB_BF16, 64, 2, kFp4Warps, 4>, grid, block, 0, s, a);
    if (dh == 128) return launch_k(paged_attn_fp4_kernel<MLB_BF16, 128, 2, kFp4Warps, 4>, grid, block, 0, s, a);
    if (dh == 256) return launch_k(paged_attn_fp4_kernel<MLB_BF16, 256, 2, kFp4Warps, 2>, grid, block, 0, s, a);
  } else if (dtype == MLB_F16) {
    if (dh == 64) return launch_k(paged_attn_fp4_kernel<MLB_F16, 64, 2, kFp4Warps, 4>, grid, block, 0, s, a);
    if (dh == 128) return launch_k(paged_attn_fp4_kernel<MLB_F16, 128, 2, kFp4Warps, 4>, grid, block, 0, s, a);
    if (dh == 256) return launch_k(paged_attn_fp4_kernel<MLB_F16, 256, 2, kFp4Warps, 2>, grid, block, 0, s, a);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_fp4_shared(const AttnArgs& a, int dtype, int dh, int64_t num_units, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(num_units * a.hkv)), block(kFp4SharedWarps * 32);
  if (dtype == MLB_BF16) {
    if (dh == 64) return launch_k(shared_fp4_kernel<MLB_BF16, 64>, grid, block, 0, s, a);
    if (dh == 128) return launch_k(shared_fp4_kernel<MLB_BF16, 128>, grid, block, 0, s, a);
    if (dh == 256) return launch_k(shared_fp4_kernel<MLB_BF16, 256>, grid, block, 0, s, a);
  } else if (dtype == MLB_F16) {
    if (dh == 64) return launch_k(shared_fp4_kernel<MLB_F16, 64>, grid, block, 0, s, a);
    if (dh == 128) return launch_k(shared_fp4_kernel<MLB_F16, 128>, grid, block, 0, s, a);
    if (dh == 256) return launch_k(shared_fp4_kernel<MLB_F16, 256>, grid, block, 0, s, a);
  }
  return cudaErrorInvalidValue;
}

}  // namespace mlb
