// Row operators around the 4-bit pools: the norm of each query / key head with the rotation by position, the
// quantising append, both in one launch, and the read-back of rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                        (norm: optional, weights of the row's dtype)
//   out[i] = y[i] c - y[i + r/2] s,  out[i + r/2] = y[i + r/2] c + y[i] s,  i < r / 2, (c, s) = table[position]
//   dims >= r pass; all in fp32, one rounding to the row's dtype.
//   stored: scale = max|x| of 32 dims / 6 in the byte format, code = x / scale in e2m1 (fp4.cuh).
//
// All of them are bound by memory for many rows and by latency for few.  A head is Dh / 16 lanes; each lane holds
// two runs of 8 dims, [8c, 8c + 8) and [r/2 + 8c, r/2 + 8c + 8): the two halves of its rotation pairs, so nothing
// is exchanged but the sum of squares (log2(Dh / 16) shuffles) and, for the codes, the maximum over the 4 lanes of
// a run of 32.  Loads and stores are 16 bytes a lane.  Heads of 128 dims: rotating 8192 tokens of 32 + 8 heads takes
// 31 us, 5.5 TB/s (with norms 33), and 64 tokens with norms 2.3 us; appending 16384 tokens of 8 heads 17 us and reading
// them back 15, 5.3 TB/s over both; norm, rotation and append of 4001 tokens of 28 + 4 heads 15 us (14 without norms).
// fp32 rows, twice the bytes: 60, 38, 38 and 33 us; the append is then bound by quant_store_any's quotients.
#include <algorithm>

#include "fp4.cuh"
#include "row_args.cuh"

namespace mlb {

namespace {

// 8 consecutive elements as they lie in memory: four pairs (16-bit types) or eight fp32.  VEC: 16-byte loads and stores
// (a template parameter: as a branch, the element-wise loads were predicated off and still issued).
template <int DT>
struct Run8 {
  static constexpr int kWords = DT == MLB_F32 ? 8 : 4;
  uint32_t w[kWords];

  template <bool VEC>
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 x = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
      }
    } else if constexpr (DT == MLB_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
      const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = static_cast<uint32_t>(e[2 * i]) | (static_cast<uint32_t>(e[2 * i + 1]) << 16);
    }
  }
  template <bool VEC>
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if constexpr (DT == MLB_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        reinterpret_cast<uint16_t*>(p)[2 * i] = static_cast<uint16_t>(w[i]);
        reinterpret_cast<uint16_t*>(p)[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (DT == MLB_F32) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (DT == MLB_BF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {  // rounds to the type
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (DT == MLB_F32)
        w[i] = __float_as_uint(x[i]);
      else
        w[i] = pack2<DT>(x[2 * i], x[2 * i + 1]);
    }
  }
};

// Where a row of a 4-bit pool lies: its record and its token in the block.
template <int DH>
struct SlotRow {
  uint8_t* rec;
  int t;
  __device__ __forceinline__ SlotRow(uint8_t* pool, int64_t slot, int hkv, int head)
      : rec(pool + (static_cast<uint64_t>(slot) / kBlockSize * hkv + head) * Fp4<DH>::kRecord),
        t(static_cast<int>(slot) & (kBlockSize - 1)) {}
};

template <int DH>
__device__ __forceinline__ void store_codes(const SlotRow<DH>& at, int c, uint32_t wa, uint32_t wb, uint32_t ba, uint32_t bb) {
  constexpr int HALF = DH / 16;  // chunks of 8 dims in half a head
  uint32_t* row = reinterpret_cast<uint32_t*>(at.rec + at.t * Fp4<DH>::kRow);
  row[c] = wa;
  row[HALF + c] = wb;
  if ((c & 3) == 0) {
    at.rec[Fp4<DH>::kScales + fp4_scale_at(c / 4, at.t)] = static_cast<uint8_t>(ba);
    at.rec[Fp4<DH>::kScales + fp4_scale_at((HALF + c) / 4, at.t)] = static_cast<uint8_t>(bb);
  }
}

// Quantise a lane's two runs of 8 dims (chunks c and DH / 16 + c of 8; the 4 lanes of a run of 32 are neighbours) and
// store codes and scales of a row.  Every lane of the warp takes part; `live` lanes store.  fp32 values, any of them
// possibly NaN or out of range.
template <int DH>
__device__ void quant_store_any(const SlotRow<DH>& at, int c, float (&a)[8], float (&b)[8], bool live) {
  float ma = 0.f, mb = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = a[i] == a[i] ? fminf(fmaxf(a[i], -kFp4TopValue), kFp4TopValue) : 0.f;  // NaN is stored as 0
    b[i] = b[i] == b[i] ? fminf(fmaxf(b[i], -kFp4TopValue), kFp4TopValue) : 0.f;
    ma = fmaxf(ma, fabsf(a[i]));
    mb = fmaxf(mb, fabsf(b[i]));
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    ma = fmaxf(ma, __shfl_xor_sync(0xffffffffu, ma, off));
    mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, off));
  }
  const uint32_t ba = fp4_scale_byte(ma), bb = fp4_scale_byte(mb);
  const float sa = fp4_scale_value(ba), sb = fp4_scale_value(bb);
  float ha, la, hb, lb;
  fp4_reciprocal(sa, ha, la);
  fp4_reciprocal(sb, hb, lb);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = fp4_quotient_32(a[i], sa, ha, la);
    b[i] = fp4_quotient_32(b[i], sb, hb, lb);
  }
  if (live) store_codes<DH>(at, c, fp4_pack8(a), fp4_pack8(b), ba, bb);
}

template <int DT, int DH>
__device__ __forceinline__ void quant_store(const SlotRow<DH>& at, int c, const Run8<DT>& ra, const Run8<DT>& rb, bool live) {
  float a[8], b[8];
  if constexpr (DT == MLB_F32) {
    ra.get(a);
    rb.get(b);
    quant_store_any<DH>(at, c, a, b, live);
  } else {
    // the largest magnitudes as integers, two at a time (the order of positive fp16 / bf16 is that of their bits, NaN
    // above all), then both runs' in one word through the two shuffles
    uint32_t ma = 0u, mb = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ma = __vmaxu2(ma, ra.w[i] & 0x7fff7fffu);
      mb = __vmaxu2(mb, rb.w[i] & 0x7fff7fffu);
    }
    uint32_t m = __vmaxu2(__byte_perm(ma, mb, 0x5410), __byte_perm(ma, mb, 0x7632));  // low: run a, high: run b
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    constexpr uint32_t kTop = DT == MLB_BF16 ? 0x4770u : 0x7b80u;  // 61440
    ra.get(a);
    rb.get(b);
    if (__any_sync(0xffffffffu, (m & 0xffffu) > kTop || (m >> 16) > kTop)) {  // NaN, infinity or a large value
      quant_store_any<DH>(at, c, a, b, live);
      return;
    }
    float fa, fb;
    if constexpr (DT == MLB_BF16) {
      fa = __uint_as_float(m << 16);
      fb = __uint_as_float(m & 0xffff0000u);
    } else {
      fa = __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
      fb = __half2float(__ushort_as_half(static_cast<unsigned short>(m >> 16)));
    }
    const uint32_t ba = fp4_scale_byte_16(fa), bb = fp4_scale_byte_16(fb);
    float ha, la, hb, lb;
    fp4_reciprocal(fp4_scale_value(ba), ha, la);
    fp4_reciprocal(fp4_scale_value(bb), hb, lb);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      fp4_quotients_16(a[i], a[i + 1], ha, la);
      fp4_quotients_16(b[i], b[i + 1], hb, lb);
    }
    if (live) store_codes<DH>(at, c, fp4_pack8(a), fp4_pack8(b), ba, bb);
  }
}

// One warp per (token, group of 32 / LANES heads of one kind: queries, keys or, with APPEND, values), over `reps`
// groups of a token so that its row of the table is read once for several groups.  (A group's rows loaded while the
// one before is worked on: no gain without APPEND, and a quarter longer with it, where the registers cost a wave.)
template <int DT, int DH, bool APPEND, bool VEC>
__global__ void __launch_bounds__(128) norm_rope_kernel(const RowArgs a, int reps, int tasks_per_token) {
  constexpr int LANES = DH / 16, PER = 32 / LANES, EB = Elt<DT>::bytes;
  griddep_begin();
  const int lane = threadIdx.x & 31, c = lane % LANES;
  const uint32_t task = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;  // at most 2^31 threads a launch
  const int64_t tok = task / static_cast<uint32_t>(tasks_per_token);
  if (tok >= a.num_tokens) return;
  const int gq = (a.h + PER - 1) / PER, gk = (a.hkv + PER - 1) / PER, groups = gq + (APPEND ? 2 : 1) * gk;
  const int g0 = static_cast<int>(task % static_cast<uint32_t>(tasks_per_token)) * reps, g_end = min(g0 + reps, groups);
  const int64_t pos = a.positions[tok];
  int64_t slot = 0;
  if constexpr (APPEND) slot = a.slots[tok];
  const bool pos_ok = pos >= 0 && pos < a.num_positions;
  const bool slot_ok = !APPEND || (slot >= 0 && slot < a.num_slots);
  if (lane == 0 && g0 == 0) {
    if (!pos_ok) flag_error(a.err, MLB_DEV_POSITION_RANGE);
    if (!slot_ok) flag_error(a.err, MLB_DEV_SLOT_RANGE);
  }
  if (!pos_ok) return;
  // this lane's dims: two runs of 8; lanes past the rotated part hold two neighbouring runs that pass
  const bool turn = c < a.rot / 16;
  const int da = turn ? 8 * c : a.rot + 16 * (c - a.rot / 16);
  const int db = turn ? a.rot / 2 + 8 * c : da + 8;
  Run8<MLB_F32> cs, sn;
  if (turn && g0 < gq + gk) {
    const char* row = reinterpret_cast<const char*>(a.cos_sin + pos * a.rot + 8 * c);
    cs.load<true>(row);
    sn.load<true>(row + a.rot / 2 * 4);
  } else {
    cs.zero();
    sn.zero();
  }
  for (int g = g0; g < g_end; ++g) {
    const int kind = g < gq ? 0 : !APPEND || g < gq + gk ? 1 : 2;  // uniform: the same for the whole warp
    const int head = (g - (kind == 0 ? 0 : kind == 1 ? gq : gq + gk)) * PER + lane / LANES;
    const bool live = head < (kind == 0 ? a.h : a.hkv);
    const char* src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const int64_t st = kind == 0 ? a.q_st : kind == 1 ? a.k_st : a.v_st;
    const int64_t sh = kind == 0 ? a.q_sh : kind == 1 ? a.k_sh : a.v_sh;
    Run8<DT> ra, rb;
    if (live) {
      src += (tok * st + head * sh) * EB;
      ra.template load<VEC>(src + da * EB);
      rb.template load<VEC>(src + db * EB);
    } else {
      ra.zero();
      rb.zero();
    }
    if (kind < 2) {  // values pass as they are
      float xa[8], xb[8];
      ra.get(xa);
      rb.get(xb);
      const char* weight = kind == 0 ? a.q_weight : a.k_weight;
      if (weight) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
#pragma unroll
        for (int off = 1; off < LANES; off <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
        const float r = rsqrtf(ss * (1.f / DH) + a.eps);
        Run8<DT> w;
        float f[8];
        w.template load<true>(weight + da * EB);
        w.get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) xa[i] = xa[i] * r * f[i];
        w.template load<true>(weight + db * EB);
        w.get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) xb[i] = xb[i] * r * f[i];
      }
      if (turn) {  // products rounded one by one, as the formula reads
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float co = __uint_as_float(cs.w[i]), si = __uint_as_float(sn.w[i]);
          const float p = __fsub_rn(__fmul_rn(xa[i], co), __fmul_rn(xb[i], si));
          xb[i] = __fadd_rn(__fmul_rn(xb[i], co), __fmul_rn(xa[i], si));
          xa[i] = p;
        }
      }
      ra.set(xa);  // a key's rounding to its own dtype, as when the two calls are made one by one
      rb.set(xb);
      if (live && (kind == 0 || !APPEND)) {
        char* dst = kind == 0 ? a.q_out + (tok * a.qo_st + head * a.qo_sh) * EB
                              : a.k_out + (tok * a.ko_st + head * a.ko_sh) * EB;
        ra.template store<VEC>(dst + da * EB);
        rb.template store<VEC>(dst + db * EB);
      }
    }
    if constexpr (APPEND) {
      if (kind > 0)
        quant_store<DT, DH>(SlotRow<DH>(kind == 1 ? a.k_cache : a.v_cache, slot_ok ? slot : 0, a.hkv, live ? head : 0), c,
                            ra, rb, live && slot_ok);
    }
  }
}

// One group of Dh / 16 lanes per (token, head): its K row and its V row, which lie at the same place of their pools.
// Bound by instructions (75% of the issue slots, half of them quotients and their roundings): 20 us for the 16384
// tokens above, cold, whose bytes take 13.
template <int DT, int DH, bool VEC>
__global__ void __launch_bounds__(128) fp4_append_kernel(const RowArgs a) {
  constexpr int LANES = DH / 16, EB = Elt<DT>::bytes;
  griddep_begin();
  const int lane = threadIdx.x & 31, c = lane % LANES;
  const uint32_t hkv = static_cast<uint32_t>(a.hkv);
  const uint32_t row = (blockIdx.x * blockDim.x + threadIdx.x) / LANES;  // at most 2^31 threads a launch
  const bool in = row < static_cast<uint32_t>(a.num_tokens) * hkv;
  const uint32_t tok = in ? row / hkv : 0;
  const int head = static_cast<int>(in ? row - tok * hkv : 0);
  Run8<DT> ka, kb, va, vb;
  int64_t slot = -1;
  if (in) {
    slot = a.slots[tok];
    const char* k = a.k + (tok * a.k_st + head * a.k_sh + 8 * c) * EB;
    const char* v = a.v + (tok * a.v_st + head * a.v_sh + 8 * c) * EB;
    ka.template load<VEC>(k);
    kb.template load<VEC>(k + DH / 2 * EB);
    va.template load<VEC>(v);
    vb.template load<VEC>(v + DH / 2 * EB);
  } else {
    ka.zero();
    kb.zero();
    va.zero();
    vb.zero();
  }
  const bool ok = slot >= 0 && slot < a.num_slots;
  if (in && !ok && head == 0 && c == 0) flag_error(a.err, MLB_DEV_SLOT_RANGE);
  SlotRow<DH> at(a.k_cache, ok ? slot : 0, a.hkv, head);
  quant_store<DT, DH>(at, c, ka, kb, ok);
  at.rec += a.v_cache - a.k_cache;
  quant_store<DT, DH>(at, c, va, vb, ok);
}

// Rows of slots as values: one group of Dh / 16 lanes per (token, head), its K row and its V row, two runs of
// 8 dims each a lane (neighbouring lanes store neighbouring 16 bytes: with 16 dims in one run, every store filled half
// of its 32-byte sectors and the kernel took 23 us instead of 17 for 16384 tokens of 8 heads of 128 dims); a slot out of
// range reads 0.
template <int DT, int DH>
__global__ void __launch_bounds__(128) fp4_read_kernel(const RowArgs a) {
  constexpr int LANES = DH / 16, EB = Elt<DT>::bytes;
  griddep_begin();
  const uint32_t hkv = static_cast<uint32_t>(a.hkv);
  const uint32_t row = (blockIdx.x * blockDim.x + threadIdx.x) / LANES;  // at most 2^31 threads a launch
  if (row >= static_cast<uint32_t>(a.num_tokens) * hkv) return;
  const int c = threadIdx.x % LANES;
  const uint32_t tok = row / hkv;
  const int head = static_cast<int>(row - tok * hkv);
  const int64_t slot = a.slots[tok];
  uint32_t w[2][2] = {}, scale[2][2] = {};  // [K, V][this lane's two runs of 8 dims]
  if (slot >= 0 && slot < a.num_slots) {
    const SlotRow<DH> at(a.k_cache, slot, a.hkv, head);
    const int64_t to_v = a.v_cache - a.k_cache;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* codes = at.rec + at.t * Fp4<DH>::kRow + 4 * (i * LANES + c);
      const uint8_t* s = at.rec + Fp4<DH>::kScales + fp4_scale_at((i * LANES + c) / 4, at.t);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        w[kv][i] = *reinterpret_cast<const uint32_t*>(codes + (kv ? to_v : 0));
        scale[kv][i] = s[kv ? to_v : 0];
      }
    }
  } else if (head == 0 && c == 0) {
    flag_error(a.err, MLB_DEV_SLOT_RANGE);
  }
  const int64_t dst = (static_cast<int64_t>(row) * DH + 8 * c) * EB;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t s2 = scale[kv][i] * 0x00010001u << 7;
      Run8<MLB_F16> h;  // code * scale is exact in fp16 (and the wider types)
      fp4_unpack8(w[kv][i], h.w[0], h.w[1], h.w[2], h.w[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) h.w[j] = hmul2_u32(h.w[j], s2);
      char* to = (kv ? a.q_out : a.k_out) + dst + i * (DH / 2) * EB;
      if constexpr (DT == MLB_F16) {
        h.template store<true>(to);
      } else {
        float x[8];
        h.get(x);
        Run8<DT> r;
        r.set(x);
        r.template store<true>(to);
      }
    }
  }
}

template <int DT, int DH>
cudaError_t launch_norm_rope_typed(const RowArgs& a, bool append, int num_sms, cudaStream_t s) {
  constexpr int PER = 32 / (DH / 16);
  const int groups = (a.h + PER - 1) / PER + (append ? 2 : 1) * ((a.hkv + PER - 1) / PER);
  // a warp takes as many groups of a token as still leaves 16 warps for every SM (with APPEND and the read-back, 4001
  // tokens of 28 + 4 heads: 8 to 24 warps 20.3 us, 32 23.5, 96 24.5; without, 8192 tokens of 32 + 8: 31 us for all)
  const int64_t warps = std::max<int64_t>(1, static_cast<int64_t>(num_sms) * 16);
  const int reps = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(groups, a.num_tokens * groups / warps)));
  const int tasks = (groups + reps - 1) / reps;
  const int64_t ctas = (a.num_tokens * tasks + 3) / 4;
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(ctas)), block(128);
  if (append)
    return a.vec ? launch_k(norm_rope_kernel<DT, DH, true, true>, grid, block, 0, s, a, reps, tasks)
                 : launch_k(norm_rope_kernel<DT, DH, true, false>, grid, block, 0, s, a, reps, tasks);
  return a.vec ? launch_k(norm_rope_kernel<DT, DH, false, true>, grid, block, 0, s, a, reps, tasks)
               : launch_k(norm_rope_kernel<DT, DH, false, false>, grid, block, 0, s, a, reps, tasks);
}

// one lane group per (token, head)
unsigned row_grid(const RowArgs& a, int dh) {
  return static_cast<unsigned>((a.num_tokens * a.hkv * (dh / 16) + 127) / 128);
}

template <int DT, int DH>
cudaError_t launch_append_typed(const RowArgs& a, cudaStream_t s) {
  const dim3 grid(row_grid(a, DH)), block(128);
  return a.vec ? launch_k(fp4_append_kernel<DT, DH, true>, grid, block, 0, s, a)
               : launch_k(fp4_append_kernel<DT, DH, false>, grid, block, 0, s, a);
}

}  // namespace

#define MLB_FP4_DISPATCH(CALL)                   \
  if (dtype == MLB_BF16) {                       \
    if (dh == 64) return CALL(MLB_BF16, 64);     \
    if (dh == 128) return CALL(MLB_BF16, 128);   \
    if (dh == 256) return CALL(MLB_BF16, 256);   \
  } else if (dtype == MLB_F16) {                 \
    if (dh == 64) return CALL(MLB_F16, 64);      \
    if (dh == 128) return CALL(MLB_F16, 128);    \
    if (dh == 256) return CALL(MLB_F16, 256);    \
  } else if (dtype == MLB_F32) {                 \
    if (dh == 64) return CALL(MLB_F32, 64);      \
    if (dh == 128) return CALL(MLB_F32, 128);    \
    if (dh == 256) return CALL(MLB_F32, 256);    \
  }                                              \
  return cudaErrorInvalidValue;

cudaError_t launch_norm_rope(const RowArgs& a, int dtype, int dh, bool append, int num_sms, cudaStream_t s) {
#define MLB_CALL(T, D) launch_norm_rope_typed<T, D>(a, append, num_sms, s)
  MLB_FP4_DISPATCH(MLB_CALL)
#undef MLB_CALL
}

cudaError_t launch_fp4_append(const RowArgs& a, int dtype, int dh, cudaStream_t s) {
#define MLB_CALL(T, D) launch_append_typed<T, D>(a, s)
  MLB_FP4_DISPATCH(MLB_CALL)
#undef MLB_CALL
}

cudaError_t launch_fp4_read(const RowArgs& a, int dtype, int dh, cudaStream_t s) {
#define MLB_CALL(T, D) launch_k(fp4_read_kernel<T, D>, dim3(row_grid(a, D)), dim3(128), 0, s, a)
  MLB_FP4_DISPATCH(MLB_CALL)
#undef MLB_CALL
}

}  // namespace mlb
