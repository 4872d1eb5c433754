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
// a run of 32.  Loads and stores are 16 bytes a lane.
#include <algorithm>

#include "fp4.cuh"
#include "row_args.cuh"

namespace mlb {

namespace {

// 8 consecutive elements -> fp32
template <int DT>
__device__ __forceinline__ void load8(const char* p, bool vec, float (&x)[8]) {
  using T = typename Elt<DT>::T;
  if (vec) {
    if constexpr (DT == MLB_F32) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == MLB_BF16) {
          x[2 * i] = __uint_as_float(w[i] << 16);
          x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(reinterpret_cast<const T*>(p)[i]);
  }
}

template <int DT>
__device__ __forceinline__ void store8(char* p, bool vec, const float (&x)[8]) {
  if (vec) {
    if constexpr (DT == MLB_F32) {
      reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]),
                                                pack2<DT>(x[6], x[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) store_f32<DT>(p + i * Elt<DT>::bytes, x[i]);
  }
}

template <int DT>
__device__ __forceinline__ float round_to(float x) {
  if constexpr (DT == MLB_F32) return x;
  if constexpr (DT == MLB_F16) return __half2float(__float2half_rn(x));
  return __bfloat162float(__float2bfloat16_rn(x));
}

// Quantise a lane's two runs of 8 dims (chunks ca and cb of 8; the 4 lanes of a run of 32 are neighbours) and
// store codes and scales of (slot, head).  Every lane of the warp takes part; `live` lanes store.
template <int DH, bool WIDE>
__device__ __forceinline__ void quant_store(uint8_t* pool, int64_t slot, int hkv, int head, int c, float (&a)[8],
                                            float (&b)[8], bool live) {
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
  const float ia = ba ? 1.f / sa : 0.f, ib = bb ? 1.f / sb : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = ba ? fp4_quotient<WIDE>(a[i], sa, ia) : copysignf(0.f, a[i]);
    b[i] = bb ? fp4_quotient<WIDE>(b[i], sb, ib) : copysignf(0.f, b[i]);
  }
  if (!live) return;
  constexpr int HALF = DH / 16;  // chunks of 8 in half a head
  const int t = static_cast<int>(slot % kBlockSize);
  uint8_t* rec = pool + (slot / kBlockSize * hkv + head) * static_cast<int64_t>(Fp4<DH>::kRecord);
  uint32_t* row = reinterpret_cast<uint32_t*>(rec + t * Fp4<DH>::kRow);
  row[c] = fp4_pack8(a);
  row[HALF + c] = fp4_pack8(b);
  if ((c & 3) == 0) {
    rec[Fp4<DH>::kScales + fp4_scale_at(c / 4, t)] = static_cast<uint8_t>(ba);
    rec[Fp4<DH>::kScales + fp4_scale_at((HALF + c) / 4, t)] = static_cast<uint8_t>(bb);
  }
}

// One warp per (token, group of 32 / LANES heads), grid-stride over `reps` groups of a token so that its row of
// the table is read once for several groups.  Heads [0, h) are queries, [h, h + hkv) keys and, with APPEND,
// [h + hkv, h + 2 hkv) values.
template <int DT, int DH, bool APPEND>
__global__ void __launch_bounds__(128) norm_rope_kernel(const RowArgs a, int groups, int reps, int tasks_per_token) {
  constexpr int LANES = DH / 16, PER = 32 / LANES, EB = Elt<DT>::bytes;
  griddep_begin();
  const int lane = threadIdx.x & 31, c = lane % LANES;
  const int64_t task = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int64_t tok = task / tasks_per_token;
  if (tok >= a.num_tokens) return;
  const int g0 = static_cast<int>(task % tasks_per_token) * reps;
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
  float cs[8], sn[8];
  if (turn) {
    const char* row = reinterpret_cast<const char*>(a.cos_sin + pos * a.rot + 8 * c);
    load8<MLB_F32>(row, true, cs);
    load8<MLB_F32>(row + a.rot / 2 * 4, true, sn);
  }
  for (int g = g0; g < g0 + reps && g < groups; ++g) {
    const int head = g * PER + lane / LANES;
    const bool is_q = head < a.h, is_k = !is_q && head < a.h + a.hkv;
    const bool live = is_q || is_k || (APPEND && head < a.h + 2 * a.hkv);
    const int kv_head = is_k ? head - a.h : head - a.h - a.hkv;
    float xa[8], xb[8];
    const char* src = is_q   ? a.q + (tok * a.q_st + head * a.q_sh) * EB
                      : is_k ? a.k + (tok * a.k_st + kv_head * a.k_sh) * EB
                             : a.v + (tok * a.v_st + kv_head * a.v_sh) * EB;
    if (live) {
      load8<DT>(src + da * EB, a.vec, xa);
      load8<DT>(src + db * EB, a.vec, xb);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) xa[i] = xb[i] = 0.f;
    }
    const char* weight = is_q ? a.q_weight : is_k ? a.k_weight : nullptr;
    if (a.q_weight || a.k_weight) {  // uniform: the shuffles below are reached by every lane
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
#pragma unroll
      for (int off = 1; off < LANES; off <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      if (weight) {
        const float r = rsqrtf(ss * (1.f / DH) + a.eps);
        float wa[8], wb[8];
        load8<DT>(weight + da * EB, true, wa);
        load8<DT>(weight + db * EB, true, wb);
#pragma unroll
        for (int i = 0; i < 8; ++i) xa[i] = xa[i] * r * wa[i], xb[i] = xb[i] * r * wb[i];
      }
    }
    if (turn && (is_q || is_k)) {  // products rounded one by one, as the formula reads
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = __fsub_rn(__fmul_rn(xa[i], cs[i]), __fmul_rn(xb[i], sn[i]));
        xb[i] = __fadd_rn(__fmul_rn(xb[i], cs[i]), __fmul_rn(xa[i], sn[i]));
        xa[i] = p;
      }
    }
    if (is_q || (!APPEND && is_k)) {
      char* dst = is_q ? a.q_out + (tok * a.qo_st + head * a.qo_sh) * EB
                       : a.k_out + (tok * a.ko_st + kv_head * a.ko_sh) * EB;
      store8<DT>(dst + da * EB, a.vec, xa);
      store8<DT>(dst + db * EB, a.vec, xb);
    }
    if constexpr (APPEND) {
      // any lane of the warp with a key or value: all of them enter (shuffles inside)
      if (g * PER + PER > a.h) {
        if (is_k) {  // the key is rounded to its own dtype first, as when the two calls are made one by one
#pragma unroll
          for (int i = 0; i < 8; ++i) xa[i] = round_to<DT>(xa[i]), xb[i] = round_to<DT>(xb[i]);
        }
        quant_store<DH, DT == MLB_F32>(is_k ? a.k_cache : a.v_cache, slot, a.hkv, kv_head, c, xa, xb,
                                       live && !is_q && slot_ok);
      }
    }
  }
}

// One group of Dh / 16 lanes per (token, head, K or V) row.
template <int DT, int DH>
__global__ void __launch_bounds__(128) fp4_append_kernel(const RowArgs a) {
  constexpr int LANES = DH / 16, EB = Elt<DT>::bytes;
  griddep_begin();
  const int lane = threadIdx.x & 31, c = lane % LANES;
  const int64_t rows = a.num_tokens * a.hkv * 2;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x / LANES;
  // every lane of a warp makes the same number of turns (shuffles inside)
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x - lane) / LANES;
  for (int64_t r0 = first; r0 < rows; r0 += step) {
    const int64_t r = r0 + lane / LANES;
    const bool live = r < rows;
    const int64_t tok = live ? r / (2 * a.hkv) : 0;
    const int which = static_cast<int>(live ? r % (2 * a.hkv) : 0), head = which % a.hkv;
    const bool is_v = which >= a.hkv;
    float xa[8], xb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) xa[i] = xb[i] = 0.f;
    int64_t slot = -1;
    if (live) {
      slot = a.slots[tok];
      const char* src = is_v ? a.v + (tok * a.v_st + head * a.v_sh) * EB : a.k + (tok * a.k_st + head * a.k_sh) * EB;
      load8<DT>(src + 8 * c * EB, a.vec, xa);
      load8<DT>(src + (DH / 2 + 8 * c) * EB, a.vec, xb);
    }
    const bool ok = slot >= 0 && slot < a.num_slots;
    if (live && !ok && which == 0 && c == 0) flag_error(a.err, MLB_DEV_SLOT_RANGE);
    quant_store<DH, DT == MLB_F32>(is_v ? a.v_cache : a.k_cache, slot, a.hkv, head, c, xa, xb, ok);
  }
}

// Rows of slots as values: one group of Dh / 16 lanes per (token, head, K or V) row; a slot out of range reads 0.
template <int DT, int DH>
__global__ void __launch_bounds__(128) fp4_read_kernel(const RowArgs a) {
  constexpr int LANES = DH / 16, EB = Elt<DT>::bytes;
  griddep_begin();
  const int64_t rows = a.num_tokens * a.hkv * 2;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x / LANES;
  const int c = threadIdx.x % LANES;
  for (int64_t r = at; r < rows; r += step) {
    const int64_t tok = r / (2 * a.hkv);
    const int which = static_cast<int>(r % (2 * a.hkv)), head = which % a.hkv;
    const bool is_v = which >= a.hkv;
    const int64_t slot = a.slots[tok];
    float x[2][8] = {};
    if (slot >= 0 && slot < a.num_slots) {
      const int t = static_cast<int>(slot % kBlockSize);
      const uint8_t* rec = (is_v ? a.v_cache : a.k_cache) +
                           (slot / kBlockSize * a.hkv + head) * static_cast<int64_t>(Fp4<DH>::kRecord);
      const uint2 w = *reinterpret_cast<const uint2*>(rec + t * Fp4<DH>::kRow + 8 * c);  // dims [16c, 16c + 16)
      const float s = fp4_scale_value(rec[Fp4<DH>::kScales + fp4_scale_at(c / 2, t)]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t p[4];
        fp4_unpack8(i ? w.y : w.x, p[0], p[1], p[2], p[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[j]));
          x[i][2 * j] = f.x * s;
          x[i][2 * j + 1] = f.y * s;
        }
      }
    } else if (which == 0 && c == 0) {
      flag_error(a.err, MLB_DEV_SLOT_RANGE);
    }
    char* dst = (is_v ? a.q_out : a.k_out) + ((tok * a.hkv + head) * DH + 16 * c) * EB;
    store8<DT>(dst, true, x[0]);
    store8<DT>(dst + 8 * EB, true, x[1]);
  }
}

template <int DT, int DH>
cudaError_t launch_norm_rope_typed(const RowArgs& a, bool append, int num_sms, cudaStream_t s) {
  constexpr int PER = 32 / (DH / 16);
  const int heads = a.h + (append ? 2 : 1) * a.hkv;
  const int groups = (heads + PER - 1) / PER;
  // a warp takes as many groups of a token as still leaves 16 warps on every SM
  const int64_t warps = std::max<int64_t>(1, static_cast<int64_t>(num_sms) * 16);
  const int reps = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(groups, a.num_tokens * groups / warps)));
  const int tasks = (groups + reps - 1) / reps;
  const int64_t ctas = (a.num_tokens * tasks + 3) / 4;
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  if (append) return launch_k(norm_rope_kernel<DT, DH, true>, dim3(static_cast<unsigned>(ctas)), dim3(128), 0, s, a, groups, reps, tasks);
  return launch_k(norm_rope_kernel<DT, DH, false>, dim3(static_cast<unsigned>(ctas)), dim3(128), 0, s, a, groups, reps, tasks);
}

unsigned row_grid(const RowArgs& a, int dh, int num_sms) {
  const int64_t threads = a.num_tokens * a.hkv * 2 * (dh / 16);
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((threads + 127) / 128, static_cast<int64_t>(num_sms) * 64)));
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

cudaError_t launch_fp4_append(const RowArgs& a, int dtype, int dh, int num_sms, cudaStream_t s) {
#define MLB_CALL(T, D) launch_k(fp4_append_kernel<T, D>, dim3(row_grid(a, dh, num_sms)), dim3(128), 0, s, a)
  MLB_FP4_DISPATCH(MLB_CALL)
#undef MLB_CALL
}

cudaError_t launch_fp4_read(const RowArgs& a, int dtype, int dh, int num_sms, cudaStream_t s) {
#define MLB_CALL(T, D) launch_k(fp4_read_kernel<T, D>, dim3(row_grid(a, dh, num_sms)), dim3(128), 0, s, a)
  MLB_FP4_DISPATCH(MLB_CALL)
#undef MLB_CALL
}

}  // namespace mlb
