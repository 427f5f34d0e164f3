// Shared device helpers of the masked attention kernels (attn_mask_fwd.hip, attn_mask_bwd.hip): fragment types of the two
// storage types, the LDS tile with its swizzle, staging through registers, and the description of a call.
#pragma once
#include "common.h"
#include "../../include/dcamd.h"

namespace dcm {

typedef _Float16 half;
template <typename T> struct Vec;
template <> struct Vec<bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
};
template <> struct Vec<half> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
};

__device__ __forceinline__ f32x16 mfma(Vec<bf16>::v8 a, Vec<bf16>::v8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(Vec<half>::v8 a, Vec<half>::v8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// A call as the kernels see it; lengths in rows, ld* in elements.
struct Call {
  const void *q, *k, *v, *dout;
  void *o, *dq, *dk, *dv;
  float* lse;
  int ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
  int nb, tq, tk, heads, kvh, grp, d;
  float scale, mul;       // score scale; what turns a score into the exponent of 2: scale log2 e, or 1 where the scores are shaped
  float cap2, icap;       // softcap log2 e, 2 log2 e scale / softcap (0: none)
  const float* slopes;
  int causal;
  const int *prefix, *kv_len, *doc_q, *doc_k;
  const int4 *sum_q, *sum_k;   // per 64 rows: least and largest document, whether a row is in none
};

// Scores of a call with a cap or a distance bias, in units of log2: s = cap2 tanh(scale s / cap), then - slope |pos - key|.
// tanh(x) = 1 - 2 / (1 + e^2x): absolute error below 2e-7, so the exponent is off by under 1e-5 at cap = 50.
__device__ __forceinline__ float cap_score(const Call& p, float s, float* slope) {
  const float t = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + exp2_raw(s * p.icap));
  if (slope) *slope = 1.0f - t * t;
  return t * p.cap2;
}

// ---------------------------------------------------------------- LDS tiles
// [rows][DP] elements, 16-byte chunk c of row r at chunk c ^ sw(r): the fragment reads (one chunk of 16 consecutive rows) and the
// transposed reads (four chunks of four rows) both meet all 64 banks once.
template <int DP>
__device__ __forceinline__ int sw(int r) {
  if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return ((r & 3) << 2) | ((r >> 2) & 3);
}
template <int DP>
__device__ __forceinline__ int tile_at(int r, int chunk) { return r * DP + ((chunk ^ sw<DP>(r)) << 3); }

// Where a lane's two transposed reads start for rows key_base.. and columns col_base..: element j of the fragment is row
// key_base + 8 (j >> 2) + 4 (lane >> 5) + (j & 3), the order in which a 32x32 accumulator holds its rows.
struct TrAt { int lo, hi; };
template <int DP>
__device__ __forceinline__ TrAt tr_at(int col_base, int lane) {
  const int g = lane >> 4, i = lane & 15;
  const int col = col_base + 16 * (g & 1) + 4 * (i & 3);
  const int r = 4 * (lane >> 5) + (i >> 2);
  return TrAt{tile_at<DP>(r, col >> 3) + (col & 7), tile_at<DP>(r + 8, col >> 3) + (col & 7)};
}
__device__ __forceinline__ Vec<bf16>::v8 tr_frag(const bf16* tile, TrAt o) {
  const auto a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((DC_LDS bf16x4*)(tile + o.lo));
  const auto b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((DC_LDS bf16x4*)(tile + o.hi));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ Vec<half>::v8 tr_frag(const half* tile, TrAt o) {
  typedef __fp16 h4 __attribute__((ext_vector_type(4)));
  const auto a = __builtin_amdgcn_ds_read_tr16_b64_v4f16((DC_LDS h4*)(tile + o.lo));
  const auto b = __builtin_amdgcn_ds_read_tr16_b64_v4f16((DC_LDS h4*)(tile + o.hi));
  const auto r = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(Vec<half>::v8, r);
}

template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 acc_frag(const f32x16& a, int half_of) {
  typename Vec<T>::v8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)a[8 * half_of + j];
  return r;
}

template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 load8_or_0(const T* p, bool ok) {
  typename Vec<T>::v8 v = {};
  if (ok) v = *reinterpret_cast<const typename Vec<T>::v8*>(p);
  return v;
}

// ROWS x DP elements by 256 threads, through registers: load() issues the global reads of a tile (rows from `last` on and
// columns from d on read a valid place instead, so that no load waits behind a branch), store() writes them to LDS with zeros
// for those and for the rows that `keep` leaves out: nothing that lies in a masked place is ever multiplied.
template <typename T, int DP, int ROWS>
struct Stage {
  static constexpr int CH = DP / 8, N = ROWS * CH / 256, STEP = 256 / CH;
  uint4 reg[N];
  __device__ __forceinline__ void load(const T* base, int ld, int d, int last) {
    const int r = threadIdx.x / CH, c = threadIdx.x % CH;
#pragma unroll
    for (int i = 0; i < N; ++i)
      reg[i] = *reinterpret_cast<const uint4*>(base + (long)min(r + STEP * i, last) * ld + (c * 8 < d ? c * 8 : 0));
  }
  __device__ __forceinline__ void store(T* tile) const {
    const int r = threadIdx.x / CH, c = threadIdx.x % CH;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<uint4*>(tile + tile_at<DP>(r + STEP * i, c)) = reg[i];
  }
  template <typename F>
  __device__ __forceinline__ void store_some(T* tile, int d, int last, F&& keep) {
    const int r = threadIdx.x / CH, c = threadIdx.x % CH;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c * 8 >= d || r + STEP * i > last || !keep(r + STEP * i)) reg[i] = make_uint4(0, 0, 0, 0);
    store(tile);
  }
};

__device__ __forceinline__ int length_of(const Call& p, int b) {
  return p.kv_len ? min(max(p.kv_len[b], 0), p.tk) : p.tk;
}
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
}
// the sum / maximum of a value over lanes l and l ^ 32, which hold the two halves of a query's scores
__device__ __forceinline__ float pair_sum(float x) { return x + __shfl_xor(x, 32, 64); }
__device__ __forceinline__ float pair_max(float x) { return fmaxf(x, __shfl_xor(x, 32, 64)); }

// Blocks are dealt to the eight XCDs in turn; this gives each a contiguous run of work, so the blocks that read the same keys
// share an L2.  Returns n where a block has nothing to do.
__device__ __forceinline__ int xcd_work(int n) {
  const int per = (n + 7) / 8;
  const int i = blockIdx.x / 8, w = (blockIdx.x % 8) * per + i;
  return i < per && w < n ? w : n;
}
inline unsigned xcd_grid(long n) { return (unsigned)((n + 7) / 8 * 8); }

// Host side: what both directions share (attn_mask_fwd.hip).
int make_call(const dc_attn_desc* d, Call& c, bool backward);
long long summary_bytes(const dc_attn_desc* d);
void launch_summaries(const dc_attn_desc* d, Call& c, char* ws, hipStream_t st);

}  // namespace dcm
