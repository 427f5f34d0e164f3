// The boundary between two blocks of a transformer in one pass (gfx950): the norm behind a block, its gate and residual scale, the
// residual sum and the norm before the next block; forward and gradients.
//
//   u = N1(y), r = a x + s g u, h = N2(r);   N(v) = (v - mean) rstd w + b, or v rstd w + b with rstd = 1 / rms, or v
//   gh = dh w2,  R = dr + rstd2 (gh - mean(gh) - n2 mean(gh n2)),  dx = a R,  du = s R,  dg = sum du u,  gy = du g w1,
//   dy = rstd1 (gy - mean(gy) - n1 mean(gy n1)),  dw1 = sum du g n1, db1 = sum du g, dw2 = sum dh n2, db2 = sum dh
//
// Bound by HBM: forward reads x and y and writes r and h; backward reads x, y, dr and dh (r is computed again, which costs what
// reading it would and keeps the 32-bit value that h came from) and writes dx and dy.  A row belongs to WPR waves, 8 columns to a
// lane, held in registers in fp32 from the load to the store; the weights are loaded once for all rows of a block.  Column sums are
// kept in registers over a block's rows, left as one row of partial sums a block, and added by a second kernel in block order.
#include "common.h"
#include "../../include/dcamd.h"
#include <type_traits>

namespace {

typedef _Float16 half;
template <typename T> struct alignas(16) Row8 { T v[8]; };

enum { NONE = 0, LAYER = 1, RMS = 2 };

struct Desc {
  dc_resnorm_desc d;
  long per_gate;      // rows to a gate row (0: no gate)
  int chunks;         // backward: blocks to a gate row, or 0: `gates` gate rows to a block
  int gates;
  long chunk;         // rows of a chunk
  int blocks;
  float *part, *gpart;   // [blocks][4][c] of dw1, db1, dw2, db2; [blocks][c] of dgate where chunks > 1
};

// Rows are read at a place that is valid in every lane (`at` of lanes behind the row's end is 0), so that no load waits behind a
// branch, and become zeros there when they are widened.
template <typename T>
__device__ __forceinline__ Row8<T> raw8(const void* p, long row, int ld, int at) {
  return *reinterpret_cast<const Row8<T>*>((const T*)p + row * ld + at);
}
template <typename T>
__device__ __forceinline__ void widen(const Row8<T>& v, bool ok, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = ok ? (float)v.v[i] : 0.0f;
}
template <typename T>
__device__ __forceinline__ void put8(T* p, bool ok, const float* f) {
  Row8<T> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v.v[i] = (T)f[i];
  if (ok) *reinterpret_cast<Row8<T>*>(p) = v;
}
// a lane's eight weights (`from`: a place that is valid in every lane)
__device__ __forceinline__ void get_w(const float* w, int from, float none, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = none;
  if (w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = w[from + i];
  }
}
__device__ __forceinline__ float sum8(const float* f) {
  return ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
}

// Sum over a wave, in every lane, by cross-lane moves (wave_sum's shuffles pass through LDS: six round trips a
// sum).
__device__ __forceinline__ float lanes_sum(float v) {
  auto moved = [](float x, auto ctrl) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v += moved(v, std::integral_constant<int, 0xb1>{});    // lane ^ 1
  v += moved(v, std::integral_constant<int, 0x4e>{});    // lane ^ 2
  v += moved(v, std::integral_constant<int, 0x141>{});   // the other four of eight
  v += moved(v, std::integral_constant<int, 0x140>{});   // the other eight of sixteen
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sum over the waves of a row; `red` has a slot of WPR floats for each of two calls in turn, so that one barrier a call is enough.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[16], int& turn) {
  v = lanes_sum(v);
  if constexpr (WPR == 1) return v;
  else {
    if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) t += red[turn][i];
    turn ^= 1;
    return t;
  }
}

// mean and 1 / deviation of a row's columns; columns behind the row's end are zero and stay out of the deviations
template <int WPR>
__device__ __forceinline__ void stats_of(const float* v, bool in, int kind, float inv_c, float eps, float (*red)[16], int& turn,
                                         float& mean, float& rstd) {
  mean = kind == LAYER ? row_sum<WPR>(sum8(v), red, turn) * inv_c : 0.0f;
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = in ? (v[i] - mean) * (v[i] - mean) : 0.0f;
  rstd = rsqrtf(row_sum<WPR>(sum8(q), red, turn) * inv_c + eps);
}

template <typename T, int WPR>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void fwd_kernel(Desc p) {
  constexpr int RP = WPR == 1 ? 4 : 1;   // rows at a time
  __shared__ float red[2][16];
  const dc_resnorm_desc& d = p.d;
  const int slot = WPR == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, at = (WPR == 1 ? threadIdx.x & 63 : threadIdx.x) * 8;
  const bool in = at < d.c;
  const int from = in ? at : 0;
  const float inv_c = 1.0f / d.c;
  float w1[8], b1[8], w2[8], b2[8], g[8];
  get_w(d.w1, from, 1.0f, w1);
  get_w(d.b1, from, 0.0f, b1);
  get_w(d.w2, from, 1.0f, w2);
  get_w(d.b2, from, 0.0f, b2);
  int turn = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = 1.0f;
  long have = -1;
  long row = (long)blockIdx.x * RP + slot;
  if (row >= d.rows) return;   // (a row's waves together)
  Row8<T> xr = raw8<T>(d.x, row, d.ldx, from), yr = raw8<T>(d.y, row, d.ldy, from);
  for (; row < d.rows; row += (long)gridDim.x * RP) {
    float x[8], y[8];
    widen(xr, in, x);
    widen(yr, in, y);
    const long next = min(row + (long)gridDim.x * RP, d.rows - 1);   // on its way while this row is computed
    xr = raw8<T>(d.x, next, d.ldx, from);
    yr = raw8<T>(d.y, next, d.ldy, from);
    if (p.per_gate && row / p.per_gate != have) {
      have = row / p.per_gate;
      widen(raw8<T>(d.gate, have, d.ldg, from), in, g);
    }
    float m1 = 0.0f, k1 = 1.0f, m2 = 0.0f, k2 = 1.0f;
    if (d.first != NONE) stats_of<WPR>(y, in, d.first, inv_c, d.eps, red, turn, m1, k1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = d.first != NONE ? (y[i] - m1) * k1 * w1[i] + b1[i] : y[i];
      x[i] = in ? d.a * x[i] + d.s * (g[i] * u) : 0.0f;
    }
    put8((T*)d.r + row * d.ldr + at, in, x);
    if (d.second != NONE) {
      stats_of<WPR>(x, in, d.second, inv_c, d.eps, red, turn, m2, k2);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (x[i] - m2) * k2 * w2[i] + b2[i];
      put8((T*)d.h + row * d.ldh + at, in, x);
    }
    if (at == 0) *reinterpret_cast<float4*>(d.stats + row * 4) = make_float4(m1, k1, m2, k2);
  }
}

// A block's column sums, those of its slots added in order.
template <int RP, typename O>
__device__ __forceinline__ void leave(const float* f, int at, int slot, bool in, float* cols, O* out) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = f[i];
  if constexpr (RP > 1) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) cols[slot * 512 + at + i] = f[i];
    __syncthreads();
    if (slot > 0) return;
    for (int k = 1; k < RP; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += cols[k * 512 + at + i];
  }
  put8(out + at, in, v);
}

// OFFS: there is an offset b1, or a gradient of an offset is wanted (24 registers of sums that a call without them does not carry).
template <typename T, int WPR, bool OFFS>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR, WPR == 16 ? 4 : WPR == 8 ? 2 : 3) void bwd_kernel(Desc p) {
  constexpr int RP = WPR == 1 ? 4 : 1;
  __shared__ float red[2][16];
  __shared__ float cols[RP == 1 ? 1 : RP * 512];
  const dc_resnorm_desc& d = p.d;
  const int slot = WPR == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, at = (WPR == 1 ? threadIdx.x & 63 : threadIdx.x) * 8;
  const bool in = at < d.c;
  const int from = in ? at : 0;
  const float inv_c = 1.0f / d.c;
  // the 16 waves of the widest rows have 128 registers each: their weights wait in LDS, each lane's own
  constexpr bool LDS_W = WPR == 16;
  __shared__ __attribute__((aligned(16))) float lds_w[LDS_W ? 3 * 8192 : 1];
  float w1[8], b1[8], w2[8], g[8];
  get_w(d.w1, from, 1.0f, w1);
  get_w(OFFS ? d.b1 : nullptr, from, 0.0f, b1);
  get_w(d.w2, from, 1.0f, w2);
  if constexpr (LDS_W)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lds_w[at + i] = w1[i];
      lds_w[8192 + at + i] = w2[i];
      if (OFFS) lds_w[16384 + at + i] = b1[i];
    }
  auto w1_of = [&](int i) __attribute__((always_inline)) { return LDS_W ? lds_w[at + i] : w1[i]; };
  auto w2_of = [&](int i) __attribute__((always_inline)) { return LDS_W ? lds_w[8192 + at + i] : w2[i]; };
  auto b1_of = [&](int i) __attribute__((always_inline)) { return !OFFS ? 0.0f : LDS_W ? lds_w[16384 + at + i] : b1[i]; };
  int turn = 0;
  float s1[8] = {}, t1[8] = {}, s2[8] = {}, t2[8] = {}, sg[8] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = 1.0f;
  Row8<T> xr, yr, rr = {}, hr = {};
  float4 str;
  auto fetch = [&](long row) __attribute__((always_inline)) {
    xr = raw8<T>(d.x, row, d.ldx, from);
    yr = raw8<T>(d.y, row, d.ldy, from);
    str = *reinterpret_cast<const float4*>(d.stats + row * 4);
    if (d.dr) rr = raw8<T>(d.dr, row, d.lddr, from);
    if (d.second != NONE) hr = raw8<T>(d.dh, row, d.lddh, from);
  };
  // chunks > 0: rows row0 .. of one gate row, dealt to the block's slots; else whole gate rows to a slot
  const long gate0 = p.chunks ? blockIdx.x / p.chunks : (long)blockIdx.x * p.gates + slot;
  const long gate1 = p.chunks ? gate0 + 1 : min((long)(blockIdx.x + 1) * p.gates, p.per_gate ? d.rows / p.per_gate : 1L);
  const long per = p.per_gate ? p.per_gate : d.rows;
  for (long gi = gate0; gi < gate1; gi += p.chunks ? 1 : RP) {
    if (p.per_gate) widen(raw8<T>(d.gate, gi, d.ldg, from), in, g);
    const long row0 = gi * per + (p.chunks ? blockIdx.x % p.chunks * p.chunk + slot : 0);
    const long row1 = min((gi + 1) * per, p.chunks ? gi * per + (blockIdx.x % p.chunks + 1) * p.chunk : d.rows);
    if (row0 < row1) fetch(row0);
    for (long row = row0; row < row1; row += p.chunks ? RP : 1) {
      if constexpr (LDS_W) asm volatile("" ::: "memory");   // read them anew for each row
      // u = n1 w1 + b1 is formed where it is used (a norm that is none: n1 = y, 1 and 0)
      float x[8], n1[8], gr[8];
      const float4 st = str;
      widen(xr, in, x);
      widen(yr, in, n1);
      widen(rr, in && d.dr, gr);
#pragma unroll
      for (int i = 0; i < 8; ++i) n1[i] = in ? (n1[i] - st.x) * st.y : 0.0f;
      if (d.second != NONE) {
        float gh[8];
        widen(hr, in, gh);
        fetch(min(row + (p.chunks ? RP : 1), row1 - 1));   // on its way while this row is computed
        float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = in ? (d.a * x[i] + d.s * (g[i] * (n1[i] * w1_of(i) + b1_of(i))) - st.z) * st.w : 0.0f;   // n2
          s2[i] += gh[i] * x[i];
          if constexpr (OFFS) t2[i] += gh[i];
          gh[i] *= w2_of(i);
          c1 += gh[i];
          c2 += gh[i] * x[i];
        }
        c2 = row_sum<WPR>(c2, red, turn) * inv_c;
        c1 = d.second == LAYER ? row_sum<WPR>(c1, red, turn) * inv_c : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) gr[i] += st.w * (gh[i] - c1 - x[i] * c2);
      } else {
        fetch(min(row + (p.chunks ? RP : 1), row1 - 1));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = d.a * gr[i];
      put8((T*)d.dx + row * d.lddx + at, in, x);
      float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        gr[i] *= d.s;
        sg[i] += gr[i] * (n1[i] * w1_of(i) + b1_of(i));
        gr[i] *= g[i];
        s1[i] += gr[i] * n1[i];
        if constexpr (OFFS) t1[i] += gr[i];
        if (d.first != NONE) {
          gr[i] = in ? gr[i] * w1_of(i) : 0.0f;
          c1 += gr[i];
          c2 += gr[i] * n1[i];
        }
      }
      if (d.first != NONE) {
        c2 = row_sum<WPR>(c2, red, turn) * inv_c;
        c1 = d.first == LAYER ? row_sum<WPR>(c1, red, turn) * inv_c : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) gr[i] = st.y * (gr[i] - c1 - n1[i] * c2);
      }
      put8((T*)d.dy + row * d.lddy + at, in, gr);
    }
    if (!p.chunks && d.dgate) {
      put8((T*)d.dgate + gi * d.lddg + at, in, sg);
#pragma unroll
      for (int i = 0; i < 8; ++i) sg[i] = 0.0f;
    }
  }
  float* part = p.part + (long)blockIdx.x * 4 * d.c;
  if (d.dw1) leave<RP>(s1, at, slot, in, cols, part);
  if (OFFS && d.db1) leave<RP>(t1, at, slot, in, cols, part + d.c);
  if (d.dw2) leave<RP>(s2, at, slot, in, cols, part + 2 * d.c);
  if (OFFS && d.db2) leave<RP>(t2, at, slot, in, cols, part + 3 * d.c);
  if (p.chunks && d.dgate) {
    if (p.chunks == 1) leave<RP>(sg, at, slot, in, cols, (T*)d.dgate + gate0 * d.lddg);
    else leave<RP>(sg, at, slot, in, cols, p.gpart + (long)blockIdx.x * d.c);
  }
}

// 64 columns of one sum to a block: its 16 waves take a run of the partial rows each, and are added in order.
template <typename T>
__global__ __launch_bounds__(1024) void fold_kernel(Desc p) {
  __shared__ float red[16][64];
  const dc_resnorm_desc& d = p.d;
  const int which = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int col = blockIdx.x * 64 + lane;
  float* const out = which == 0 ? d.dw1 : which == 1 ? d.db1 : which == 2 ? d.dw2 : d.db2;
  const float* src = p.part + (long)which * d.c;
  int n = p.blocks;
  long stride = 4L * d.c;
  if (which >= 4) {   // a gate row's chunks
    n = p.chunks;
    stride = d.c;
    src = p.gpart + (long)(which - 4) * n * d.c;
  } else if (!out) {
    return;
  }
  const int each = (n + 15) / 16, i0 = w * each, i1 = min(n, i0 + each);
  float s[8] = {};
  if (col < d.c) {
    src += col;
    int i = i0;
    for (; i + 8 <= i1; i += 8)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] += src[(i + k) * stride];
    for (; i < i1; ++i) s[0] += src[i * stride];
  }
  red[w][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (w > 0 || col >= d.c) return;
  float v = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) v += red[k][lane];
  if (which < 4) out[col] = v;
  else ((T*)d.dgate)[(long)(which - 4) * d.lddg + col] = (T)v;
}

// Backward blocks that leave partial sums: as many as the card holds at once (12 waves to a CU, of the 16-wave blocks one).
int most_blocks(int c) { return c <= 512 ? 768 : c <= 1024 ? 1536 : c <= 2048 ? 768 : 256; }

void plan(const dc_resnorm_desc* d, Desc& p) {
  p.d = *d;
  p.per_gate = d->gates > 0 ? d->rows / d->gates : 0;
  const long gates = d->gates > 0 ? d->gates : 1, per = d->rows / gates;
  const int rp = d->c <= 512 ? 4 : 1;
  const int most = most_blocks(d->c);
  p.gates = 0;
  p.chunks = 0;
  if (gates <= most) {
    p.chunks = (int)max(1L, min(most / gates, (per + rp - 1) / rp));
    p.chunk = (per + p.chunks - 1) / p.chunks;
    p.chunks = (int)((per + p.chunk - 1) / p.chunk);
    p.blocks = (int)(gates * p.chunks);
  } else {
    p.gates = (int)((gates + most - 1) / most);
    p.gates = (p.gates + rp - 1) / rp * rp;
    p.blocks = (int)((gates + p.gates - 1) / p.gates);
  }
}

long part_floats(const Desc& p) {
  const dc_resnorm_desc& d = p.d;
  return d.dw1 || d.db1 || d.dw2 || d.db2 ? 4L * p.blocks * d.c : 0;
}
long long ws_of(const Desc& p) { return 4LL * (part_floats(p) + (p.d.dgate && p.chunks > 1 ? (long)p.blocks * p.d.c : 0)); }

int check(const dc_resnorm_desc* d, bool backward) {
  if (!d || d->type < 0 || d->type > 2 || !d->x || !d->y || !d->stats || d->rows <= 0 || d->c <= 0 || d->c % 8 || d->c > 8192)
    return DC_ERR_ARG;
  if (d->first < 0 || d->first > 2 || d->second < 0 || d->second > 2 || d->rows > (1LL << 40) / d->c) return DC_ERR_ARG;
  if ((d->first == NONE && (d->w1 || d->b1)) || (d->second == NONE && (d->w2 || d->b2))) return DC_ERR_ARG;
  if (d->gates < 0 || (d->gates > 0) != (d->gate != nullptr) || (d->gates > 0 && d->rows % d->gates)) return DC_ERR_ARG;
  if (!(d->eps >= 0.0f)) return DC_ERR_ARG;
  const int c = d->c;
  if (d->ldx < c || d->ldy < c || (d->gate && d->ldg < c)) return DC_ERR_ARG;
  uintptr_t at = (uintptr_t)d->x | (uintptr_t)d->y | (uintptr_t)d->gate | (uintptr_t)d->stats;
  int ld = d->ldx | d->ldy | (d->gate ? d->ldg : 0);
  const uintptr_t words = (uintptr_t)d->w1 | (uintptr_t)d->b1 | (uintptr_t)d->w2 | (uintptr_t)d->b2 | (uintptr_t)d->dw1 |
                          (uintptr_t)d->db1 | (uintptr_t)d->dw2 | (uintptr_t)d->db2;
  if (!backward) {
    if (!d->r || d->ldr < c || (d->second != NONE) != (d->h != nullptr) || (d->h && d->ldh < c)) return DC_ERR_ARG;
    at |= (uintptr_t)d->r | (uintptr_t)d->h;
    ld |= d->ldr | (d->h ? d->ldh : 0);
  } else {
    if (!d->dx || !d->dy || d->lddx < c || d->lddy < c || (!d->dr && !d->dh) || (d->dr && d->lddr < c)) return DC_ERR_ARG;
    if ((d->second != NONE) != (d->dh != nullptr) || (d->dh && d->lddh < c) || (d->dgate && (!d->gate || d->lddg < c)))
      return DC_ERR_ARG;
    if (((d->dw1 || d->db1) && d->first == NONE) || ((d->dw2 || d->db2) && d->second == NONE)) return DC_ERR_ARG;
    at |= (uintptr_t)d->dx | (uintptr_t)d->dy | (uintptr_t)d->dr | (uintptr_t)d->dh | (uintptr_t)d->dgate;
    ld |= d->lddx | d->lddy | (d->dr ? d->lddr : 0) | (d->dh ? d->lddh : 0) | (d->dgate ? d->lddg : 0);
  }
  return (at & 15) || (words & 3) || ld % 8 ? DC_ERR_ALIGN : DC_OK;
}

template <typename T, int W>
void forward(const Desc& p, hipStream_t st) {
  const int rp = W == 1 ? 4 : 1, threads = W == 1 ? 256 : 64 * W;
  const long blocks = min((long)((p.d.rows + rp - 1) / rp), 256L * 2048 / threads);   // what the card holds at once
  hipLaunchKernelGGL((fwd_kernel<T, W>), dim3((unsigned)blocks), dim3(threads), 0, st, p);
}
template <typename T, int W>
void backward(const Desc& p, hipStream_t st) {
  const dim3 grid((unsigned)p.blocks), block(W == 1 ? 256 : 64 * W);
  if (p.d.b1 || p.d.db1 || p.d.db2) hipLaunchKernelGGL((bwd_kernel<T, W, true>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((bwd_kernel<T, W, false>), grid, block, 0, st, p);
}

// 8 columns to a lane: a row takes as many waves as that needs
template <typename T>
void launch(const Desc& p, bool back, hipStream_t st) {
  const int c = p.d.c;
  if (c <= 512) back ? backward<T, 1>(p, st) : forward<T, 1>(p, st);
  else if (c <= 1024) back ? backward<T, 2>(p, st) : forward<T, 2>(p, st);
  else if (c <= 2048) back ? backward<T, 4>(p, st) : forward<T, 4>(p, st);
  else if (c <= 4096) back ? backward<T, 8>(p, st) : forward<T, 8>(p, st);
  else back ? backward<T, 16>(p, st) : forward<T, 16>(p, st);
  const bool gate = p.d.dgate && p.chunks > 1;
  if (back && (part_floats(p) || gate))
    hipLaunchKernelGGL((fold_kernel<T>), dim3((unsigned)((c + 63) / 64), (unsigned)(4 + (gate ? p.d.gates : 0))), dim3(1024), 0,
                       st, p);
}
void launch(const Desc& p, bool back, hipStream_t st) {
  if (p.d.type == 0) launch<bf16>(p, back, st);
  else if (p.d.type == 1) launch<half>(p, back, st);
  else launch<float>(p, back, st);
}

}  // namespace

extern "C" int dc_resnorm_fwd(const dc_resnorm_desc* d, void* stream) {
  if (const int rc = check(d, false)) return rc;
  Desc p{};
  plan(d, p);
  hipStream_t st = (hipStream_t)stream;
  launch(p, false, st);
  DC_CHECK_LAUNCH();
  return DC_OK;
}

extern "C" long long dc_resnorm_ws_bytes(const dc_resnorm_desc* d) {
  if (!d || d->rows <= 0 || d->c <= 0 || d->rows > (1LL << 40) / d->c || (d->gates > 0 && d->rows < d->gates)) return 0;
  Desc p{};
  plan(d, p);
  return ws_of(p);
}

extern "C" int dc_resnorm_bwd(const dc_resnorm_desc* d, void* ws, long long ws_bytes, void* stream) {
  if (const int rc = check(d, true)) return rc;
  Desc p{};
  plan(d, p);
  if (ws_of(p) > (ws ? ws_bytes : 0)) return DC_ERR_ARG;
  if ((uintptr_t)ws & 15) return DC_ERR_ALIGN;
  p.part = static_cast<float*>(ws);
  p.gpart = p.part + part_floats(p);
  hipStream_t st = (hipStream_t)stream;
  launch(p, true, st);
  DC_CHECK_LAUNCH();
  return DC_OK;
}
