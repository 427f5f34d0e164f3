// Masked attention backward (gfx950): the gradients of q, k and v from the inputs, the output, its log-sum and its gradient.
//
//   P = exp(s - lse), dP = dO V^T, dS = P (dP - rowsum(dO o)) (1 - tanh^2), dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO
//
// Two kernels, each holding one side in registers and sweeping the other through LDS, so every sum has one owner and a fixed
// order: dq_kernel (128 query rows of a head; it also leaves the row constants), then dkv_kernel (128 keys of a key head, over all
// query heads of its group).  Both compute S and dP again: 7 products for 5, for no exchange of dQ between blocks.
//
// fp16: dS is scaled by a power of two before it is rounded, by the row's (dQ) or the key head's (dK) largest |dO| so that this
// lies in [2^-4, 2^-3): gradients far below 1 keep their digits.  P in dV is held 2^14 times as large for the same reason.  Both
// factors are taken out of the fp32 sums again.  With values in the thousands dS could leave the type so.  dK, whose keys are there,
// takes a smaller factor where |dP| <= d max |dO| max |v| or |rowsum(dO o)| asks for it; dQ, which meets its keys as it goes, looks
// at its sums at the end (inf times anything left none of a row finite) and sweeps once more with 2^-6 of these rows' factors, which
// holds for every finite v: |dP - rowsum| to 2 x 128 x 2^-9 x 65504 = 32752.
#include "attn_mask.h"
#include <type_traits>

namespace dcm {
namespace {

struct Back {
  float *nlse, *ndel;   // [nb heads][32 n32]: -lse log2 e (-inf: the row sees no key, or lies behind the last), -rowsum(dO o)
  int2* rows32;         // [nb heads][n32]: of 32 rows, whether one sees no key, and the largest |dO|, or kRoom |rowsum(dO o)| (its bits)
  int n32;
  int nq, nk;           // splits of dq_kernel's sweep over the keys, of dkv_kernel's over the queries
  float *part_q, *part; // [nq][nb tq][heads][DP]; [nk][2][nb tk][kvh][DP]
};

template <typename T> constexpr bool is_half = __is_same(T, half);
constexpr float kLess = 0.015625f;   // 2^-6, for dS that left the type's range
constexpr float kRoom = 7.62939453125e-06f;   // 2^-17: what is kept below 2^-3 when it is multiplied by this stays below 2^14 itself
__device__ __forceinline__ bool left_range(float sum) { return !(fabsf(sum) < INFINITY); }

// what dS as the kernels hold it lacks (cap_score gives a quarter of the slope)
__device__ __forceinline__ float ds_scale(const Call& p) { return p.cap2 != 0.0f ? 4.0f * p.scale : p.scale; }

template <typename T>
__device__ __forceinline__ void put4(T* out, f32x4 a) {
  typename Vec<T>::v4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (T)a[e];
  *reinterpret_cast<typename Vec<T>::v4*>(out) = v;
}

// power of two that brings a positive finite x into [2^-4, 2^-3)
__device__ __forceinline__ float near_sixteenth(float x) {
  if (!(x > 0.0f && x < INFINITY)) return 1.0f;
  const int e = (int)(__float_as_uint(x) >> 23) - 127;
  return ldexpf(1.0f, min(max(-4 - e, -100), 100));
}

// rowsum(dO o) from the rounded o is off by a rounding of o, the same for all keys of the row.  Rows of few keys, whose gradients
// are small differences, take it from a sweep of its own over P dP: of 750 gradients of random calls of 8 to 6000 keys the furthest
// (12 keys) was off by 0.46 % of its norm without and 0.36 % with (2009 keys), 264 and 49 of them by more than one rounding and a half.
// A block does so where all its rows together meet at most kExact tiles (4 x 108 x 20 heads, forward and gradients: 34 us, 31 without), whatever
// the length of the call that they are part of and the parts that they are split in.  SHORT: no block of the call meets more, and
// none reads o (which costs 8 x 1024 x 16 heads, causal, 9 us of 165).
constexpr int kExact = 16;
template <typename T, int DP, int FORM, bool SHORT>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void dq_kernel(Call p, Back bk) {
  typedef typename Vec<T>::v8 v8;
  constexpr int S = DP == 64 ? 3 : 2, TILE = 64 * DP, OPS = 2 * Dma<T, DP>::N;
  typedef KeyRing<T, DP, S> Ring;
  __shared__ typename Ring::Lds lds;
  __shared__ int range[6];
  const int lane = threadIdx.x & 63, hh = lane >> 5;
  QueryBlock q;
  q.init(p, bk.nq);
  if (q.idle) return;
  const long row = ((long)q.b * p.heads + q.h) * p.tq + (q.live ? q.qi : 0), trow = (long)q.b * p.tq + (q.live ? q.qi : 0);
  const float lse = p.lse[row];
  const bool sees = q.live && lse != -INFINITY;
  v8 qf[DP / 16], df[DP / 16], of[DP / 16];
  float del = 0.0f, most = 0.0f;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int c = 16 * s + 8 * hh;
    const bool ok = sees && c < p.d;
    qf[s] = load8_or_0((const T*)p.q + trow * p.ldq + q.h * p.d + c, ok);
    df[s] = load8_or_0((const T*)p.dout + trow * p.lddo + q.h * p.d + c, ok);
    of[s] = load8_or_0((const T*)p.o + trow * p.ldo + q.h * p.d + c, ok);
  }
#pragma unroll
  for (int s = 0; s < DP / 16; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      del = fmaf((float)df[s][j], (float)of[s][j], del);
      most = fmaxf(most, fabsf((float)df[s][j]));
    }
  del = pair_sum(del);
  most = pair_max(most);
  const float nl = sees ? -lse * kLog2e : -INFINITY;
  float f = is_half<T> ? near_sixteenth(most) : 1.0f;
  int t0, t1;
  int holes;
  q.tiles(p, sees, range, t0, t1, holes);
  const int each = (t1 - t0 + q.parts - 1) / q.parts, part0 = min(t1, t0 + q.part * each), part1 = min(t1, part0 + each);

  if (is_half<T> && threadIdx.x == 0) range[0] = 0;   // whether the sums have been swept again
  Ring ring;
  ring.init(p, q, holes);
  f32x16 dq[DP / 32];
#pragma unroll
  for (int n = 0; n < DP / 32; ++n) dq[n] = f32x16{};
  const float slope = FORM != PLAIN && p.slopes ? p.slopes[q.h] * p.bend : 0.0f;
  int koff[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) koff[s] = tile_at<DP>(lane & 31, 2 * s + hh);
  TrAt ka[2];
  TrAt4 ka4;
  if constexpr (DP == 128) ka4.init(lds.tiles[0], lane);
  else
#pragma unroll
    for (int n = 0; n < 2; ++n) ka[n] = tr_at<DP>(32 * n, lane);
  WaveRange range_of;
  range_of.init(q, sees);
  // FIRST: the sum of P dP goes to `exact`; else dS K to dq
  float exact = 0.0f;
  auto tile = [&](int t, auto B, const int* id, bool masked, auto F) __attribute__((always_inline)) {
    constexpr int buf = decltype(B)::value;
    constexpr bool FIRST = decltype(F)::value;
    const T* kt = lds.tiles[buf];
    const T* vt = kt + TILE;
    auto half_tile = [&](auto K) __attribute__((always_inline)) {
      constexpr int kb2 = decltype(K)::value;
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        s = mfma(*reinterpret_cast<const v8*>(kt + 32 * kb2 * DP + koff[c]), qf[c], s);
        dp = mfma(*reinterpret_cast<const v8*>(vt + 32 * kb2 * DP + koff[c]), df[c], dp);
      }
      if constexpr (!FIRST)
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] -= del;
      if constexpr (FORM != PLAIN) {
        if (p.cap2 != 0.0f) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float g;
            s[r] = cap_score<FORM>(p, s[r], &g);
            if constexpr (!FIRST) dp[r] *= g;
          }
        }
        if (p.slopes) {
          const float dist = (float)(q.pos - t * 64 - 4 * hh);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[r] = fmaf(-slope, fabsf(dist - (float)(32 * kb2 + (r & 3) + 8 * (r >> 2))), s[r]);
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float pw = exp2_raw(fmaf(s[r], p.mul, nl));
        s[r] = (is_half<T> && !FIRST ? pw * f : pw) * dp[r];
      }
      if (masked) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int key = 32 * kb2 + 8 * g + 4 * hh;
          int4 i4 = make_int4(0, 0, 0, 0);
          if (id) i4 = *reinterpret_cast<const int4*>(&id[key]);
          const int id4[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t * 64 + key + e >= q.lim || (id && id4[e] != q.mine)) s[4 * g + e] = 0.0f;
        }
      }
      if constexpr (FIRST) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r & 3] += s[r];
        exact += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        return;
      }
      auto add = [&](auto C) __attribute__((always_inline)) {
        constexpr int c = decltype(C)::value, at = (32 * kb2 + 16 * c) * DP;
        v8 f2[DP / 32];
        if constexpr (DP == 128) tr_frags<T, (buf * 2 * TILE + at) * 2>(ka4, f2);
        else
#pragma unroll
          for (int n = 0; n < 2; ++n) f2[n] = tr_frag(kt + at, ka[n]);
        const v8 sf = acc_frag<T>(s, c);
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) dq[n] = mfma(f2[n], sf, dq[n]);
      };
      add(std::integral_constant<int, 0>{});
      add(std::integral_constant<int, 1>{});
    };
    half_tile(std::integral_constant<int, 0>{});
    __builtin_amdgcn_sched_barrier(0);   // (halves that overlap need 20 registers more, which spill: 8 x 4096 x 16 heads 2007 us for 2076)
    half_tile(std::integral_constant<int, 1>{});
  };
  auto step = [&](int t, auto B, auto F) __attribute__((always_inline)) {   // as the forward's
    constexpr int buf = decltype(B)::value;
    if (S == 3 && t + 1 < t1) vm_wait<OPS>();
    else vm_wait<0>();
    tile_barrier();
    if (S == 2 && t + 1 < t1) ring.load(p, lds, t + 1, buf ^ 1);
    const int* id = ring.kid ? lds.ids[buf] : nullptr;
    const int look = range_of.look(t, id);
    if (look != WaveRange::NOTHING) tile(t, B, id, look == WaveRange::MASKED, F);
    if (S == 3 && t + 2 < t1) ring.load(p, lds, t + 2, (buf + 2) % 3);
  };
  auto sweep = [&](auto F) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(F)::value;
    for (;;) {
      int t = t0;
      if constexpr (is_half<T> && !FIRST) asm volatile("" : "+s"(t));   // (what the loads start from is not kept for a second time)
      if (t < t1) ring.load(p, lds, t, 0);
      if (S == 3 && t + 1 < t1) ring.load(p, lds, t + 1, 1);
      for (; t < t1; t += S) {
        step(t, std::integral_constant<int, 0>{}, F);
        if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{}, F);
        if constexpr (S == 3)
          if (t + 2 < t1) step(t + 2, std::integral_constant<int, 2>{}, F);
      }
      if constexpr (!is_half<T> || FIRST) break;
      tile_barrier();
      const bool twice = range[0], over = left_range(dq[0][0]);
      tile_barrier();
      if (over) range[0] = 1;
      tile_barrier();
      if (twice || !range[0]) break;
      if (over) f *= kLess;
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) dq[n] = f32x16{};
    }
  };
  if (SHORT || t1 - t0 <= kExact) {
    sweep(std::true_type{});
    del = pair_sum(exact);
    tile_barrier();
  }
  t0 = part0;
  t1 = part1;
  const float wave_most = is_half<T> ? wave_max(fmaxf(most, kRoom * fabsf(del))) : 0.0f;
  const bool blind = __any(q.live && !sees);
  if (lane == 0 && q.part == 0) bk.rows32[((long)q.b * p.heads + q.h) * bk.n32 + q.qi / 32] = make_int2(blind, __float_as_int(wave_most));
  // (rows behind the last too: what dkv_kernel reads there has to weigh nothing, whatever its scores become)
  if (hh == 0 && q.part == 0) {
    const long at = ((long)q.b * p.heads + q.h) * 32 * bk.n32 + q.qi;
    bk.nlse[at] = nl;
    bk.ndel[at] = -del;
  }
  sweep(std::false_type{});
  if (!q.live) return;
  const float k = ds_scale(p) / f;
  T* out = (T*)p.dq + ((long)q.b * p.tq + q.qi) * p.lddq + q.h * p.d;
  float* pq = q.parts > 1 ? bk.part_q + ((((long)q.part * p.nb + q.b) * p.tq + q.qi) * p.heads + q.h) * DP : nullptr;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * n + 8 * g + 4 * hh;
      if (col >= p.d) continue;
      f32x4 a;
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = sees ? dq[n][4 * g + e] * k : 0.0f;
      if (pq) *reinterpret_cast<f32x4*>(pq + col) = a;
      else put4(out + col, a);
    }
}

// what the factor of dS in dK goes by for a key head: the largest of its query heads' rows32, the same in every block that asks
__device__ __forceinline__ float head_most(const Call& p, const Back& bk, int b, int kh, float* scratch) {
  const int2* r = bk.rows32 + ((long)b * p.heads + kh * p.grp) * bk.n32;
  float most = 0.0f;
  for (int i = threadIdx.x; i < p.grp * bk.n32; i += blockDim.x) most = fmaxf(most, __int_as_float(r[i].y));
  most = wave_max(most);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = most;
  __syncthreads();
  for (int i = 0; i < (int)blockDim.x / 64; ++i) most = fmaxf(most, scratch[i]);
  return most;
}

constexpr float kPShift = 14.0f;   // fp16: P in dV is 2^14 times as large

// 128 keys to a block, held in registers; tiles of 64 query rows pass through LDS, three of them in turn.
// 64 columns: a wave has 32 keys with both of their sums.  128 columns: a pair of waves has 32 keys.  Of a tile each takes 32 rows to
// P and dS; the first then sums dV and needs P of all rows, the second dK and dS of all: they exchange the half that the other sums
// (2 KB each way), and a wave carries one sum, not two, which is what lets two waves share a SIMD (one wave with both took 416
// registers and 24 % of the matrix units' time: 4097 x 32/8 heads causal 511 us for 398; at 64 columns, where both fit, pairs lose:
// 8 x 4096 x 16 heads with dQ 2020 us for 2824).
template <typename T, int DP, int FORM>
__global__ __launch_bounds__(DP == 64 ? 256 : 512, 2) void dkv_kernel(Call p, Back bk) {
  typedef typename Vec<T>::v8 v8;
  constexpr bool PAIR = DP == 128;
  constexpr int NT = PAIR ? 512 : 256;
  typedef Dma<T, DP, NT> D;
  constexpr int TILE = 64 * DP, OPS = 2 * D::N;
  __shared__ __attribute__((aligned(16))) T tiles[3][2 * TILE];   // Q, dO
  __shared__ __attribute__((aligned(16))) float cn[3][64], cd[3][64];
  __shared__ __attribute__((aligned(16))) int ids[3][64];
  __shared__ __attribute__((aligned(16))) T swap[PAIR ? 8 : 1][2][64 * 8];
  __shared__ int range[4], blind_rows;
  __shared__ float scratch[8];
  const int lane = threadIdx.x & 63, hh = lane >> 5, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), second = PAIR ? wid & 1 : 0;
  // (the first keys of a causal call have the longest columns; 128 columns have one block to a CU, and what comes later fills the gaps)
  const int nkb = (p.tk + 127) / 128;
  const Place place = p.list_k ? place_of(p.kvh, p.entries_k, 1, true, !PAIR)
                               : place_of(p.nb * p.kvh, nkb, bk.nk, gridDim.x <= kSpread, !PAIR);
  const int2 e = p.list_k ? entry_of(p.list_k, place.item) : make_int2(place.item, place.part | bk.nk << 8);
  if (e.x < 0) return;
  const int b = p.list_k ? e.x / nkb : place.unit / p.kvh, kh = place.unit % p.kvh;
  const int part = e.y & 255, parts = e.y >> 8, k0 = (p.list_k ? e.x % nkb : e.x) * 128;
  const int len = length_of(p, b), pre = p.prefix ? p.prefix[b] : 0, shift = len - p.tq;
  const int key = k0 + (PAIR ? wid >> 1 : wid) * 32 + (lane & 31);
  const int mine = p.doc_q ? (key < len ? p.doc_k[(long)b * p.tk + key] : -1) : 0;
  const bool ok = key < len && mine >= 0;
  v8 kf[DP / 16], vf[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int c = 16 * s + 8 * hh;
    kf[s] = load8_or_0((const T*)p.k + ((long)b * p.tk + key) * p.ldk + kh * p.d + c, ok && c < p.d);
    vf[s] = load8_or_0((const T*)p.v + ((long)b * p.tk + key) * p.ldv + kh * p.d + c, ok && c < p.d);
  }
  float f = 1.0f;   // of the lane's key
  if constexpr (is_half<T>) {
    float v = 0.0f;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) v = fmaxf(v, fabsf((float)vf[s][j]));
    f = near_sixteenth(head_most(p, bk, b, kh, scratch) * fmaxf(1.0f, kRoom * DP * pair_max(v)));
  }
  // the lane's key is seen from position `from` on
  const int from = !ok ? 0x7fffffff : p.causal && key >= pre ? key : -0x7fffffff;
  const int from_last = __builtin_amdgcn_readfirstlane(wave_max_i(from)), from_first = __builtin_amdgcn_readfirstlane(wave_min_i(from));
  const int id_least = __builtin_amdgcn_readfirstlane(wave_min_i(mine >= 0 ? mine : 0x7fffffff));
  const int id_most = __builtin_amdgcn_readfirstlane(wave_max_i(mine));
  int t0 = 0, t1 = (p.tq + 63) / 64;
  if (p.causal && k0 >= pre) t0 = max(0, k0 - shift) / 64;
  if (k0 >= len) t1 = 0;
  if (p.sum_q) {
    const int nt = (p.tq + 63) / 64;
    if (threadIdx.x == 0) { range[0] = 0x7fffffff; range[1] = 0; range[2] = 0x7fffffff; range[3] = -1; }
    __syncthreads();
    if (ok) { atomicMin(&range[2], mine); atomicMax(&range[3], mine); }
    __syncthreads();
    const int least = range[2], largest = range[3];
    int first = 0x7fffffff, last = -1;
    for (int t = t0 + threadIdx.x; t < t1; t += NT) {
      const int4 s = p.sum_q[(long)b * nt + t];
      if (s.y >= least && s.x <= largest) { first = min(first, t); last = t; }
    }
    if (last >= 0) { atomicMin(&range[0], first); atomicMax(&range[1], last + 1); }
    __syncthreads();
    t0 = __builtin_amdgcn_readfirstlane(range[0]);
    t1 = __builtin_amdgcn_readfirstlane(range[1]);
  }
  const int nt = max(0, t1 - t0), steps = nt * p.grp;
  // the first tile with a row that sees no key (asked for each tile, the answer would be waited for in each)
  if (threadIdx.x == 0) blind_rows = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < steps; i += NT) {
    const int2* fl = bk.rows32 + ((long)b * p.heads + kh * p.grp + i / nt) * bk.n32 + (t0 + i % nt) * 2;
    if (fl[0].x | fl[1].x) atomicMin(&blind_rows, t0 + i % nt);
  }
  __syncthreads();
  const int blind = __builtin_amdgcn_readfirstlane(blind_rows);
  const int each = (steps + parts - 1) / parts, i0 = min(steps, part * each), i1 = min(steps, i0 + each);

  D qs, ds;
  qs.init(p.ldq, p.d);
  ds.init(p.lddo, p.d);
  int hg_next = nt ? i0 / nt : 0, t_next = nt ? t0 + i0 % nt : 0;
  auto load = [&](int buf) __attribute__((always_inline)) {   // the next (query head, tile) of the sweep
    const int h = kh * p.grp + hg_next, r0 = t_next * 64, last = p.tq - 1 - r0;
    const long trow = (long)b * p.tq + r0, head = (long)b * p.heads + h, at = head * 32 * bk.n32 + r0;
    const T *qa = (const T*)p.q + trow * p.ldq + h * p.d, *da = (const T*)p.dout + trow * p.lddo + h * p.d;
    const int2* fl = bk.rows32 + head * bk.n32 + r0 / 32;
    if (t_next >= blind && (fl[0].x | fl[1].x)) {   // a row that sees no key: it may hold anything
      auto keep = [&](int r) __attribute__((always_inline)) { return bk.nlse[at + min(r, last)] != -INFINITY; };
      qs.load_some(qa, tiles[buf], last, keep);
      ds.load_some(da, tiles[buf] + TILE, last, keep);
    } else {
      qs.load(qa, tiles[buf], last);
      ds.load(da, tiles[buf] + TILE, last);
    }
    if (wid == 0) {
      dma_words(bk.nlse + at, cn[buf], 63);
      dma_words(bk.ndel + at, cd[buf], 63);
      if (p.doc_q) dma_words(p.doc_q + trow, ids[buf], last);
    }
    if (++t_next == t1) { t_next = t0; ++hg_next; }
  };
  f32x16 dv[DP / 32], dk[PAIR ? 1 : DP / 32];   // (a pair has dv alone: dV in the first wave, dK in the second)
#pragma unroll
  for (int n = 0; n < DP / 32; ++n) {
    dv[n] = f32x16{};
    if constexpr (!PAIR) dk[n] = f32x16{};
  }
  int qoff[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) qoff[s] = tile_at<DP>(lane & 31, 2 * s + hh) + 32 * second * DP;
  TrAt ta[DP / 32];   // (of a pair: dO^T for the first wave, Q^T for the second)
#pragma unroll
  for (int n = 0; n < DP / 32; ++n) {
    ta[n] = tr_at<DP>(32 * n, lane);
    if (PAIR && !second) { ta[n].lo += TILE; ta[n].hi += TILE; }
  }
  if (i0 < i1) load(0);
  if (i0 + 1 < i1) load(1);
  int hg = nt ? i0 / nt : 0, t = nt ? t0 + i0 % nt : 0;
  auto step = [&](int i, auto B) __attribute__((always_inline)) {
    constexpr int buf = decltype(B)::value;
    if (i + 1 < i1) vm_wait<OPS>();
    else vm_wait<0>();
    tile_barrier();
    const T* qt = tiles[buf];
    const T* dt = qt + TILE;
    const int id = p.doc_q ? ids[buf][lane] : 0;
    // none of the wave's keys is seen from the tile
    const bool nothing = from_first > t * 64 + shift + 63 || (p.doc_q && !__any(id >= id_least && id <= id_most));
    const bool mixed = p.doc_q && (id_least != id_most || __any(id != id_least));
    // P and dS of 32 rows of the tile (a pair's: qoff is at the wave's own)
    auto weights = [&](int at, v8 (&pf)[2], v8 (&sf)[2]) __attribute__((always_inline)) {
      const int rows = at + 32 * second, row0 = rows + 4 * hh, pos0 = t * 64 + shift + row0;   // of the lane's first row
      f32x16 s = {}, dp;
      f32x4 nl[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        nl[g] = *reinterpret_cast<const f32x4*>(&cn[buf][row0 + 8 * g]);
        const f32x4 nd = *reinterpret_cast<const f32x4*>(&cd[buf][row0 + 8 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * g + e] = nd[e];
      }
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        s = mfma(*reinterpret_cast<const v8*>(qt + at * DP + qoff[c]), kf[c], s);
        dp = mfma(*reinterpret_cast<const v8*>(dt + at * DP + qoff[c]), vf[c], dp);
      }
      if constexpr (FORM != PLAIN) {
        if (p.cap2 != 0.0f) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float g;
            s[r] = cap_score<FORM>(p, s[r], &g);
            dp[r] *= g;
          }
        }
        if (p.slopes) {
          const float slope = p.slopes[kh * p.grp + hg] * p.bend, dist = (float)(pos0 - key);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(-slope, fabsf(dist + (float)((r & 3) + 8 * (r >> 2))), s[r]);
        }
      }
      const float fs = is_half<T> ? f * 6.103515625e-05f : 1.0f;   // 2^-14
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float up = is_half<T> ? kPShift : 0.0f;
        s[r] = exp2_raw(fmaf(s[r], p.mul, nl[r >> 2][r & 3] + up));
        dp[r] *= is_half<T> ? s[r] * fs : s[r];
      }
      if (mixed || from_last > t * 64 + shift + rows) {
        asm volatile("" ::: "memory");   // a branch, not selects in every tile
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          int4 i4 = make_int4(0, 0, 0, 0);
          if (p.doc_q) i4 = *reinterpret_cast<const int4*>(&ids[buf][row0 + 8 * g]);
          const int id4[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (pos0 + 8 * g + e < from || (p.doc_q && id4[e] != mine)) {
              s[4 * g + e] = 0.0f;
              dp[4 * g + e] = 0.0f;
            }
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        pf[c] = acc_frag<T>(s, c);
        sf[c] = acc_frag<T>(dp, c);
      }
    };
    v8 pf[2], sf[2];
    if constexpr (PAIR) {
      if (!nothing) {
        weights(0, pf, sf);
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) pf[c] = sf[c] = v8{};
      }
      v8 own[2], other[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        own[c] = second ? sf[c] : pf[c];
        *reinterpret_cast<v8*>(&swap[wid][c][lane * 8]) = second ? pf[c] : sf[c];
      }
      tile_barrier();
#pragma unroll
      for (int c = 0; c < 2; ++c) other[c] = *reinterpret_cast<const v8*>(&swap[wid ^ 1][c][lane * 8]);
      if (!nothing)   // (the same for both of a pair)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const v8 mid = (c >> 1) == second ? own[c & 1] : other[c & 1];
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) dv[n] = mfma(tr_frag(qt + 16 * c * DP, ta[n]), mid, dv[n]);
      }
    } else if (!nothing) {
#pragma unroll
      for (int rows = 0; rows < 64; rows += 32) {
        weights(rows, pf, sf);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int n = 0; n < DP / 32; ++n) {
            dv[n] = mfma(tr_frag(dt + (rows + 16 * c) * DP, ta[n]), pf[c], dv[n]);
            dk[n] = mfma(tr_frag(qt + (rows + 16 * c) * DP, ta[n]), sf[c], dk[n]);
          }
      }
    }
    if (++t == t1) { t = t0; ++hg; }
    if (i + 2 < i1) load((buf + 2) % 3);
  };
  for (int i = i0; i < i1; i += 3) {
    step(i, std::integral_constant<int, 0>{});
    if (i + 1 < i1) step(i + 1, std::integral_constant<int, 1>{});
    if (i + 2 < i1) step(i + 2, std::integral_constant<int, 2>{});
  }
  if (key >= p.tk) return;
  const long krow = (long)b * p.tk + key;
  auto leave = [&](const f32x16 (&acc)[DP / 32], float k, int which, T* out) __attribute__((always_inline)) {   // which: 0 dK, 1 dV
    float* pk = parts > 1 ? bk.part + ((((long)part * 2 + which) * p.nb * p.tk + krow) * p.kvh + kh) * DP : nullptr;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int col = 32 * n + 8 * g + 4 * hh;
        if (col >= p.d) continue;
        f32x4 a;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = ok ? acc[n][4 * g + e] * k : 0.0f;
        if (pk) *reinterpret_cast<f32x4*>(pk + col) = a;
        else put4(out + col, a);
      }
  };
  T *to_k = (T*)p.dk + krow * p.lddk + kh * p.d, *to_v = (T*)p.dv + krow * p.lddv + kh * p.d;
  const float of_k = ds_scale(p) / f, of_v = is_half<T> ? 6.103515625e-05f : 1.0f;
  if constexpr (PAIR) {
    leave(dv, second ? of_k : of_v, !second, second ? to_k : to_v);
  } else {
    leave(dk, of_k, 0, to_k);
    leave(dv, of_v, 1, to_v);
  }
}

// The parts of split sweeps added in their order, four columns to a thread: [n][rows][per][DP] to rows of `per` heads of d columns.
struct Parts {
  const float* part;
  int n, per;
  long rows, stride;   // stride: from a part to the next
  void* out;
  int ld;
  const int* parts;    // of each block of 128 rows of a sequence of t, or NULL: n everywhere
  int t;
};
template <typename T, int DP>
__global__ __launch_bounds__(256) void add_parts_kernel(Parts a, Parts b, Parts c, int d) {
  const Parts p = blockIdx.y == 0 ? a : blockIdx.y == 1 ? b : c;
  const long i = (long)blockIdx.x * 256 + threadIdx.x, rh = i / (DP / 4);
  const int col = (int)(i % (DP / 4)) * 4;
  if (rh >= p.rows * p.per || col >= d) return;
  const long row = rh / p.per;
  const int n = p.parts ? p.parts[row / p.t * ((p.t + 127) / 128) + row % p.t / 128] : p.n;
  if (n == 1) return;   // it is there
  const float* src = p.part + rh * DP + col;
  f32x4 s = {};
#pragma unroll 4
  for (int k = 0; k < n; ++k) s += *reinterpret_cast<const f32x4*>(src + k * p.stride);
  put4((T*)p.out + row * p.ld + rh % p.per * d + col, s);
}

// Splits of dkv_kernel's sweep, where its blocks do not fill the card: no shorter than 8 tiles each.  us of the whole backward with
// 1, 2, 3, 4, 8: 6912 x 5 heads of 64 (270 blocks) 390, 354, 325, 328, 344; 4608 x 5 (180) 200, 166, 184, 166, 176; 8 x 1728 x 10 (1120)
// 294, 312, 345, 365, 508; causal, heads of 128: 4096 x 32/8 (256) 691, 520, 553, 542, 617; 2 x 2500 x 16/4 (160) 401, 269, 254, 257, 282.
int dkv_splits(const dc_attn_desc* d) {
  if (const Lists l = lists_of(d); l.on) return l.most_k;
  const long blocks = (long)d->nb * d->kv_heads * ((d->tk + 127L) / 128);
  const long steps = (long)(d->heads / d->kv_heads) * ((d->tq + 63L) / 64);
  return (int)max(1L, min(min((d->d > 64 ? 600 : 900) / blocks, steps / 8), 8L));
}
long pad16(long bytes) { return (bytes + 15) / 16 * 16; }

long rows_bytes(const dc_attn_desc* d) { return 4L * d->nb * d->heads * ((d->tq + 127L) / 128 * 128); }
long rows32_bytes(const dc_attn_desc* d) { return pad16(8L * d->nb * d->heads * ((d->tq + 127L) / 128 * 4)); }
long part_bytes(const dc_attn_desc* d) {
  const int n = dkv_splits(d);
  return n > 1 ? 8L * n * d->nb * d->tk * d->kv_heads * (d->d > 64 ? 128 : 64) : 0;
}
long part_q_bytes(const dc_attn_desc* d) {
  const int n = tile_splits(d, true);
  return n > 1 ? 4L * n * d->nb * d->tq * d->heads * (d->d > 64 ? 128 : 64) : 0;
}
long bwd_ws_bytes(const dc_attn_desc* d) {
  return summary_bytes(d, true) + 2 * rows_bytes(d) + rows32_bytes(d) + part_bytes(d) + part_q_bytes(d);
}

template <typename T, int DP, int FORM>
void launch_bwd(const Call& c, const Back& bk, hipStream_t st) {
  const long nqb = (long)c.nb * ((c.tq + 127) / 128), nkb = (long)c.nb * ((c.tk + 127) / 128);
  const dim3 grid((unsigned)(c.heads * (c.list_q ? c.entries_q : nqb * bk.nq)));
  if (c.tk <= kExact * 64) hipLaunchKernelGGL((dq_kernel<T, DP, FORM, true>), grid, dim3(256), 0, st, c, bk);
  else hipLaunchKernelGGL((dq_kernel<T, DP, FORM, false>), grid, dim3(256), 0, st, c, bk);
  hipLaunchKernelGGL((dkv_kernel<T, DP, FORM>), dim3((unsigned)(c.kvh * (c.list_k ? c.entries_k : nkb * bk.nk))),
                     dim3(DP == 64 ? 256 : 512), 0, st, c, bk);
  const long nk = (long)c.nb * c.tk * c.kvh, nq = (long)c.nb * c.tq * c.heads;
  const Parts none{};
  const Parts dk{bk.part, bk.nk, c.kvh, (long)c.nb * c.tk, 2 * nk * DP, c.dk, c.lddk, c.parts_k, c.tk}, dv{bk.part + nk * DP, bk.nk, c.kvh,
                 (long)c.nb * c.tk, 2 * nk * DP, c.dv, c.lddv, c.parts_k, c.tk}, dq{bk.part_q, bk.nq, c.heads, (long)c.nb * c.tq, nq * DP, c.dq, c.lddq, c.parts_q, c.tq};
  const long most = max(bk.nk > 1 ? nk : 0, bk.nq > 1 ? nq : 0);
  if (most)
    hipLaunchKernelGGL((add_parts_kernel<T, DP>), dim3((unsigned)((most * (DP / 4) + 255) / 256), bk.nk > 1 ? 3 : 1), dim3(256), 0,
                       st, bk.nq > 1 ? dq : none, bk.nk > 1 ? dk : none, bk.nk > 1 ? dv : none, c.d);
}
template <typename T, int DP>
void launch_bwd(const Call& c, const Back& bk, hipStream_t st) {
  if (c.wide != 0.0f) launch_bwd<T, DP, WIDE>(c, bk, st);
  else if (c.cap2 != 0.0f || c.slopes) launch_bwd<T, DP, SHAPED>(c, bk, st);
  else launch_bwd<T, DP, PLAIN>(c, bk, st);
}

}  // namespace

long long fwd_ws_bytes(const dc_attn_desc* d);

}  // namespace dcm

using namespace dcm;

extern "C" long long dc_attn_mask_ws_bytes(const dc_attn_desc* d, int backward) {
  if (!shape_ok(d)) return 0;
  return backward ? bwd_ws_bytes(d) : fwd_ws_bytes(d);
}

extern "C" int dc_attn_mask_bwd(const dc_attn_desc* d, void* scratch, long long ws_bytes, void* stream) {
  Call c;
  if (const int rc = make_call(d, c, true)) return rc;
  if (!scratch || bwd_ws_bytes(d) > ws_bytes) return DC_ERR_ARG;
  if ((uintptr_t)scratch & 15) return DC_ERR_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  char* ws = static_cast<char*>(scratch);
  launch_summaries(d, c, true, ws, st);
  ws += summary_bytes(d, true);
  Back bk;
  bk.nlse = reinterpret_cast<float*>(ws);
  bk.ndel = reinterpret_cast<float*>(ws + rows_bytes(d));
  bk.rows32 = reinterpret_cast<int2*>(ws + 2 * rows_bytes(d));
  bk.n32 = (d->tq + 127) / 128 * 4;
  bk.nq = tile_splits(d, true);
  bk.nk = dkv_splits(d);
  bk.part = reinterpret_cast<float*>(ws + 2 * rows_bytes(d) + rows32_bytes(d));
  bk.part_q = reinterpret_cast<float*>(ws + 2 * rows_bytes(d) + rows32_bytes(d) + part_bytes(d));
  if (d->type == 0) d->d > 64 ? launch_bwd<bf16, 128>(c, bk, st) : launch_bwd<bf16, 64>(c, bk, st);
  else d->d > 64 ? launch_bwd<half, 128>(c, bk, st) : launch_bwd<half, 64>(c, bk, st);
  DC_CHECK_LAUNCH();
  return DC_OK;
}
