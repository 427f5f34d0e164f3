// Masked attention forward (gfx950): grouped heads, documents, causal with a prefix, filled key lengths, tanh-capped scores and a
// bias that falls with distance; head dims to 128, bf16 and fp16, 32x32x16 MFMA.
//
// Scores are held transposed (S^T = K Q^T, a query to a lane), so the running maximum and sum of a row stay in the lane and
// P feeds O^T += V^T P^T straight from the accumulator.  Two kernels share that product:
//   fwd_kernel    128 query rows of one head to a block; tiles of 64 keys pass through LDS, two of them on their way.
//   token_kernel  few query rows: all rows of a key head's query heads (up to 32) to a wave, each wave its own 32 keys at a time,
//                 keys read straight into fragments.  It reads every key and value once, whatever the group.
// Where rows are few the keys are split over blocks; each writes (m, l, O) in 32 bits and join_kernel adds them in split order.
#include "attn_mask.h"
#include <type_traits>

namespace dcm {
namespace {

// least and largest document of 64 rows (rows in none left out), and whether a row is in none: the keys' tiles, then the queries'
__global__ __launch_bounds__(256) void summary_kernel(const int* doc_k, int tk, int nk, const int* doc_q, int tq, int nq, int nb,
                                                      int4* out) {
  int i = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (i >= nb * (nk + nq)) return;
  int4* to = out + i;
  const bool q = i >= nb * nk;
  if (q) i -= nb * nk;
  const int* doc = q ? doc_q : doc_k;
  const int t = q ? tq : tk, nt = q ? nq : nk;
  const int b = i / nt, r = (i % nt) * 64 + lane;
  const int id = r < t ? doc[(long)b * t + r] : -1;
  const int lo = wave_min_i(id >= 0 ? id : 0x7fffffff), hi = wave_max_i(id);
  const bool none = __any(r < t && id < 0);
  if (lane == 0) *to = make_int4(lo, hi, none, 0);
}

// The same tiles by one block, for calls of few blocks, and the lists of what these take: blocks of 128 rows in parts of as many tiles
// as give the card its fill, the longest first.  A block's tiles are those of the other side that its documents meet (a prefix left
// out).  list_k is NULL in the forward.  What it costs (12 us for 9001 rows, where summary_kernel takes 5) buys the balance: us unsorted with even parts and so, forward
// and with the gradients, 5 heads of 64, 9001 rows: the longest document first 91 88, 324 323, last 156 114, 518 377; 4 x 4700 111 104,
// 397 365; 10 heads, 4700 67 59, 236 207.
constexpr int kSorted = 1024;   // tiles, and blocks of either side
__global__ __launch_bounds__(1024) void plan_kernel(Call p, int nk, int nq, Lists l, int4* out, int2* list_q, int* parts_q, int2* list_k,
                                                    int* parts_k) {
  __shared__ int4 sum[kSorted];
  __shared__ int cost[kSorted], sums[16];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // a tile to a wave, eight on their way
  auto side = [&](const int* doc, int rows, int nt, int4* to, int4* copy) __attribute__((always_inline)) {
    int b = 0, t = wid;   // of the wave's next tile
    auto settle = [&]() __attribute__((always_inline)) {
      while (t >= nt && b < p.nb) { t -= nt; ++b; }
    };
    settle();
    while (b < p.nb) {
      int id[8], at[8], left[8], m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (b >= p.nb) break;
        left[k] = rows - t * 64;
        at[k] = b * nt + t;
        id[k] = doc[(long)b * rows + t * 64 + min(lane, left[k] - 1)];
        t += 16;
        settle();
        m = k + 1;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k >= m) break;
        // (lanes behind the last row have its document)
        const int lo = wave_min_i(id[k] >= 0 ? id[k] : 0x7fffffff), hi = wave_max_i(max(id[k], -1));
        const bool none = __any(id[k] < 0);
        if (lane == 0) to[at[k]] = copy[at[k]] = make_int4(lo, hi, none, 0);
      }
    }
  };
  side(p.doc_k, p.tk, nk, out, sum);
  if (nq) side(p.doc_q, p.tq, nq, out + p.nb * nk, sum + p.nb * nk);
  const int4* sum_q = nq ? sum + p.nb * nk : sum;
  const int nt_q = (p.tq + 63) / 64;
  auto fill = [&](bool keys, int2* list, int* parts) __attribute__((always_inline)) {   // a block of rows to a wave
    const int nt = keys ? nk : nt_q, blocks = (nt + 1) / 2, items = p.nb * blocks;
    const int entries = keys ? l.entries_k : l.entries_q, most_parts = keys ? l.most_k : l.most_q;
    __syncthreads();
    int b = 0, w = wid;
    for (int i = wid; i < items; i += 16, w += 16) {
      while (w >= blocks) { w -= blocks; ++b; }
      const int len = length_of(p, b), shift = len - p.tq;
      const int4 *own = (keys ? sum : sum_q) + b * nt, first = own[2 * w], second = own[min(2 * w + 1, nt - 1)];
      const int least = min(first.x, second.x), most = max(first.y, second.y);
      const int4* other = keys ? sum_q + b * nt_q : sum + b * nk;
      const int seen = min(len, p.causal ? w * 128 + 128 + shift : len);   // keys that the queries w 128 .. see
      const int from = keys && p.causal ? max(0, w * 128 - shift) / 64 : 0;
      const int to = !keys ? (max(seen, 0) + 63) / 64 : w * 128 < len ? nt_q : 0;
      int c = 0;
      for (int t = from; t < to; t += 64) {
        const int4 o = other[min(t + lane, to - 1)];
        c += __popcll(__ballot(t + lane < to && o.y >= least && o.x <= most));
      }
      if (lane == 0) cost[i] = c;
    }
    __syncthreads();
    // the least of 16 lengths of a part, from an even share to the longest block, whose parts fit the list: a length to a wave
    int total = 0, longest = 0;
    for (int i = lane; i < items; i += 64) {
      total += cost[i];
      longest = max(longest, cost[i]);
    }
    total = lanes_reduce(total, [](int a, int b) __attribute__((always_inline)) { return a + b; });
    longest = wave_max_i(longest);
    const float share = fmaxf((float)total / entries, keys ? fmaxf(1.0f, 8.0f / p.grp) : 8.0f);
    auto length = [&](int k) __attribute__((always_inline)) { return share + fmaxf(longest - share, 0.0f) * (k / 15.0f); };
    // (of the longest length the list holds all: no more than `even` parts each; its blocks are one part though the quotient is rounded)
    const int even = entries / items;
    auto parts_of = [&](int c, float len) __attribute__((always_inline)) {
      return max(1, min(most_parts, max((int)ceilf(c * __builtin_amdgcn_rcpf(len) - 1e-3f), min(even, (c + 7) / 8))));
    };
    int sum_parts = 0;
    for (int i = lane; i < items; i += 64) sum_parts += parts_of(cost[i], length(wid));
    sum_parts = lanes_reduce(sum_parts, [](int a, int b) __attribute__((always_inline)) { return a + b; });
    if (lane == 0) sums[wid] = sum_parts;
    __syncthreads();
    const int k = __ffsll(__ballot(sums[lane & 15] <= entries || lane >= 15)) - 1, filled = sums[k];
    const float len = length(k);
    for (int i = threadIdx.x; i < items; i += 1024) {
      const int n = parts_of(cost[i], len);
      parts[i] = n;
      cost[i] = (cost[i] + n - 1) / n * 16 + n;
    }
    for (int i = filled + threadIdx.x; i < entries; i += 1024) list[i] = make_int2(-1, 0);
    __syncthreads();
    for (int i = wid; i < items; i += 16) {
      const int c = cost[i], n = c & 15;
      int at = 0;   // parts of the blocks before this one
      for (int j = lane; j < items; j += 64) {
        const int o = cost[j];
        if (o >> 4 > c >> 4 || (o >> 4 == c >> 4 && j < i)) at += o & 15;
      }
      at = lanes_reduce(at, [](int a, int b) __attribute__((always_inline)) { return a + b; });
      if (lane < n && at + lane < entries) list[at + lane] = make_int2(i, lane | n << 8);
    }
  };
  fill(false, list_q, parts_q);
  if (list_k) fill(true, list_k, parts_k);
}

// Running softmax of one lane's query over tiles of scores.  m is the reference of the weights 2^(x - m); it follows the row's
// maximum only when that has grown by more than 8 log2 e, so that most tiles leave O alone.  A row that has seen no key keeps
// m = -inf and weights of zero.  fp16 weights are held 2^4 times as large: with the slack they reach 2^15.6, and one key among
// many may weigh 2^-28 before it is rounded away.
template <typename T, int DP>
struct Row {
  static constexpr int NO = DP / 32;
  static constexpr float SHIFT = sizeof(Vec<T>) && __is_same(T, half) ? 4.0f : 0.0f;
  float m, l;
  f32x16 o[NO];
  __device__ __forceinline__ void init() {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int n = 0; n < NO; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;
  }
  // weights of NB blocks of scores, in place; mul turns a score into an exponent of 2
  template <int NB>
  __device__ __forceinline__ void weigh(f32x16 (&s)[NB], float mul) {
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
    mx = pair_max(mx) * mul;
    if (__any(mx > m + 8.0f * kLog2e)) {
      const float up = fmaxf(m, mx);
      const float k = up > m ? exp2_raw(m - up) : 1.0f;
#pragma unroll
      for (int n = 0; n < NO; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] *= k;
      l *= k;
      m = up;
    }
    const float ref = (m == -INFINITY ? 0.0f : m) - SHIFT;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = exp2_raw(fmaf(s[b][r], mul, -ref));
        sum[r & 3] += s[b][r];
      }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
  __device__ __forceinline__ void merge(float m2, float l2, const float* o2, int stride) {
    const float up = fmaxf(m, m2);
    const float a = up > m ? exp2_raw(m - up) : 1.0f, b = up > m2 ? exp2_raw(m2 - up) : 1.0f;
    l = l * a + l2 * b;
#pragma unroll
    for (int n = 0; n < NO; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[n][r] = o[n][r] * a + o2[(16 * n + r) * stride] * b;
    m = up;
  }
};

struct Split {
  int n;        // splits of the keys
  int tiles;    // token_kernel: 32-key steps of a split
  float* o;     // [row][n][DP]
  float* ml;    // [row][n][2], row = (sequence, head, query)
};

// O and the log-sum of a finished row; hh: which half of each eight columns the lane holds
template <typename T, int DP>
__device__ __forceinline__ void put_row(const Call& p, const Row<T, DP>& s, float l, long row, long orow, int h, int hh) {
  const float inv = 1.0f / l;
  const bool none = l == 0.0f;
  T* o = (T*)p.o + orow * p.ldo + h * p.d;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * n + 8 * g + 4 * hh;
      if (col >= p.d) continue;
      typename Vec<T>::v4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)(none ? 0.0f : s.o[n][4 * g + e] * inv);
      *reinterpret_cast<typename Vec<T>::v4*>(o + col) = v;
    }
  if (hh == 0) p.lse[row] = none ? -INFINITY : (s.m + (__builtin_amdgcn_logf(l) - s.SHIFT)) * kLn2;
}
template <typename T, int DP>
__device__ __forceinline__ void put_part(const Split& sp, const Row<T, DP>& s, float l, long row, int part, int hh) {
  float* o = sp.o + (row * sp.n + part) * DP;
  if (hh == 0) *reinterpret_cast<float2*>(sp.ml + (row * sp.n + part) * 2) = make_float2(s.m, l);
  if (s.m == -INFINITY) return;   // no weight in it: join_kernel does not read O
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = s.o[n][4 * g + e];
      *reinterpret_cast<f32x4*>(o + 32 * n + 8 * g + 4 * hh) = v;
    }
}

// A step: tile i has landed (waited for, barrier), S, softmax, P V; then tile i + 2 is sent to the buffer that tile i - 1 left.  The
// transposed reads carry no alias information, so the compiler waits for every load into LDS before them: sent any earlier, a tile
// would be waited for at once.  128 columns hold two tiles alone (three would leave one block to a CU): there tile i + 1 is sent when
// the step begins, and the reads are waited for in blocks of their own (tr_frags).
template <typename T, int DP, int FORM>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void fwd_kernel(Call p, Split sp) {
  typedef typename Vec<T>::v8 v8;
  constexpr int S = DP == 64 ? 3 : 2, TILE = 64 * DP, OPS = 2 * Dma<T, DP>::N;
  typedef KeyRing<T, DP, S> Ring;
  __shared__ typename Ring::Lds lds;
  __shared__ int range[6];
  const int lane = threadIdx.x & 63, hh = lane >> 5;
  QueryBlock q;
  q.init(p, sp.n);
  if (q.idle) return;
  const T* qrow = (const T*)p.q + ((long)q.b * p.tq + q.qi) * p.ldq + q.h * p.d;
  v8 qf[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) qf[s] = load8_or_0(qrow + 16 * s + 8 * hh, q.live && 16 * s + 8 * hh < p.d);
  int t0, t1;
  int holes;
  q.tiles(p, q.live, range, t0, t1, holes);
  if (q.parts > 1) {
    const int each = (t1 - t0 + q.parts - 1) / q.parts;
    t0 = min(t1, t0 + q.part * each);
    t1 = min(t1, t0 + each);
  }
  Ring ring;
  ring.init(p, q, holes);
  Row<T, DP> st;
  st.init();
  const float slope = FORM != PLAIN && p.slopes ? p.slopes[q.h] * p.bend : 0.0f;
  int koff[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) koff[s] = tile_at<DP>(lane & 31, 2 * s + hh);
  TrAt va[2];
  TrAt4 va4;
  if constexpr (DP == 128) va4.init(lds.tiles[0], lane);
  else
#pragma unroll
    for (int n = 0; n < 2; ++n) va[n] = tr_at<DP>(32 * n, lane);
  WaveRange range_of;
  range_of.init(q, q.live);

  if (t0 < t1) ring.load(p, lds, t0, 0);
  if (S == 3 && t0 + 1 < t1) ring.load(p, lds, t0 + 1, 1);
  auto tile = [&](int t, auto B, const int* id, bool masked) __attribute__((always_inline)) {
    constexpr int buf = decltype(B)::value;
    const T* kt = lds.tiles[buf];
    const T* vt = kt + TILE;
    f32x16 s[2];
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2) {
      s[kb2] = f32x16{};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) s[kb2] = mfma(*reinterpret_cast<const v8*>(kt + 32 * kb2 * DP + koff[c]), qf[c], s[kb2]);
    }
    if constexpr (FORM != PLAIN) {
      if (p.cap2 != 0.0f) {
#pragma unroll
        for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb2][r] = cap_score<FORM>(p, s[kb2][r], nullptr);
      }
      if (p.slopes) {
        const float dist = (float)(q.pos - t * 64 - 4 * hh);
#pragma unroll
        for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[kb2][r] = fmaf(-slope, fabsf(dist - (float)(32 * kb2 + (r & 3) + 8 * (r >> 2))), s[kb2][r]);
      }
    }
    if (masked) {
      asm volatile("" ::: "memory");   // a branch, not selects in every tile
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int key = 32 * kb2 + 8 * g + 4 * hh;
          int4 i4 = make_int4(0, 0, 0, 0);
          if (id) i4 = *reinterpret_cast<const int4*>(&id[key]);
          const int id4[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t * 64 + key + e >= q.lim || (id && id4[e] != q.mine)) s[kb2][4 * g + e] = -INFINITY;
        }
    }
    st.weigh(s, p.mul);
    auto add = [&](auto C) __attribute__((always_inline)) {
      constexpr int c = decltype(C)::value;
      v8 f[DP / 32];
      if constexpr (DP == 128) tr_frags<T, (buf * 2 * TILE + TILE + 16 * c * DP) * 2>(va4, f);
      else
#pragma unroll
        for (int n = 0; n < 2; ++n) f[n] = tr_frag(vt + 16 * c * DP, va[n]);
      const v8 pf = acc_frag<T>(s[c >> 1], c & 1);
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) st.o[n] = mfma(f[n], pf, st.o[n]);
    };
    add(std::integral_constant<int, 0>{});
    add(std::integral_constant<int, 1>{});
    add(std::integral_constant<int, 2>{});
    add(std::integral_constant<int, 3>{});
  };
  auto step = [&](int t, auto B) __attribute__((always_inline)) {
    constexpr int buf = decltype(B)::value;
    if (S == 3 && t + 1 < t1) vm_wait<OPS>();
    else vm_wait<0>();
    tile_barrier();
    if (S == 2 && t + 1 < t1) ring.load(p, lds, t + 1, buf ^ 1);
    const int* id = ring.kid ? lds.ids[buf] : nullptr;
    const int look = range_of.look(t, id);
    if (look != WaveRange::NOTHING) tile(t, B, id, look == WaveRange::MASKED);
    if (S == 3 && t + 2 < t1) ring.load(p, lds, t + 2, (buf + 2) % 3);
  };
  for (int t = t0; t < t1; t += S) {
    step(t, std::integral_constant<int, 0>{});
    if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{});
    if constexpr (S == 3)
      if (t + 2 < t1) step(t + 2, std::integral_constant<int, 2>{});
  }
  const float l = pair_sum(st.l);
  if (!q.live) return;
  const long row = ((long)q.b * p.heads + q.h) * p.tq + q.qi;
  if (q.parts > 1) put_part<T, DP>(sp, st, l, row, q.part, hh);
  else put_row<T, DP>(p, st, l, row, (long)q.b * p.tq + q.qi, q.h, hh);
}

// One block: up to 32 of the rows (query, head of the group) of one key head, `sp.tiles` steps of 4 x 32 keys.
template <typename T, int DP, int FORM>
__global__ __launch_bounds__(256, 2) void token_kernel(Call p, Split sp) {
  typedef typename Vec<T>::v8 v8;
  constexpr int SUB = 32 * DP, NV = SUB / 8 / 64, CH = DP / 8, RED = (2 + DP / 2) * 64;
  constexpr int BYTES = 4 * SUB * 2 > 3 * RED * 4 ? 4 * SUB * 2 : 3 * RED * 4;
  __shared__ __attribute__((aligned(16))) char smem[BYTES];
  const int lane = threadIdx.x & 63, hh = lane >> 5, wid = threadIdx.x >> 6;
  const int rows = p.tq * p.grp, nrb = (rows + 31) / 32;
  const Place at = place_of(p.nb * p.kvh, sp.n, nrb, false, false);
  const int b = at.unit / p.kvh, kh = at.unit % p.kvh;
  const int rb = at.part, part = at.item;
  const int r = rb * 32 + (lane & 31);
  const bool live = r < rows;
  const int qi = live ? r / p.grp : 0, h = kh * p.grp + (live ? r % p.grp : 0);
  const int len = length_of(p, b), pos = qi + len - p.tq, pre = p.prefix ? p.prefix[b] : 0;
  int lim = p.causal ? min(len, max(pos + 1, pre)) : len;
  const int mine = p.doc_q ? p.doc_q[(long)b * p.tq + qi] : 0;
  if (mine < 0 || !live) lim = 0;
  const int end = wave_max_i(lim);   // the same in the four waves
  const T* qrow = (const T*)p.q + ((long)b * p.tq + qi) * p.ldq + h * p.d;
  v8 qf[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) qf[s] = load8_or_0(qrow + 16 * s + 8 * hh, live && 16 * s + 8 * hh < p.d);
  const T* kb = (const T*)p.k + (long)b * p.tk * p.ldk + kh * p.d;
  const T* vb = (const T*)p.v + (long)b * p.tk * p.ldv + kh * p.d;
  const int* kid = p.doc_q ? p.doc_k + (long)b * p.tk : nullptr;
  T* vt = reinterpret_cast<T*>(smem) + wid * SUB;
  const float slope = FORM != PLAIN && p.slopes ? p.slopes[h] * p.bend : 0.0f;
  TrAt va[DP / 32];
#pragma unroll
  for (int n = 0; n < DP / 32; ++n) va[n] = tr_at<DP>(32 * n, lane);

  Row<T, DP> st;
  st.init();
  v8 kf[DP / 16];
  uint4 vr[NV];
  const int steps = (end + 31) / 32, u1 = min(steps, (part + 1) * sp.tiles * 4);
  // keys from `end` on, and columns from d on, read a place that is valid; their weights, or their columns, are zeroed
  auto fetch = [&](int u) __attribute__((always_inline)) {
    const long key = min(u * 32 + (lane & 31), end - 1);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int c = 16 * s + 8 * hh;
      kf[s] = *reinterpret_cast<const v8*>(kb + key * p.ldk + (c < p.d ? c : 0));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int piece = lane + 64 * i, c = piece % CH * 8;
      vr[i] = *reinterpret_cast<const uint4*>(vb + (long)min(u * 32 + piece / CH, end - 1) * p.ldv + (c < p.d ? c : 0));
    }
  };
  int u = part * sp.tiles * 4 + wid;
  if (u < u1) fetch(u);
  for (; u < u1; u += 4) {
    int my_key_id = 0;
    if (kid) {   // a key in no document: its row may hold anything
      my_key_id = kid[min(u * 32 + (lane & 31), end - 1)];
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
        if (my_key_id < 0) kf[s] = v8{};
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (__shfl(my_key_id, (lane + 64 * i) / CH, 64) < 0) vr[i] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int piece = lane + 64 * i;
      *reinterpret_cast<uint4*>(vt + tile_at<DP>(piece / CH, piece % CH)) = vr[i];
    }
    f32x16 s[1] = {f32x16{}};
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) s[0] = mfma(kf[c], qf[c], s[0]);   // qf is zero where the columns end
    if (u + 4 < u1) fetch(u + 4);
    if constexpr (FORM != PLAIN) {
      if (p.cap2 != 0.0f) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[0][e] = cap_score<FORM>(p, s[0][e], nullptr);
      }
      if (p.slopes) {
        const float dist = (float)(pos - u * 32 - 4 * hh);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[0][e] = fmaf(-slope, fabsf(dist - (float)((e & 3) + 8 * (e >> 2))), s[0][e]);
      }
    }
    if (kid || __any(lim < u * 32 + 32)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = 8 * (e >> 2) + 4 * hh + (e & 3);
        const bool other = kid && __shfl(my_key_id, key, 64) != mine;
        if (u * 32 + key >= lim || other) s[0][e] = -INFINITY;
      }
    }
    st.weigh(s, p.mul);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const v8 pf = acc_frag<T>(s[0], c);
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) st.o[n] = mfma(tr_frag(vt + 16 * c * DP, va[n]), pf, st.o[n]);
    }
  }
  float l = pair_sum(st.l);
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
  if (wid > 0) {
    float* dst = red + (wid - 1) * RED + lane;
    dst[0] = st.m;
    dst[64] = l;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) dst[(2 + 16 * n + e) * 64] = st.o[n][e];
  }
  __syncthreads();
  if (wid > 0) return;
  st.l = l;
#pragma unroll
  for (int o = 0; o < 3; ++o) {
    const float* src = red + o * RED + lane;
    st.merge(src[0], src[64], src + 128, 64);
  }
  if (!live) return;
  const long row = ((long)b * p.heads + h) * p.tq + qi;
  if (sp.n > 1) put_part<T, DP>(sp, st, st.l, row, part, hh);
  else put_row<T, DP>(p, st, st.l, row, (long)b * p.tq + qi, h, hh);
}

// A row's splits joined, four columns to a lane.  G groups of lanes take every G-th split each and are added in order: one group to a
// row where there are many rows, a whole block where there are few.  us of calls with one group and with a block to a row: one token
// over 131072 keys in 64 splits 142 119, 4 tokens over 4096 keys, 32/8 heads of 128, 19 16; 512 over 4096, 16 of 64, 32 38; 4608 x 5
// of 64 45 61.
template <typename T, int DP, int G>
__global__ __launch_bounds__(256) void join_kernel(Call p, Split sp, long rows) {
  constexpr int LANES = DP / 4;
  __shared__ float red[G == 1 ? 1 : G][G == 1 ? 1 : LANES][5];
  const long row = ((long)blockIdx.x * 256 + threadIdx.x) / (LANES * G);
  const int lane = threadIdx.x % LANES, col = lane * 4, grp = G == 1 ? 0 : threadIdx.x / LANES;
  if (row >= rows) return;
  const long bh = row / p.tq, q = row % p.tq, b = bh / p.heads;
  const int n = p.parts_q ? p.parts_q[b * ((p.tq + 127) / 128) + q / 128] : sp.n;
  if (p.parts_q && n == 1) return;   // it is there
  const float2* ml = reinterpret_cast<const float2*>(sp.ml) + row * sp.n;
  float top = -INFINITY;
  if constexpr (G == 1) {
#pragma unroll 4
    for (int i = 0; i < n; ++i) top = fmaxf(top, ml[i].x);
  } else {
    top = wave_max((int)(threadIdx.x & 63) < n ? ml[threadIdx.x & 63].x : -INFINITY);   // (at most 64 splits)
  }
  float l = 0.0f;
  f32x4 o = {};
  const float* src = sp.o + row * sp.n * DP + col;
#pragma unroll 4
  for (int i = grp; i < n; i += G) {
    const float2 x = ml[i];
    // a split without weights left no O; one that saw NaN scores alone has m = -inf and l = NaN, which has to reach the result
    const float k = x.x == -INFINITY ? 0.0f : exp2_raw(x.x - top);
    l += x.y != x.y ? x.y : x.y * k;
    if (x.x != -INFINITY) o += *reinterpret_cast<const f32x4*>(src + (long)i * DP) * k;
  }
  if constexpr (G > 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) red[grp][lane][e] = o[e];
    red[grp][lane][4] = l;
    __syncthreads();
    if (grp) return;
    for (int i = 1; i < G; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += red[i][lane][e];
      l += red[i][lane][4];
    }
  }
  const int h = (int)(bh % p.heads);
  const bool none = l == 0.0f;
  const float inv = 1.0f / l;
  if (col < p.d) {
    typename Vec<T>::v4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)(none ? 0.0f : o[e] * inv);
    *reinterpret_cast<typename Vec<T>::v4*>((T*)p.o + (b * p.tq + q) * p.ldo + h * p.d + col) = v;
  }
  if (col == 0) p.lse[row] = none ? -INFINITY : (top + (__builtin_amdgcn_logf(l) - Row<T, DP>::SHIFT)) * kLn2;
}

// Few query rows (at most 64 in a sequence, half of fwd_kernel's block): token_kernel.  us with token_kernel and fwd_kernel for 8, 32, 64
// and 96 rows a sequence: 1 x 4096 keys, 32/8 heads of 128: 16 33, 17 34, 27 36, 35 39; 8 x 4096, 32/8 of 128: 42 100, 74 104, 113 114,
// 157 121; 16 x 2048, 16/2 of 64: 13 27, 25 27, 33 33, 43 37; 4 x 1000, 20 of 64: 13 22, 14 22, 16 23, 17 23.
bool few_rows(int tq) { return tq <= 64; }

// How the keys of few rows are split: enough blocks to give every CU four where the keys allow it, each with 4 steps of 128 keys or
// more (the steps a block has cover its start and its merge); of many rows, tile_splits.
Split split_of(const dc_attn_desc* d) {
  Split s{1, 0, nullptr, nullptr};
  const long grp = d->heads / d->kv_heads;
  if (few_rows(d->tq)) {
    const long blocks = (long)d->nb * d->kv_heads * ((d->tq * grp + 31) / 32), steps = (d->tk + 127L) / 128;
    long n = (1024 + blocks - 1) / blocks;
    n = min(min(n, (steps + 3) / 4), (long)kMaxSplit);
    s.tiles = (int)((steps + n - 1) / n);
    s.n = (int)((steps + s.tiles - 1) / s.tiles);
  } else {
    s.n = tile_splits(d, false);
  }
  return s;
}

long part_floats(const dc_attn_desc* d, const Split& s) {
  if (s.n <= 1) return 0;
  return (long)d->nb * d->heads * d->tq * s.n * ((d->d > 64 ? 128 : 64) + 2);
}

template <typename T, int DP, int FORM>
void launch_fwd(const Call& c, const dc_attn_desc* d, Split s, hipStream_t st) {
  if (few_rows(d->tq)) {
    const long blocks = (long)c.nb * c.kvh * ((c.tq * c.grp + 31) / 32) * s.n;
    hipLaunchKernelGGL((token_kernel<T, DP, FORM>), dim3((unsigned)blocks), dim3(256), 0, st, c, s);
  } else {
    const long blocks = c.heads * (c.list_q ? (long)c.entries_q : (long)c.nb * ((c.tq + 127) / 128) * s.n);
    hipLaunchKernelGGL((fwd_kernel<T, DP, FORM>), dim3((unsigned)blocks), dim3(256), 0, st, c, s);
  }
  const long rows = (long)c.nb * c.heads * c.tq, threads = rows * (DP / 4);
  if (s.n <= 1) return;
  if (threads >= 65536)   // a thread to every lane of the card
    hipLaunchKernelGGL((join_kernel<T, DP, 1>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, c, s, rows);
  else
    hipLaunchKernelGGL((join_kernel<T, DP, 1024 / DP>), dim3((unsigned)rows), dim3(256), 0, st, c, s, rows);
}
template <typename T, int DP>
void launch_fwd(const Call& c, const dc_attn_desc* d, Split s, hipStream_t st) {
  if (c.wide != 0.0f) launch_fwd<T, DP, WIDE>(c, d, s, st);
  else if (c.cap2 != 0.0f || c.slopes) launch_fwd<T, DP, SHAPED>(c, d, s, st);
  else launch_fwd<T, DP, PLAIN>(c, d, s, st);
}

}  // namespace

// Splits of the keys of blocks of 128 rows: only where the card is not full, to 4/3 of what it holds (a few long blocks more than it
// has CUs for would double the time), each split 8 tiles of 64 or
// more, 3 where blocks are very few, 16 in the backward (whose short rows are not split).  Forward, us with 1, 2, 4, 8 splits: 6912 x 5 heads of 64
// (270 blocks) 147, 108, 100, 106; 4608 x 5 (180) 86, 59, 50, 56; 1728 x 10 (140 blocks of 27 tiles) 33, 33, 31, 34; 8 x 1728 x 10
// (1120) 94, 106, 125, 194: the 32-bit parts cost their writing and reading.  With splits of 16, 8, 5 and 3
// tiles: 92 x 829 keys, 3 heads of 128 (3 blocks) 25, 25, 19, 15; 100 x 1000, 20 of 64 (20) 20, 18, 16, 15; 1000 x 8 of 128 (64) 30, 26,
// 25, 26; 432 x 20 (80) 12, 12, 12, 15; 1000 x 16 (128) 21, 23, 25, 27; 1728 x 10 (140) 34, 28, 30, 34.  With documents (where no list is
// made) many of the blocks are short, and what the card holds is enough.
int tile_splits(const dc_attn_desc* d, bool backward) {
  const long blocks = (long)d->nb * d->heads * ((d->tq + 127L) / 128), tiles = (d->tk + 63L) / 64;
  const long slots = 256 * (d->d > 64 ? 2 : 3);   // blocks that the card holds at once
  if (const Lists l = lists_of(d); l.on) return l.most_q;
  if (3 * blocks >= 2 * slots) return 1;
  const long n = d->doc_q ? slots / blocks : (4 * slots / 3 + blocks - 1) / blocks;
  return (int)min(min(n, max(tiles / (backward ? 16 : blocks > 64 ? 8 : 3), 1L)), (long)kMaxSplit);
}

// Short rows go without summaries: the kernels visit every tile, and look at the documents of every key that they load.  us with and
// without, 10 heads of 64, forward and gradients: 8 x 256 in 2 documents 47 38, 4 x 512 in 1 76 70, in 4 47 51, 4 x 1024 in 2 112 131.
// token_kernel does not ask for them.
bool summarised(const dc_attn_desc* d, bool backward) {
  return d->doc_q && (d->tq > 512 || d->tk > 512) && (backward || !few_rows(d->tq));
}
// Lists where blocks are few (place_of) and one block can look at all tiles.  Entries: as many as the card holds (4/3 of it: 4 to 10 %
// slower), or a block of rows each; a block has twice its even share of parts at most, as its documents may be the longest.
Lists lists_of(const dc_attn_desc* d) {
  const long nk = (d->tk + 63L) / 64, nq = (d->tq + 63L) / 64, bq = d->nb * ((nq + 1) / 2), bk = d->nb * ((nk + 1) / 2);
  Lists l{};
  l.on = summarised(d, false) && d->nb * (nk + nq) <= kSorted && bq * d->heads <= kSpread;
  if (!l.on) return l;
  l.items_q = (int)bq;
  l.items_k = (int)bk;
  const long slots = 256 * (d->d > 64 ? 2 : 3) / d->heads, slots_k = (d->d > 64 ? 600 : 900) / d->kv_heads;
  l.most_q = (int)max(1L, min(min(8L, 2 * slots / bq), nk / 16));
  l.most_k = (int)max(1L, min(min(8L, 2 * slots_k / bk), nq * (d->heads / d->kv_heads) / 16));
  l.entries_q = (int)(l.most_q > 1 ? max(bq, slots) : bq);
  l.entries_k = (int)(l.most_k > 1 ? max(bk, slots_k) : bk);
  return l;
}
// the queries' tiles are the keys' where the documents are the same rows; the forward asks for them only to sort
bool query_tiles(const dc_attn_desc* d, bool backward) {
  return (backward || lists_of(d).on) && !(d->doc_q == d->doc_k && d->tq == d->tk);
}

long long summary_bytes(const dc_attn_desc* d, bool backward) {
  if (!summarised(d, backward)) return 0;
  const long long sums = 16LL * d->nb * ((d->tk + 63L) / 64 + (query_tiles(d, backward) ? (d->tq + 63L) / 64 : 0));
  const Lists l = lists_of(d);
  return sums + (l.on ? (8LL * (l.entries_q + l.entries_k) + 4LL * (l.items_q + l.items_k) + 15) / 16 * 16 : 0);
}

void launch_summaries(const dc_attn_desc* d, Call& c, bool backward, char* ws, hipStream_t st) {
  if (!summarised(d, backward)) return;
  const int nk = (d->tk + 63) / 64, nq = query_tiles(d, backward) ? (d->tq + 63) / 64 : 0;
  int4* k = reinterpret_cast<int4*>(ws);
  c.sum_k = k;
  c.sum_q = nq ? k + (long)d->nb * nk : k;
  if (const Lists l = lists_of(d); l.on) {
    int2 *lq = reinterpret_cast<int2*>(k + (long)d->nb * (nk + nq)), *lk = backward ? lq + l.entries_q : nullptr;
    int *pq = reinterpret_cast<int*>(lq + l.entries_q + l.entries_k), *pk = pq + l.items_q;
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, st, c, nk, nq, l, k, lq, pq, lk, pk);
    c.list_q = lq;
    c.list_k = lk;
    c.parts_q = pq;
    c.parts_k = pk;
    c.entries_q = l.entries_q;
    c.entries_k = l.entries_k;
    return;
  }
  hipLaunchKernelGGL(summary_kernel, dim3((unsigned)((d->nb * (nk + nq) + 3) / 4)), dim3(256), 0, st, d->doc_k, d->tk, nk, d->doc_q,
                     d->tq, nq, d->nb, k);
}

// Lengths and heads that make sense, with row counts within 31 bits (splits included) and the threads of a launch within 32.
bool shape_ok(const dc_attn_desc* d) {
  if (!d || d->nb <= 0 || d->tq <= 0 || d->tk <= 0 || d->heads <= 0 || d->kv_heads <= 0 || d->heads % d->kv_heads) return false;
  const long long q = (long long)d->nb * d->heads, k = (long long)d->nb * d->kv_heads;
  return q < (1LL << 30) / d->tq && k < (1LL << 30) / d->tk && q * ((d->tq + 127LL) / 128) < (1LL << 23) &&
         k * ((d->tk + 127LL) / 128) < (1LL << 23);
}

int make_call(const dc_attn_desc* d, Call& c, bool backward) {
  if (!shape_ok(d) || !d->q || !d->k || !d->v || !d->o || !d->lse || d->type < 0 || d->type > 1) return DC_ERR_ARG;
  if (d->d <= 0 || d->d > 128 || d->d % 8 || !(d->scale > 0.0f) || !(d->softcap >= 0.0f)) return DC_ERR_ARG;
  if (!(d->scale <= 1e30f) || !(d->softcap <= 1e30f) || (d->softcap > 0.0f && !(d->scale / d->softcap <= 1e30f))) return DC_ERR_ARG;
  if ((d->prefix && !d->causal) || (d->slopes && !(d->scale >= 1e-30f))) return DC_ERR_ARG;
  if (!d->doc_q != !d->doc_k) return DC_ERR_ARG;
  const long long hq = (long long)d->heads * d->d, hk = (long long)d->kv_heads * d->d;
  if (d->ldq < hq || d->ldo < hq || d->ldk < hk || d->ldv < hk) return DC_ERR_ARG;
  if (d->ldk > (1 << 23) || d->ldv > (1 << 23)) return DC_ERR_ARG;   // 128 rows within 32 bits
  if (d->ldq % 8 || d->ldk % 8 || d->ldv % 8 || d->ldo % 8) return DC_ERR_ALIGN;
  const uintptr_t at = (uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v | (uintptr_t)d->o;
  if (at & 15) return DC_ERR_ALIGN;
  if (backward) {
    if (!d->dout || !d->dq || !d->dk || !d->dv) return DC_ERR_ARG;
    if (d->ldq > (1 << 23) || d->lddo > (1 << 23) || d->lddo < hq || d->lddq < hq || d->lddk < hk || d->lddv < hk) return DC_ERR_ARG;
    if (d->lddo % 8 || d->lddq % 8 || d->lddk % 8 || d->lddv % 8) return DC_ERR_ALIGN;
    if (((uintptr_t)d->dout | (uintptr_t)d->dq | (uintptr_t)d->dk | (uintptr_t)d->dv) & 15) return DC_ERR_ALIGN;
  }
  c = Call{};
  c.q = d->q; c.k = d->k; c.v = d->v; c.o = d->o; c.lse = d->lse;
  c.dout = d->dout; c.dq = d->dq; c.dk = d->dk; c.dv = d->dv;
  c.ldq = d->ldq; c.ldk = d->ldk; c.ldv = d->ldv; c.ldo = d->ldo;
  c.lddo = d->lddo; c.lddq = d->lddq; c.lddk = d->lddk; c.lddv = d->lddv;
  c.nb = d->nb; c.tq = d->tq; c.tk = d->tk; c.heads = d->heads; c.kvh = d->kv_heads; c.grp = d->heads / d->kv_heads; c.d = d->d;
  c.scale = d->scale;
  c.mul = d->softcap > 0.0f ? 1.0f : d->scale * kLog2e;
  c.bend = d->softcap > 0.0f ? kLog2e : 1.0f / d->scale;
  if (d->softcap > 0.0f) {
    c.cap2 = d->softcap * kLog2e;
    c.icap = 2.0f * kLog2e * d->scale / d->softcap;
    c.wide = d->softcap > kWideCap ? 1.0f / d->softcap : 0.0f;
  }
  c.slopes = d->slopes;
  c.causal = d->causal;
  c.prefix = d->prefix; c.kv_len = d->kv_len; c.doc_q = d->doc_q; c.doc_k = d->doc_k;
  return DC_OK;
}

long long fwd_ws_bytes(const dc_attn_desc* d) { return summary_bytes(d, false) + 4LL * part_floats(d, split_of(d)); }

}  // namespace dcm

using namespace dcm;

extern "C" int dc_attn_mask_fwd(const dc_attn_desc* d, void* scratch, long long ws_bytes, void* stream) {
  Call c;
  if (const int rc = make_call(d, c, false)) return rc;
  if (fwd_ws_bytes(d) > (scratch ? ws_bytes : 0)) return DC_ERR_ARG;
  if ((uintptr_t)scratch & 15) return DC_ERR_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  char* ws = static_cast<char*>(scratch);
  launch_summaries(d, c, false, ws, st);
  Split s = split_of(d);
  if (s.n > 1) {
    s.o = reinterpret_cast<float*>(ws + summary_bytes(d, false));
    s.ml = s.o + (long)d->nb * d->heads * d->tq * s.n * (d->d > 64 ? 128 : 64);
  }
  if (d->type == 0) d->d > 64 ? launch_fwd<bf16, 128>(c, d, s, st) : launch_fwd<bf16, 64>(c, d, s, st);
  else d->d > 64 ? launch_fwd<half, 128>(c, d, s, st) : launch_fwd<half, 64>(c, d, s, st);
  DC_CHECK_LAUNCH();
  return DC_OK;
}
