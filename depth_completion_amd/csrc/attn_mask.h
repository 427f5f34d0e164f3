// Shared device helpers of the masked attention kernels (attn_mask_fwd.hip, attn_mask_bwd.hip): fragment types of the two
// storage types, the LDS tile with its swizzle and the loads into it, which block takes what, and the description of a call.
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
  float scale, mul;       // score scale; what turns a score into the exponent of 2: scale log2 e, or 1 where the scores are capped
  float wide;             // 1 / softcap of a cap above kWideCap, else 0
  float cap2, icap, bend; // softcap log2 e, 2 log2 e scale / softcap (0: none); what makes slopes fit scores: 1 / scale, log2 e with a cap
  const float* slopes;
  int causal;
  const int *prefix, *kv_len, *doc_q, *doc_k;
  const int4 *sum_q, *sum_k;   // per 64 rows: least and largest document, whether a row is in none (NULL: short rows, no documents)
  // documents in few blocks: (block of 128 rows, part | parts << 8) or (-1, 0), the longest parts first; parts of each block (NULL: not)
  const int2 *list_q, *list_k;
  const int *parts_q, *parts_k;
  int entries_q, entries_k;
};

// What the scores pass: nothing but their scale; a cap or a bias; a cap above kWideCap (and a bias).
enum { PLAIN, SHAPED, WIDE };
// Scores of a call with a cap, in units of log2: cap2 tanh(scale s / cap), with tanh(x) = 1 - 2 r, r = 1 / (1 + e^2x).  slope: r - r^2,
// a quarter of 1 - tanh^2.  The difference leaves tanh an absolute error below 2e-7, and the cap multiplies it: a score is off by
// under 1.3e-5 at a cap of 64, by 0.2 at 1e6.  Wider caps, whose scores lie far below them, take the function whose error is relative
// (kernels of their own: as a branch beside the other form it takes dQ's at 64 columns past their 168 registers).
constexpr float kWideCap = 64.0f;
template <int FORM>
__device__ __forceinline__ float cap_score(const Call& p, float s, float* slope) {
  if constexpr (FORM == WIDE) {
    const float t = tanhf(s * p.scale * p.wide);
    if (slope) *slope = 0.25f * fmaf(-t, t, 1.0f);
    return p.cap2 * t;
  }
  const float r = __builtin_amdgcn_rcpf(1.0f + exp2_raw(s * p.icap));
  if (slope) *slope = fmaf(-r, r, r);
  return fmaf(-2.0f * p.cap2, r, p.cap2);
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

// Four transposed fragments of 128 columns (rows from tile + IMM bytes on), read and waited for in one block: the compiler, which
// takes the builtin's reads for reads of what is still on its way into LDS, would wait for the next tile here.
struct TrAt4 {
  unsigned lo[4], hi[4];
  template <typename T>
  __device__ __forceinline__ void init(const T* lds, int lane) {
    const unsigned base = (unsigned)(unsigned long)((DC_LDS const char*)lds);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const TrAt o = tr_at<128>(32 * n, lane);
      lo[n] = base + o.lo * 2;
      hi[n] = base + o.hi * 2;
    }
  }
};
template <typename T, int IMM>
__device__ __forceinline__ void tr_frags(const TrAt4& a, typename Vec<T>::v8 (&f)[4]) {
  struct Two { unsigned long long lo, hi; } r[4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%16\n\tds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
      "ds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
      "ds_read_b64_tr_b16 %6, %14 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%16\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0].lo), "=&v"(r[0].hi), "=&v"(r[1].lo), "=&v"(r[1].hi), "=&v"(r[2].lo), "=&v"(r[2].hi), "=&v"(r[3].lo),
        "=&v"(r[3].hi)
      : "v"(a.lo[0]), "v"(a.hi[0]), "v"(a.lo[1]), "v"(a.hi[1]), "v"(a.lo[2]), "v"(a.hi[2]), "v"(a.lo[3]), "v"(a.hi[3]), "n"(IMM));
#pragma unroll
  for (int n = 0; n < 4; ++n) f[n] = __builtin_bit_cast(typename Vec<T>::v8, r[n]);
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

// 64 x DP elements into an LDS tile by NT threads, straight from memory (16 bytes a lane, no registers between).  A lane's offsets
// are the same for every tile; the tile's first row is in the scalar base (64 bits, so a long cache needs no wide offsets).  Rows
// behind `last`, rows that `keep` leaves out and columns from d on take an offset outside the descriptor and arrive as zeros:
// nothing that lies in a masked place is ever multiplied.
template <typename T, int DP, int NT = 256>
struct Dma {
  static constexpr int CH = DP / 8, N = 64 * CH / NT, STEP = NT / CH;
  static constexpr unsigned OUT = 0x80000000u;
  unsigned off[N];
  int row, wave;
  __device__ __forceinline__ void init(int ld, int d) {
    row = threadIdx.x / CH;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = row + STEP * i, c = (int)(threadIdx.x % CH) ^ sw<DP>(r);
      off[i] = c * 8 < d ? ((unsigned)r * ld + c * 8) * sizeof(T) : OUT;
    }
  }
  __device__ __forceinline__ static __amdgpu_buffer_rsrc_t rsrc(const T* base) {
    const unsigned long long a = (unsigned long long)base;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
    return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | lo), (short)0, 0x7fffffff, 0x00020000);
  }
  __device__ __forceinline__ void put(__amdgpu_buffer_rsrc_t r, T* tile, int i, unsigned o) const {
#if defined(__HIP_DEVICE_COMPILE__)   // (the builtin exists in the device pass alone)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (DC_LDS char*)(tile + (64 * wave + NT * i) * 8), 16, o, 0, 0, 0);
#endif
  }
  __device__ __forceinline__ void load(const T* base, T* tile, int last) const {
    const __amdgpu_buffer_rsrc_t r = rsrc(base);
    if (last >= 63) {
#pragma unroll
      for (int i = 0; i < N; ++i) put(r, tile, i, off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) put(r, tile, i, row + STEP * i <= last ? off[i] : OUT);
    }
  }
  template <typename F>
  __device__ __forceinline__ void load_some(const T* base, T* tile, int last, F&& keep) const {
    const __amdgpu_buffer_rsrc_t r = rsrc(base);
    bool in[N];
#pragma unroll
    for (int i = 0; i < N; ++i) in[i] = row + STEP * i <= last && keep(row + STEP * i);
#pragma unroll
    for (int i = 0; i < N; ++i) put(r, tile, i, in[i] ? off[i] : OUT);
  }
};
// 64 words into LDS, by one wave
__device__ __forceinline__ void dma_words(const void* base, void* lds, int last) {
  const int lane = threadIdx.x & 63;
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(Dma<bf16, 64>::rsrc((const bf16*)base), (DC_LDS char*)lds, 4,
                                           lane <= last ? lane * 4u : Dma<bf16, 64>::OUT, 0, 0, 0);
#endif
}
// Waits until at most N vector-memory operations of this wave are under way: those issued before the last N have landed (whatever
// else was issued before them among these).
template <int N>
__device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// All waves: what each has waited for is there for all, and what each has read may be overwritten.  (__syncthreads() would also
// wait for the tiles that are on their way.)
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ int length_of(const Call& p, int b) {
  return p.kv_len ? min(max(p.kv_len[b], 0), p.tk) : p.tk;
}
// over a wave, in every lane, by cross-lane moves
template <int CTRL>
__device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
template <typename F>
__device__ __forceinline__ int lanes_reduce(int v, F&& f) {
  v = f(v, moved<0xb1>(v));    // lane ^ 1
  v = f(v, moved<0x4e>(v));    // lane ^ 2
  v = f(v, moved<0x141>(v));   // the other four of eight
  v = f(v, moved<0x140>(v));   // the other eight of sixteen
  auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = f((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f((int)r[0], (int)r[1]);
}
__device__ __forceinline__ int wave_min_i(int v) {
  return lanes_reduce(v, [](int a, int b) __attribute__((always_inline)) { return min(a, b); });
}
__device__ __forceinline__ int wave_max_i(int v) {
  return lanes_reduce(v, [](int a, int b) __attribute__((always_inline)) { return max(a, b); });
}
// the sum / maximum of a value over lanes l and l ^ 32, which hold the two halves of a query's scores
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Which unit (a key head of a sequence, or of all where the items are sorted), item (its blocks of rows, the longest first) and part of
// an item a block takes.  Blocks are dealt to the eight XCDs in turn, and by these to their CUs in turn, 256 at a time.
//   Many blocks (or the decode's): units go to an XCD whole as far as they come by eights, so that the blocks that read the same keys
//   share an L2; the blocks of the rest are spread over all (whole units left over would leave XCDs idle).
//   At most 1536, which are on the card at once or nearly, so that no later block evens out what the first have left: the longest items
//   of all units first, and the second 256 in the reverse order (`fold`), a short block beside each long one.  Causal, forward and
//   gradients, us by whole units and so: 4096 x 16 heads of 64 306 255, 2 x 2048 x 16 170 145, 8 x 1024 x 16 210 191, 4608 x 5 155 134.
constexpr int kSpread = 1536;
struct Place { int unit, item, part; };
__device__ __forceinline__ Place place_of(int units, int items, int parts, bool spread, bool fold) {
  Place at;
  int i = blockIdx.x;
  if (spread) {
    const int j = i / 8, end = min((int)gridDim.x, 512) / 8;
    if (fold && j >= 32 && j < end) i = (31 + end - j) * 8 + i % 8;
    at.unit = i % units;
    i /= units;
  } else {
    const int per_unit = items * parts, whole = units / 8 * 8, n = whole * per_unit;
    at.unit = i < n ? i / 8 / per_unit * 8 + i % 8 : whole + (i - n) / per_unit;
    i = i < n ? i / 8 % per_unit : (i - n) % per_unit;
  }
  at.part = i % parts;
  at.item = i / parts;
  return at;
}

// (the same for all lanes, which the compiler does not see of a load)
__device__ __forceinline__ int2 entry_of(const int2* list, int i) {
  const int2 e = list[i];
  return make_int2(__builtin_amdgcn_readfirstlane(e.x), __builtin_amdgcn_readfirstlane(e.y));
}

// The query rows of a block of fwd_kernel or dq_kernel: 4 x 32 rows of one head.
struct QueryBlock {
  int b, kh, h, part, parts, qi, len, pos, lim, mine;   // lim: the lane's query sees the keys below it (of its document `mine`)
  bool live, idle;   // idle: the block has nothing to do
  int4 sum0;   // the thread's first tile summary, read along with the rows
  __device__ __forceinline__ void init(const Call& p, int splits) {
    const int nqb = (p.tq + 127) / 128;
    const Place at = p.list_q ? place_of(p.kvh, p.entries_q, p.grp, true, true)
                              : place_of(p.nb * p.kvh, nqb, p.grp * splits, gridDim.x <= kSpread, true);
    const int2 e = p.list_q ? entry_of(p.list_q, at.item)
                            : make_int2(p.causal ? nqb - 1 - at.item : at.item, at.part / p.grp | splits << 8);
    const int item = max(e.x, 0);
    idle = e.x < 0;
    b = p.list_q ? item / nqb : at.unit / p.kvh;
    kh = at.unit % p.kvh;
    h = kh * p.grp + at.part % p.grp;
    part = e.y & 255;
    parts = e.y >> 8;
    len = length_of(p, b);
    qi = (p.list_q ? item % nqb : item) * 128 + (threadIdx.x >> 6) * 32 + (threadIdx.x & 31);
    live = qi < p.tq;
    pos = qi + len - p.tq;
    lim = p.causal ? min(len, max(pos + 1, p.prefix ? p.prefix[b] : 0)) : len;
    mine = p.doc_q ? (live ? p.doc_q[(long)b * p.tq + qi] : -1) : 0;
    if (mine < 0) lim = 0;
    if (p.sum_k) {
      const int nt = (p.tk + 63) / 64;
      sum0 = p.sum_k[(long)b * nt + min((int)threadIdx.x, nt - 1)];
    }
  }
  // The 64-key tiles [t0, t1) in which some row with `sees` may see a key; holes: the first of them with a key that is (or may be)
  // in no document.
  __device__ __forceinline__ void tiles(const Call& p, bool sees, int* range, int& t0, int& t1, int& holes) const {
    if (threadIdx.x == 0) { range[0] = 0x7fffffff; range[1] = 0; range[2] = 0x7fffffff; range[3] = -1; range[4] = 0; range[5] = 0x7fffffff; }
    __syncthreads();
    const int most = wave_max_i(sees ? lim : 0);
    if ((threadIdx.x & 63) == 0) atomicMax(&range[1], most);
    if (p.sum_k && sees && mine >= 0) { atomicMin(&range[2], mine); atomicMax(&range[3], mine); }
    __syncthreads();
    t0 = 0;
    t1 = (range[1] + 63) / 64;
    if (p.sum_k) {
      const int nt = (p.tk + 63) / 64, least = range[2], largest = range[3];
      const int4* sum = p.sum_k + (long)b * nt;
      int first = 0x7fffffff, last = -1;
      for (int t = threadIdx.x; t < t1; t += 256) {
        const int4 s = t < 256 ? sum0 : sum[t];
        if (s.y >= least && s.x <= largest) { first = min(first, t); last = t; }
      }
      if (last >= 0) { atomicMin(&range[0], first); atomicMax(&range[4], last + 1); }
      __syncthreads();
      t1 = range[4];
      t0 = min(range[0], t1);
      for (int t = threadIdx.x; t < t1; t += 256)
        if (t >= t0 && (t < 256 ? sum0 : sum[t]).z) { atomicMin(&range[5], t); break; }
      __syncthreads();
    }
    holes = p.doc_q && !p.sum_k ? 0 : __builtin_amdgcn_readfirstlane(range[5]);
    t0 = __builtin_amdgcn_readfirstlane(t0);
    t1 = __builtin_amdgcn_readfirstlane(t1);
  }
};

// What a wave has to do with a tile of keys: nothing (no row sees one of them), all without a mask, or a mask.
struct WaveRange {
  int all, any, least, most;   // keys that every live row sees, that some row does; the rows' documents
  __device__ __forceinline__ void init(const QueryBlock& q, bool live) {
    all = __builtin_amdgcn_readfirstlane(wave_min_i(live ? q.lim : 0x7fffffff));
    any = __builtin_amdgcn_readfirstlane(wave_max_i(live ? q.lim : 0));
    least = __builtin_amdgcn_readfirstlane(wave_min_i(live && q.mine >= 0 ? q.mine : 0x7fffffff));
    most = __builtin_amdgcn_readfirstlane(wave_max_i(live ? q.mine : -1));
  }
  enum { NOTHING, WHOLE, MASKED };
  // id: the keys' documents, or NULL
  __device__ __forceinline__ int look(int t, const int* id) const {
    if (t * 64 >= any) return NOTHING;
    bool masked = t * 64 + 64 > all;
    if (id) {
      const int i = id[threadIdx.x & 63];
      if (!__any(i >= least && i <= most)) return NOTHING;
      masked |= least != most || __any(i != least);
    }
    return masked ? MASKED : WHOLE;
  }
};

// The keys' tiles of a query block in LDS, S of them in turn: K, V and the keys' documents.
template <typename T, int DP, int S>
struct KeyRing {
  static constexpr int TILE = 64 * DP;
  struct Lds {
    __attribute__((aligned(16))) T tiles[S][2 * TILE];
    __attribute__((aligned(16))) int ids[S][64];
  };
  Dma<T, DP> k, v;
  const T *kb, *vb;
  const int* kid;
  const int4* sum;
  int len, holes;
  __device__ __forceinline__ void init(const Call& p, const QueryBlock& q, int first_hole) {
    holes = first_hole;
    k.init(p.ldk, p.d);
    v.init(p.ldv, p.d);
    kb = (const T*)p.k + (long)q.b * p.tk * p.ldk + q.kh * p.d;
    vb = (const T*)p.v + (long)q.b * p.tk * p.ldv + q.kh * p.d;
    kid = p.doc_q ? p.doc_k + (long)q.b * p.tk : nullptr;
    sum = p.sum_k ? p.sum_k + (long)q.b * ((p.tk + 63) / 64) : nullptr;
    len = q.len;
  }
  // tile t on its way (each wave issues 2 Dma::N operations or more)
  __device__ __forceinline__ void load(const Call& p, Lds& lds, int t, int buf) const {
    const int r0 = t * 64, last = len - 1 - r0;
    const T *ka = kb + (long)r0 * p.ldk, *va = vb + (long)r0 * p.ldv;
    // a key in no document: its row may hold anything (asked for each tile, the answer would be waited for in each; rows in none lie
    // behind the last document, as a rule)
    if (t >= holes && (!sum || sum[t].z)) {
      auto keep = [&](int r) __attribute__((always_inline)) { return kid[min(r0 + r, len - 1)] >= 0; };
      k.load_some(ka, lds.tiles[buf], last, keep);
      v.load_some(va, lds.tiles[buf] + TILE, last, keep);
    } else {
      k.load(ka, lds.tiles[buf], last);
      v.load(va, lds.tiles[buf] + TILE, last);
    }
    if (kid && k.wave == 0) dma_words(kid + r0, lds.ids[buf], last);
  }
};

// Host side: what both directions share (attn_mask_fwd.hip).
constexpr int kMaxSplit = 64;
bool shape_ok(const dc_attn_desc* d);
int tile_splits(const dc_attn_desc* d, bool backward);
struct Lists { bool on; int items_q, items_k, entries_q, entries_k, most_q, most_k; };   // most: parts of a block
Lists lists_of(const dc_attn_desc* d);
int make_call(const dc_attn_desc* d, Call& c, bool backward);
long long summary_bytes(const dc_attn_desc* d, bool backward);
void launch_summaries(const dc_attn_desc* d, Call& c, bool backward, char* ws, hipStream_t st);

}  // namespace dcm
