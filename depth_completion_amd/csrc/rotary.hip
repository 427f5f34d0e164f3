// Rotary positions (gfx950): pairs of a head's columns turned by position x frequency, forward and gradient (the turn back).
//
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t), t = pos f_i;  pairs (i, i + rot / 2) or (2 i, 2 i + 1) of the rot columns
//   from `off`; the other columns are copied (or stay, in place).
//
// Bound by HBM: every value is read and written once.  A thread holds the sines of V pairs of one row and takes them through
// several heads, so the angles cost little; these are formed in 64 bits and reduced to a turn there, since pos f_i at position 1e6
// keeps no digits of its fraction in 32.  16-bit types take the sine unit (turns in, absolute error about 2^-20), fp32 sincospif.
#include "common.h"
#include "../../include/dcamd.h"
#include <math.h>

namespace {

typedef _Float16 half;

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

template <typename T>
__device__ __forceinline__ void sin_cos(double pos, double f, float& s, float& c) {
  const double turns = pos * f * 0.15915494309189535;
  const float r = (float)(turns - rint(turns));
  if constexpr (sizeof(T) == 2) {
    s = __builtin_amdgcn_sinf(r);
    c = __builtin_amdgcn_cosf(r);
  } else {
    sincospif(2.0f * r, &s, &c);
  }
}

struct Rotary {
  const void* x;
  void* y;
  long ldx, ldy, rows;
  int heads, d, off, rot;
  const double* freqs;
  const int* pos;
  int pos0, t;
  float mag;
  int inverse, hpt, nturn, units;   // heads to a thread; of a head's units, those that turn
};

// A unit: V pairs (two packs of V columns), or two packs that are copied (the last of an odd count twice).  Both run the same loads
// and stores, the copied ones keep their bits by a select, so a wave whose lanes lie over a whole head stays together.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(Rotary p) {
  typedef Pack<T, V> P;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = i / p.units;
  const int u = (int)(i - row * p.units);
  const int h0 = blockIdx.y * p.hpt, h1 = min(p.heads, h0 + p.hpt);
  if (row >= p.rows) return;
  const bool turns = u < p.nturn;
  int at[2];
  float s[V], c[V];
  if (turns) {
    at[0] = INTER ? p.off + u * 2 * V : p.off + u * V;
    at[1] = INTER ? at[0] + V : at[0] + p.rot / 2;
    const double pos = p.pos ? (double)p.pos[row] : (double)p.pos0 + (double)(row % p.t);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      sin_cos<T>(pos, p.freqs[u * V + k], s[k], c[k]);
      s[k] *= p.inverse ? -p.mag : p.mag;
      c[k] *= p.mag;
    }
  } else {
    const int rest = (p.d - p.rot) / V;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = min(2 * (u - p.nturn) + k, rest - 1) * V;
      at[k] = j < p.off ? j : j + p.rot;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) s[k] = c[k] = 0.0f;
  }
  const T* x = (const T*)p.x + row * p.ldx + (long)h0 * p.d;
  T* y = (T*)p.y + row * p.ldy + (long)h0 * p.d;
  auto turn = [&](const P& a, const P& b, T* to) __attribute__((always_inline)) {
    P r[2] = {a, b};
    if (turns) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        // elements 2 k and 2 k + 1 of the 2 V columns, or k of either half
        const int n0 = INTER ? 2 * k / V : 0, n1 = INTER ? (2 * k + 1) / V : 1;
        const int e0 = INTER ? 2 * k % V : k, e1 = INTER ? (2 * k + 1) % V : k;
        const float e = (float)(n0 ? b : a).v[e0], f = (float)(n1 ? b : a).v[e1];
        r[n0].v[e0] = (T)(e * c[k] - f * s[k]);
        r[n1].v[e1] = (T)(e * s[k] + f * c[k]);
      }
    }
    *reinterpret_cast<P*>(to + at[0]) = r[0];
    *reinterpret_cast<P*>(to + at[1]) = r[1];
  };
  int h = h0;
  for (; h + 4 <= h1; h += 4, x += 4 * p.d, y += 4 * p.d) {   // four heads' reads before the first is used
    P a[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[k] = *reinterpret_cast<const P*>(x + k * p.d + at[0]);
      b[k] = *reinterpret_cast<const P*>(x + k * p.d + at[1]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) turn(a[k], b[k], y + k * p.d);
  }
  for (; h < h1; ++h, x += p.d, y += p.d)
    turn(*reinterpret_cast<const P*>(x + at[0]), *reinterpret_cast<const P*>(x + at[1]), y);
}

template <typename T, int V>
int launch(Rotary p, int interleaved, hipStream_t st) {
  p.nturn = p.rot / (2 * V);
  p.units = p.nturn + (p.x == p.y ? 0 : ((p.d - p.rot) / V + 1) / 2);
  if (p.rows >= (1LL << 32) / p.units) return DC_ERR_ARG;   // a launch's threads
  // enough threads to fill the card (2^19) come before heads that share their sines; past 8 heads these cost nothing
  const long all = p.rows * p.units * p.heads;
  p.hpt = (int)min((long)min(p.heads, 8), max(1L, all >> 19));
  const dim3 grid((unsigned)((p.rows * p.units + 255) / 256), (unsigned)((p.heads + p.hpt - 1) / p.hpt));
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, V, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((rotary_kernel<T, V, false>), grid, dim3(256), 0, st, p);
  DC_CHECK_LAUNCH();
  return DC_OK;
}

// Packs of 16 bytes where every pack of a head starts on one, else single columns.
template <typename T>
int launch_type(const Rotary& p, int interleaved, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = p.rot % (2 * V) == 0 && p.off % V == 0 && p.d % V == 0 && p.ldx % V == 0 && p.ldy % V == 0 &&
                    (((uintptr_t)p.x | (uintptr_t)p.y) & 15) == 0;
  return wide ? launch<T, V>(p, interleaved, st) : launch<T, 1>(p, interleaved, st);
}

}  // namespace

extern "C" int dc_rotary(const dc_rotary_desc* r, void* stream) {
  if (!r || !r->x || !r->y || !r->freqs || r->type < 0 || r->type > 2 || r->rows <= 0 || r->heads <= 0 || r->d <= 0) return DC_ERR_ARG;
  const int d = r->d, heads = r->heads;
  if (r->rot <= 0 || r->rot % 2 || r->off < 0 || r->off > d || r->rot > d - r->off || d > 65536 || heads > 65535) return DC_ERR_ARG;
  if ((long long)heads * d >= (1LL << 31) || (r->x == r->y && r->ldx != r->ldy)) return DC_ERR_ARG;
  if (r->ldx < (long long)heads * d || r->ldy < (long long)heads * d || (!r->pos && r->t <= 0)) return DC_ERR_ARG;
  if (r->rows > (1LL << 38) / d) return DC_ERR_ARG;
  const uintptr_t size = r->type == 2 ? 4 : 2;
  if ((((uintptr_t)r->x | (uintptr_t)r->y) & (size - 1)) || ((uintptr_t)r->freqs & 7) || ((uintptr_t)r->pos & 3)) return DC_ERR_ALIGN;
  Rotary p{r->x, r->y, (long)r->ldx, (long)r->ldy, (long)r->rows, heads, d, r->off, r->rot, r->freqs, r->pos, r->pos0, r->t, r->mag,
           r->inverse, 0, 0, 0};
  hipStream_t st = (hipStream_t)stream;
  if (r->type == 0) return launch_type<bf16>(p, r->interleaved, st);
  if (r->type == 1) return launch_type<half>(p, r->interleaved, st);
  return launch_type<float>(p, r->interleaved, st);
}

extern "C" int dc_rotary_freqs(int rot, double theta, int scaling, double factor, double trained, double fast, double slow,
                               double* freqs, float* mag) {
  if (rot <= 0 || rot % 2 || !(theta > 1.0) || !(theta <= 1e300) || !freqs || !mag || scaling < 0 || scaling > 3) return DC_ERR_ARG;
  if (scaling && !(factor >= 1.0 && factor <= 1e9)) return DC_ERR_ARG;
  if (scaling == 2 && rot < 4) return DC_ERR_ARG;
  if (scaling == 3 && !(trained > 0.0 && trained <= 1e12 && fast > slow && slow >= 0.0 && fast <= 1e12)) return DC_ERR_ARG;
  const double base = scaling == 2 ? theta * pow(factor, (double)rot / (rot - 2)) : theta;
  *mag = 1.0f;
  for (int i = 0; i < rot / 2; ++i) {
    double f = pow(base, -2.0 * i / rot);
    if (scaling == 1) f /= factor;
    if (scaling == 3) {   // turns over the trained length: many stay as they are, few are slowed down, a ramp between
      const double turns = trained * f * 0.15915494309189535;
      const double keep = fmin(1.0, fmax(0.0, (turns - slow) / (fast - slow)));
      f = f * keep + f / factor * (1.0 - keep);
    }
    freqs[i] = f;
  }
  if (scaling == 3) *mag = (float)(0.1 * log(factor) + 1.0);
  return DC_OK;
}
