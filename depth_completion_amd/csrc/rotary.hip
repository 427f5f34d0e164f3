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

// A unit: V pairs (two packs of V columns), or two packs of V columns that are copied.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(Rotary p) {
  typedef Pack<T, V> P;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = i / p.units;
  const int u = (int)(i - row * p.units);
  const int h0 = blockIdx.y * p.hpt, h1 = min(p.heads, h0 + p.hpt);
  if (row >= p.rows) return;
  const T* x = (const T*)p.x + row * p.ldx;
  T* y = (T*)p.y + row * p.ldy;
  if (u >= p.nturn) {
    const int rest = (p.d - p.rot) / V;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = 2 * (u - p.nturn) + k;
      if (j >= rest) break;
      const int at = j * V < p.off ? j * V : j * V + p.rot;
      for (int h = h0; h < h1; ++h) *reinterpret_cast<P*>(y + h * p.d + at) = *reinterpret_cast<const P*>(x + h * p.d + at);
    }
    return;
  }
  const double pos = p.pos ? (double)p.pos[row] : (double)p.pos0 + (double)(row % p.t);
  const int a0 = INTER ? p.off + u * 2 * V : p.off + u * V, b0 = INTER ? a0 + V : a0 + p.rot / 2;
  float s[V], c[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    sin_cos<T>(pos, p.freqs[u * V + k], s[k], c[k]);
    s[k] *= p.inverse ? -p.mag : p.mag;
    c[k] *= p.mag;
  }
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const P a = *reinterpret_cast<const P*>(x + h * p.d + a0), b = *reinterpret_cast<const P*>(x + h * p.d + b0);
    P ya, yb;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      // element 2 k and 2 k + 1 of the 2 V columns, or k of either half
      const float e = (float)(!INTER ? a.v[k] : 2 * k < V ? a.v[2 * k % V] : b.v[2 * k % V]);
      const float f = (float)(!INTER ? b.v[k] : 2 * k + 1 < V ? a.v[(2 * k + 1) % V] : b.v[(2 * k + 1) % V]);
      const T r0 = (T)(e * c[k] - f * s[k]), r1 = (T)(e * s[k] + f * c[k]);
      if constexpr (!INTER) {
        ya.v[k] = r0;
        yb.v[k] = r1;
      } else {
        (2 * k < V ? ya.v[2 * k % V] : yb.v[2 * k % V]) = r0;
        (2 * k + 1 < V ? ya.v[(2 * k + 1) % V] : yb.v[(2 * k + 1) % V]) = r1;
      }
    }
    *reinterpret_cast<P*>(y + h * p.d + a0) = ya;
    *reinterpret_cast<P*>(y + h * p.d + b0) = yb;
  }
}

template <typename T, int V>
void launch(Rotary p, int interleaved, hipStream_t st) {
  p.nturn = p.rot / (2 * V);
  p.units = p.nturn + (p.x == p.y ? 0 : ((p.d - p.rot) / V + 1) / 2);
  // as many heads to a thread as leave 2^18 threads, four to a lane of the card
  const long all = p.rows * p.units * p.heads;
  p.hpt = (int)min((long)p.heads, max(1L, all >> 18));
  const dim3 grid((unsigned)((p.rows * p.units + 255) / 256), (unsigned)((p.heads + p.hpt - 1) / p.hpt));
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, V, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((rotary_kernel<T, V, false>), grid, dim3(256), 0, st, p);
}

// Packs of 16 bytes where every pack of a head starts on one, else single columns.
template <typename T>
void launch_type(const Rotary& p, int interleaved, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = p.rot % (2 * V) == 0 && p.off % V == 0 && p.d % V == 0 && p.ldx % V == 0 && p.ldy % V == 0 &&
                    (((uintptr_t)p.x | (uintptr_t)p.y) & 15) == 0;
  if (wide) launch<T, V>(p, interleaved, st);
  else launch<T, 1>(p, interleaved, st);
}

}  // namespace

extern "C" int dc_rotary(const void* x, long long ldx, void* y, long long ldy, int type, long long rows, int heads, int d, int off,
                         int rot, const double* freqs, const int* pos, int pos0, int t, float mag, int interleaved, int inverse,
                         void* stream) {
  if (!x || !y || !freqs || type < 0 || type > 2 || rows <= 0 || heads <= 0 || d <= 0) return DC_ERR_ARG;
  if (rot <= 0 || rot % 2 || off < 0 || off > d || rot > d - off || d > 65536 || heads > 65535) return DC_ERR_ARG;
  if ((long long)heads * d >= (1LL << 31) || (x == y && ldx != ldy)) return DC_ERR_ARG;
  if (ldx < (long long)heads * d || ldy < (long long)heads * d || (!pos && t <= 0) || rows > (1LL << 40) / d) return DC_ERR_ARG;
  const uintptr_t size = type == 2 ? 4 : 2;
  if ((((uintptr_t)x | (uintptr_t)y) & (size - 1)) || ((uintptr_t)freqs & 7) || ((uintptr_t)pos & 3)) return DC_ERR_ALIGN;
  if ((rows * d + 255) / 256 >= (1LL << 31)) return DC_ERR_ARG;
  Rotary p{x, y, (long)ldx, (long)ldy, (long)rows, heads, d, off, rot, freqs, pos, pos0, t, mag, inverse, 0, 0, 0};
  hipStream_t st = (hipStream_t)stream;
  if (type == 0) launch_type<bf16>(p, interleaved, st);
  else if (type == 1) launch_type<half>(p, interleaved, st);
  else launch_type<float>(p, interleaved, st);
  DC_CHECK_LAUNCH();
  return DC_OK;
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
