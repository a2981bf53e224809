// Activation checkpoints in 8 bits: what the backward pass needs of an activation, kept as e4m3 values with
// one power-of-two scale per 32 columns of a row (1 + 1/32 bytes per value instead of 2).
//
//   block of 32 columns, a = max |u|:   2^e = the smallest power of two with a / 2^e <= 448, -126 <= e <= 126
//   q = e4m3(u / 2^e), s = e + 127;     the checkpoint stands for  u^ = q 2^e
//
// The division by a power of two is exact and no value exceeds the largest e4m3 value, so the only
// error is e4m3's rounding: half a step, 2^-4 relative (2^-10 2^e absolute below 2^-6 2^e).  A block
// that holds an infinity or a NaN is kept as NaN throughout (s = 255), so that the gradient is
// non-finite where the activation was.
//
// bias + GELU:  y = gelu(u), u = x + b;  backward  du = dy gelu'(u^), db = column sums of du, and on
// request y^ = gelu(u^), the input of the following layer's weight gradient.  Everything is a
// stream over (T, D): bound by memory.  gelu is the tanh form, through sigmoid (v_exp, v_rcp);
// arithmetic and column sums are fp32.
//
// A thread takes 8 consecutive columns of a row (16-byte accesses of bf16, 8-byte of q) and four
// neighbours share a block's maximum by two lane exchanges.  The accesses are declared with their element's
// alignment, so rows of any length take them (global memory is read and written at any address).  The piece
// that a row ends in (ODD: rows that are no multiple of 8, kernels of their own: with this code in, 73728 x 2048
// bias + GELU took 328 us instead of 317) reads the row's last 8 columns and shifts its own down; it is stored by
// elements.  Rows of fewer than 8 columns are read by elements too.
#include "common.h"

namespace pv {
namespace ckpt8 {

constexpr int BLK = 32;
constexpr float kGeluK = 0.7978845608028654f, kGeluC = 0.044715f, kLog2e = 1.4426950408889634f;

// s = e + 127 of a block with largest magnitude a; 255 if a is not finite
__device__ __forceinline__ int scale_byte(float a) {
  const unsigned b = __float_as_uint(a);
  if (b >= 0x7F800000u) return 255;
  // a = 1.m 2^(E - 127): 448 = 1.75 2^8
  const int s = (int)(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return max(s, 1);
}
__device__ __forceinline__ float pow2(int s) { return __uint_as_float((unsigned)s << 23); }       // 2^(s - 127), 1 <= s <= 254
__device__ __forceinline__ float inv_pow2(int s) { return __uint_as_float((unsigned)(254 - s) << 23); }

// largest magnitude with NaN kept: the comparison of bit patterns orders |x| and puts NaN on top
__device__ __forceinline__ unsigned mag(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const unsigned short* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(unsigned short* p, float v) { *p = f32_to_bf16(v); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4_a4 a = reinterpret_cast<const f32x4_a4*>(p)[0], b = *reinterpret_cast<const f32x4_a4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
    const u32x4_a2 a = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(a[i] << 16);
      x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
  }
}
// columns c .. of a row of D, of which n count (n >= 8: all); what lies behind them is zero
template <bool ODD, typename T>
__device__ __forceinline__ void load_cols(const T* row, int c, int D, int n, float (&x)[8]) {
  if (!ODD) {
    load8(row + c, x);
  } else if (D < 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? load1(row + i) : 0.f;
  } else {
    const int by = max(0, 8 - n);
    load8(row + c - by, x);
#pragma unroll
    for (int s = 4; s; s >>= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = by & s ? (i + s < 8 ? x[i + s] : 0.f) : x[i];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&x)[8]) {
  if (n < 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) store1(p + i, x[i]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4_a4*>(p) = f32x4_a4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4_a4*>(p + 4) = f32x4_a4{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<u32x4_a2*>(p) =
        u32x4_a2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
  }
}
template <bool ODD>
__device__ __forceinline__ u32x2 load_bytes(const unsigned char* row, int c, int D, int n) {
  if (ODD && D < 8) {
    u32x2 w{0u, 0u};
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) w[i / 4] |= (unsigned)row[i] << (8 * (i % 4));
    return w;
  }
  const int by = ODD ? max(0, 8 - n) : 0;
  const u32x2_a1 v = *reinterpret_cast<const u32x2_a1*>(row + c - by);
  const unsigned long long w = (((unsigned long long)v[1] << 32) | v[0]) >> (8 * by);
  return u32x2{(unsigned)w, (unsigned)(w >> 32)};
}
__device__ __forceinline__ void store_bytes(unsigned char* p, int n, u32x2 w) {
  if (n >= 8) {
    *reinterpret_cast<u32x2_a1*>(p) = u32x2_a1{w[0], w[1]};
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = (unsigned char)(w[i / 4] >> (8 * (i % 4)));
  }
}

// 8 values / 2^(s-127) -> e4m3 bytes (round to nearest even)
__device__ __forceinline__ u32x2 quant8(const float (&x)[8], int s) {
  if (s == 255) return u32x2{0x7F7F7F7Fu, 0x7F7F7F7Fu};
  const float r = inv_pow2(s);
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * r, x[4 * i + 1] * r, 0, false);
    w[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * r, x[4 * i + 3] * r, v, true);
  }
  return w;
}
__device__ __forceinline__ float scale_of(int s) { return s == 255 ? __uint_as_float(0x7FC00000u) : pow2(s); }
__device__ __forceinline__ void dequant8(u32x2 w, int s, float (&x)[8]) {
  const float r = scale_of(s);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    x[4 * i] = a[0] * r;
    x[4 * i + 1] = a[1] * r;
    x[4 * i + 2] = b[0] * r;
    x[4 * i + 3] = b[1] * r;
  }
}

// sigmoid(2 k (x + c x^3)): gelu = x sg, gelu' = sg + x sg (1 - sg) (2 k + 6 k c x^2)
__device__ __forceinline__ float sig(float x) {
  const float e = __builtin_amdgcn_exp2f(x * fmaf(x * x, -2.f * kGeluK * kGeluC * kLog2e, -2.f * kGeluK * kLog2e));
  return __builtin_amdgcn_rcpf(1.f + e);
}
// behind |x| = 16 sg (1 - sg) is exactly 0 in fp32; the clamp keeps its factor finite
__device__ __forceinline__ float slope(float x, float sg) {
  const float c = __builtin_amdgcn_fmed3f(x, -16.f, 16.f);
  const float q = c * fmaf(c * c, 6.f * kGeluK * kGeluC, 2.f * kGeluK);
  return fmaf(q, fmaf(-sg, sg, sg), sg);
}

// How a workgroup of 256 threads covers (T, D): `tpr` threads (a multiple of 4) per row, 256 / tpr rows per
// pass, rows r0 .. r1; D behind 2048 columns in further workgroups (grid.y).
struct Shape {
  long T;
  int D, nb;     // nb = blocks per row
  int tpr, rpb;  // rpb = rows per workgroup
};
struct Place {
  int c, n, sub, step;  // n = columns from c to the row's end
  long r0, r1;
  bool on;
};
template <bool ODD>
__device__ __forceinline__ Place place(const Shape& s) {
  Place p;
  p.sub = threadIdx.x / s.tpr;
  p.c = blockIdx.y * 2048 + (threadIdx.x - p.sub * s.tpr) * 8;
  p.n = ODD ? s.D - p.c : 8;
  p.step = 256 / s.tpr;
  p.r0 = (long)blockIdx.x * s.rpb + p.sub;
  p.r1 = min(s.T, (long)(blockIdx.x + 1) * s.rpb);
  p.on = p.sub < p.step && p.c < s.D;
  return p;
}
// Bound by memory: 256000 x 768 bf16 in 134 us (4.4 TB/s), with bias and GELU 73728 x 2048 in 148 (5.1 TB/s); a
// column per lane instead of 8 took 348 against 114 us at 73728 x 2047.  Slabs of columns that leave fewer threads
// idle than whole rows do (64 of 256 are, at 768) were no faster: 202 -> 218 us with GELU.
// MODE 0: pack x;  1: u = x + b, y = gelu(u), pack u.  U rows in flight per thread.
template <typename T, int MODE, int U, bool ODD>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ x, const float* __restrict__ b,
                                                   T* __restrict__ y, unsigned char* __restrict__ q,
                                                   unsigned char* __restrict__ sc, Shape s) {
  const Place p = place<ODD>(s);
  float bias[8];
  if constexpr (MODE == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bias[i] = p.on && i < p.n ? b[p.c + i] : 0.f;
  }
  for (long r = p.r0; r < p.r1; r += U * p.step) {  // lanes that share a block leave together: same sub
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long rr = min(r + u * p.step, p.r1 - 1);
      if (p.on) load_cols<ODD>(x + rr * s.D, p.c, s.D, p.n, v[u]);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long rr = r + u * p.step;
      if (rr >= p.r1) break;
      unsigned m = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (MODE == 1) v[u][i] += bias[i];  // zero behind the row
        m = max(m, mag(v[u][i]));
      }
      m = max(m, (unsigned)__shfl_xor((int)m, 1, 64));
      m = max(m, (unsigned)__shfl_xor((int)m, 2, 64));
      if (!p.on) continue;
      const int e = scale_byte(__uint_as_float(m));
      store_bytes(q + rr * s.D + p.c, p.n, quant8(v[u], e));
      if ((p.c & 31) == 0) sc[rr * s.nb + p.c / BLK] = (unsigned char)e;
      if constexpr (MODE == 1) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = v[u][i] * sig(v[u][i]);
        store8(y + rr * s.D + p.c, p.n, o);
      }
    }
  }
}

// y = gelu(x + b) where nothing is kept, in pack_kernel's arithmetic.  A workgroup takes a slab of 1024 columns of `rows`
// rows, slabs of a row in neighbouring workgroups.  Bound by memory: 73728 x 2048 in 117 us (5.2 TB/s), 256000 x 768 in 152;
// as a form of pack_kernel that stores no checkpoint 124 and 158.
template <bool ODD>
__global__ __launch_bounds__(128) void gelu_kernel(const unsigned short* __restrict__ x, const float* __restrict__ b,
                                                   unsigned short* __restrict__ y, long T, int D, int slabs, int rows) {
  const int c = (int)(blockIdx.x % slabs) * 1024 + threadIdx.x * 8, n = ODD ? D - c : 8;
  if (c >= D) return;
  float bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bias[i] = i < n ? b[c + i] : 0.f;
  const long r0 = (long)(blockIdx.x / slabs) * rows, r1 = min(T, r0 + rows);
  for (long r = r0; r < r1; ++r) {
    float v[8];
    load_cols<ODD>(x + r * D, c, D, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] += bias[i];
      v[i] *= sig(v[i]);
    }
    store8(y + r * D + c, n, v);
  }
}

// 256000 x 768 into bf16: 104 us (5.7 TB/s)
template <typename T, int U, bool ODD>
__global__ __launch_bounds__(256) void unpack_kernel(const unsigned char* __restrict__ q,
                                                     const unsigned char* __restrict__ sc, T* __restrict__ x, Shape s) {
  const Place p = place<ODD>(s);
  if (!p.on) return;
  for (long r = p.r0; r < p.r1; r += U * p.step) {
    u32x2 w[U];
    int e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long rr = min(r + u * p.step, p.r1 - 1);
      w[u] = load_bytes<ODD>(q + rr * s.D, p.c, s.D, p.n);
      e[u] = sc[rr * s.nb + p.c / BLK];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long rr = r + u * p.step;
      if (rr >= p.r1) break;
      float v[8];
      dequant8(w[u], e[u], v);
      store8(x + rr * s.D + p.c, p.n, v);
    }
  }
}

// Bound by memory: 73728 x 2048 in 167 us (4.5 TB/s), column sums in the same pass, 5 us for their partial rows.
// du = dy gelu'(u^) -> dx, column partials of this workgroup's rows -> part[blockIdx.x][D]; Y: y^ = gelu(u^) too
template <int U, bool Y, bool ODD>
__global__ __launch_bounds__(256) void gelu_bwd_kernel(const unsigned char* __restrict__ q,
                                                       const unsigned char* __restrict__ sc,
                                                       const unsigned short* __restrict__ dy,
                                                       unsigned short* __restrict__ dx,
                                                       unsigned short* __restrict__ yh, float* __restrict__ part,
                                                       Shape s) {
  __shared__ __attribute__((aligned(16))) float sh[256 * 8];
  const Place p = place<ODD>(s);
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  if (p.on)
    for (long r = p.r0; r < p.r1; r += U * p.step) {
      u32x2 w[U];
      float gv[U][8];
      int e[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long rr = min(r + u * p.step, p.r1 - 1);
        w[u] = load_bytes<ODD>(q + rr * s.D, p.c, s.D, p.n);
        load_cols<ODD>(dy + rr * s.D, p.c, s.D, p.n, gv[u]);
        e[u] = sc[rr * s.nb + p.c / BLK];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long rr = r + u * p.step;
        if (rr >= p.r1) break;
        float v[8], d[8], o[8];
        dequant8(w[u], e[u], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float sg = sig(v[i]);
          d[i] = gv[u][i] * slope(v[i], sg);
          acc[i] += d[i];
          o[i] = v[i] * sg;
        }
        store8(dx + rr * s.D + p.c, p.n, d);
        if constexpr (Y) store8(yh + rr * s.D + p.c, p.n, o);
      }
    }
  // rows of the workgroup's passes: sub 0 adds the others in order
#pragma unroll
  for (int i = 0; i < 8; ++i) sh[threadIdx.x * 8 + i] = acc[i];
  __syncthreads();
  if (p.sub == 0 && p.on) {
    for (int k = 1; k < p.step; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += sh[(k * s.tpr + threadIdx.x) * 8 + i];
    store8(part + (size_t)blockIdx.x * s.D + p.c, p.n, acc);
  }
}

// out[c] (+)= sum of the S partial rows, in row order within each of the 16 row lanes, then over the lanes
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float* __restrict__ part, float* __restrict__ out, int S,
                                                         int D, int add) {
  __shared__ float sh[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  float a = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int r = w; r < S; r += 16) a += part[(size_t)r * D + c];
  }
  sh[w][threadIdx.x & 63] = a;
  __syncthreads();
  if (w == 0 && c < D) {
#pragma unroll
    for (int k = 1; k < 16; ++k) a += sh[k][threadIdx.x];
    out[c] = add ? out[c] + a : a;
  }
}

__host__ inline Shape shape(long T, int D, long want) {
  Shape s{};
  s.T = T;
  s.D = D;
  s.nb = (D + BLK - 1) / BLK;
  s.tpr = min(256, s.nb * 4);
  const int pass = 256 / s.tpr;
  // `want` workgroups, each a whole number of passes
  const long rows = (T + want - 1) / want;
  s.rpb = (int)((rows + pass - 1) / pass * pass);
  return s;
}
// workgroups over the rows of a stream without column sums: many, so that the last ones end together
__host__ inline long many(long T, int D) {
  const int pass = 256 / min(256, (D + BLK - 1) / BLK * 4);
  return max(1L, min(8192L, (T + 4 * pass - 1) / (4 * pass)));
}
// row groups of the GELU backward, each of which leaves one partial row of column sums
__host__ inline long groups(long T) { return T <= 128 ? 1 : min(1024L, T / 16); }

__host__ inline int sizes(long T, long D) {
  if (T < 0 || D <= 0) return -1;
  return (T > 0x7FFFFFFFL || D > (1L << 24)) ? -2 : 0;
}
__host__ inline int cols(int D) { return (D + 2047) / 2048; }

template <typename T, int MODE>
int pack(const T* x, const float* b, T* y, unsigned char* q, unsigned char* sc, long rows, int D, hipStream_t st) {
  if (rows == 0) return 0;
  const Shape s = shape(rows, D, many(rows, D));
  const dim3 grid((unsigned)((rows + s.rpb - 1) / s.rpb), cols(D));
  if (D % 8) hipLaunchKernelGGL((pack_kernel<T, MODE, 4, true>), grid, dim3(256), 0, st, x, b, y, q, sc, s);
  else hipLaunchKernelGGL((pack_kernel<T, MODE, 4, false>), grid, dim3(256), 0, st, x, b, y, q, sc, s);
  PV_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int unpack(const unsigned char* q, const unsigned char* sc, T* x, long rows, int D, hipStream_t st) {
  if (rows == 0) return 0;
  const Shape s = shape(rows, D, many(rows, D));
  const dim3 grid((unsigned)((rows + s.rpb - 1) / s.rpb), cols(D));
  if (D % 8) hipLaunchKernelGGL((unpack_kernel<T, 4, true>), grid, dim3(256), 0, st, q, sc, x, s);
  else hipLaunchKernelGGL((unpack_kernel<T, 4, false>), grid, dim3(256), 0, st, q, sc, x, s);
  PV_LAUNCH_CHECK();
  return 0;
}

}  // namespace ckpt8
}  // namespace pv

using namespace pv;
using namespace pv::ckpt8;

// x (T, D) bf16 (x16 = 1) or fp32 -> q (T, D) e4m3 bytes, s (T, ceil(D / 32)) exponent bytes
PV_API int pv_ckpt8_pack(const void* x, int x16, void* q, void* s, long T, int D, void* stream) {
  if (const int rc = sizes(T, D)) return rc;
  hipStream_t st = (hipStream_t)stream;
  unsigned char *qq = (unsigned char*)q, *ss = (unsigned char*)s;
  return x16 ? pack<unsigned short, 0>((const unsigned short*)x, nullptr, nullptr, qq, ss, T, D, st)
             : pack<float, 0>((const float*)x, nullptr, nullptr, qq, ss, T, D, st);
}

PV_API int pv_ckpt8_unpack(const void* q, const void* s, void* x, int x16, long T, int D, void* stream) {
  if (const int rc = sizes(T, D)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const unsigned char *qq = (const unsigned char*)q, *ss = (const unsigned char*)s;
  return x16 ? unpack(qq, ss, (unsigned short*)x, T, D, st) : unpack(qq, ss, (float*)x, T, D, st);
}

// x (T, D) bf16, b (D) fp32 -> y = gelu(x + b) bf16 and the checkpoint of x + b (q and s both null: y alone)
PV_API int pv_ckpt8_gelu_fwd(const void* x, const float* b, void* y, void* q, void* s, long T, int D, void* stream) {
  if (const int rc = sizes(T, D)) return rc;
  if (!q != !s) return -3;
  hipStream_t st = (hipStream_t)stream;
  if (q) return pack<unsigned short, 1>((const unsigned short*)x, b, (unsigned short*)y, (unsigned char*)q, (unsigned char*)s, T, D, st);
  if (T == 0) return 0;
  // 16 rows per workgroup; more where there are so many that the grid would pass 2^32 threads
  const int slabs = (D + 1023) / 1024, rows = (int)max(16L, (T * slabs + (1L << 24) - 1) >> 24);
  const dim3 grid((unsigned)((T + rows - 1) / rows * slabs));
  if (D % 8) hipLaunchKernelGGL((gelu_kernel<true>), grid, dim3(128), 0, st, (const unsigned short*)x, b, (unsigned short*)y, T, D, slabs, rows);
  else hipLaunchKernelGGL((gelu_kernel<false>), grid, dim3(128), 0, st, (const unsigned short*)x, b, (unsigned short*)y, T, D, slabs, rows);
  PV_LAUNCH_CHECK();
  return 0;
}

// floats of workspace of pv_ckpt8_gelu_bwd
PV_API long pv_ckpt8_gelu_bwd_ws(long T, int D) { return groups(T) * D; }

// dy (T, D) bf16 and the checkpoint of u -> dx = dy gelu'(u^) bf16; db (D) fp32 (+)= column sums (db_add); yh
// (optional) = gelu(u^) bf16
PV_API int pv_ckpt8_gelu_bwd(const void* q, const void* s, const void* dy, void* dx, void* yh, float* db, int db_add,
                             float* ws, long T, int D, void* stream) {
  if (const int rc = sizes(T, D)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const unsigned char *qq = (const unsigned char*)q, *ss = (const unsigned char*)s;
  const unsigned short* g = (const unsigned short*)dy;
  unsigned short *d = (unsigned short*)dx, *y = (unsigned short*)yh;
  const Shape p = shape(T, D, groups(T));
  const int S = T ? (int)((T + p.rpb - 1) / p.rpb) : 0;
  float* part = S == 1 && !db_add ? db : ws;  // one row group: its sums are the result
  if (S) {
    const dim3 grid(S, cols(D));
    const auto kernel = D % 8 ? (y ? gelu_bwd_kernel<4, true, true> : gelu_bwd_kernel<4, false, true>)
                              : (y ? gelu_bwd_kernel<4, true, false> : gelu_bwd_kernel<4, false, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, qq, ss, g, d, y, part, p);
    PV_LAUNCH_CHECK();
  }
  if (part != db) {
    hipLaunchKernelGGL(sum_parts_kernel, dim3((D + 63) / 64), dim3(1024), 0, st, (const float*)ws, db, S, D, db_add);
    PV_LAUNCH_CHECK();
  }
  return 0;
}
