// Token-embedding lookup with scaling, and its table gradient summed over the sorted tokens.
//
//   out[t] = scale W[id[t]]  (+ pos[l(t)] + typ: the transformer's front end)
//   dW[v]  = scale sum of g[t] over the tokens t with id[t] = v, v != pad
//
// The lookup moves T rows out and reads T rows of a table that the caches mostly hold; the
// gradient reads T rows and writes V: both are bound by memory.
//
// Gradient.  Float atomics would make the sums depend on arrival order and serialise on frequent
// ids (a word of a Zipf text is several percent of all tokens).  Here every row has one writer:
//   * few tokens (T <= SMALL_T): one launch.  A workgroup per token; the first token of an id adds
//     all rows of that id, found by comparing ids; other workgroups zero the rows without a token.
//   * else the tokens are sorted by id (two launches per 8 bits, which zero the gradient on the way; stable), a wave
//     adds the rows of CHUNK consecutive sorted tokens, writing the runs that lie inside its chunk, and the runs that
//     cross a chunk's border are joined from the chunks' fp32 partial rows by a second launch.
// All sums are fp32, in an order that depends on the sizes and ids alone.
#include "common.h"

namespace pv {
namespace temb {

// Up to here one launch, which compares every token with all others: at 4096 tokens 18 / 23 / 48 / 42 us where sorting
// takes 31 / 31 / 43 / 50 (tables of 5000 x 64, 1024 x 300, 30522 x 768, 60000 x 512, Zipf ids), at 8192 30 / 45 / 94 / 75
// against 33 / 32 / 48 / 53; the sort's five further launches cost another 15 us of host time.  The worst ids, all
// the same: 173 against 29 us at 4096 tokens (a padded batch whose padding is not excluded comes near).
constexpr int SMALL_T = 4096;
constexpr int CHUNK = 32;  // sorted tokens per wave
constexpr long MAX_T = 0x7FFFFFFFL - 4 * CHUNK;  // token numbers in 31 bits, and a grid of fewer than 2^32 threads for them
constexpr int ZROWS = 64;  // table rows per zeroing workgroup of the small path

struct Groups {
  int off[4], L[4], n;
};

struct Ids {
  const void* p;
  int is64;
  __device__ __forceinline__ long at(long t) const {
    return is64 ? reinterpret_cast<const long*>(p)[t] : (long)reinterpret_cast<const int*>(p)[t];
  }
  // the table row whose gradient token t adds to; V (none) for the padding id and ids out of range
  __device__ __forceinline__ unsigned key(long t, long V, long pad) const {
    const long i = at(t);
    return (i < 0 || i >= V || i == pad) ? (unsigned)V : (unsigned)i;
  }
};

template <typename T>
__device__ __forceinline__ float load1(const T* p);
template <>
__device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load1<unsigned short>(const unsigned short* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(unsigned short* p, float v) { *p = f32_to_bf16(v); }

// Vectors of the element's alignment: global memory is read and written at any address, rows of any length take them
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const f32x4_a4 a = *reinterpret_cast<const f32x4_a4*>(p), b = *reinterpret_cast<const f32x4_a4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}
__device__ __forceinline__ void load8(const unsigned short* p, float (&x)[8]) {
  const u32x4_a2 a = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(a[i] << 16), x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<f32x4_a4*>(p) = f32x4_a4{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f32x4_a4*>(p + 4) = f32x4_a4{x[4], x[5], x[6], x[7]};
}
__device__ __forceinline__ void store8(unsigned short* p, const float (&x)[8]) {
  *reinterpret_cast<u32x4_a2*>(p) =
      u32x4_a2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}

// ------------------------------------------------------------------------------------ lookup
// A workgroup owns `rows` consecutive tokens; a thread takes pieces of C columns of them, four at a time so that
// four rows are on their way at once.  C = 8: a row's last piece is its last 8 columns, which two threads may write
// alike; C = 1: rows of fewer columns (a column per thread took 106 us instead of 37 at 73728 x 767).
// 73728 tokens x 768 fp32 -> bf16: 42 us (2.7 TB/s written, 5.4 read, the table from the
// caches); 256000 x 512: 82 us.
template <typename TW, typename TO, int C>
__global__ __launch_bounds__(256) void lookup_kernel(Ids ids, const TW* __restrict__ W, TO* __restrict__ out, long T,
                                                     long V, int E, float scale, int rows,
                                                     const float* __restrict__ pos, const float* __restrict__ typ,
                                                     Groups gr) {
  const long t0 = (long)blockIdx.x * rows;
  const int n = (int)min((long)rows, T - t0), per = (E + C - 1) / C, all = n * per;
  for (int x0 = threadIdx.x; x0 < all; x0 += 1024) {
    int r[4], c[4];
    long id[4];
    float v[4][C];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int x = min(x0 + 256 * u, all - 1);
      r[u] = x / per;
      c[u] = min((x - r[u] * per) * C, E - C);
      id[u] = ids.at(t0 + r[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const TW* w = W + (id[u] >= 0 && id[u] < V ? id[u] : 0) * E + c[u];
      if constexpr (C == 8) load8(w, v[u]);
      else v[u][0] = load1(w);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (x0 + 256 * u >= all) break;
      const long t = t0 + r[u];
      const bool ok = id[u] >= 0 && id[u] < V;
#pragma unroll
      for (int i = 0; i < C; ++i) v[u][i] = ok ? v[u][i] * scale : __uint_as_float(0x7FC00000u);
      if (pos) {
        int g = 0;
        while (g + 1 < gr.n && t >= gr.off[g + 1]) ++g;
        const float* pp = pos + (size_t)((t - gr.off[g]) % gr.L[g]) * E + c[u];
#pragma unroll
        for (int i = 0; i < C; ++i) v[u][i] = (v[u][i] + pp[i]) + typ[c[u] + i];
      }
      if constexpr (C == 8) store8(out + t * E + c[u], v[u]);
      else store1(out + t * E + c[u], v[u][0]);
    }
  }
}

// ------------------------------------------------------------------------------------ gradient
// A lane owns W consecutive columns (4, or 1 of rows with fewer than 4) of a slab of 64 W columns (grid.y).
// One slab per wave: a wave over a whole row of 768 has a third of the waves and as many loads under way
// (walk_kernel 87 us instead of 44 at 73728 tokens x 768).
// Where a row is no multiple of 4, the lane that it ends in takes the row's last 4 columns: those that it shares with its
// neighbour come out the same in both, and both write them, but where the row is added to (a column per lane: 126 us
// instead of 70 for the gradient of 73728 tokens x 767).
template <typename TG, int W>
struct Cols {
  float a[W];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) a[i] = 0.f;
  }
  __device__ __forceinline__ static int col() { return (blockIdx.y * 64 + (threadIdx.x & 63)) * W; }
  __device__ __forceinline__ void load(const TG* row, int E) {
    const int c = col();
    if (c >= E) {
      zero();
    } else if constexpr (W == 1) {
      a[0] = load1(row + c);
    } else if constexpr (sizeof(TG) == 4) {
      const f32x4_a4 v = *reinterpret_cast<const f32x4_a4*>(row + min(c, E - 4));
#pragma unroll
      for (int i = 0; i < W; ++i) a[i] = v[i];
    } else {
      const u32x2_a2 v = *reinterpret_cast<const u32x2_a2*>(row + min(c, E - 4));
      a[0] = __uint_as_float(v[0] << 16);
      a[1] = __uint_as_float(v[0] & 0xFFFF0000u);
      a[2] = __uint_as_float(v[1] << 16);
      a[3] = __uint_as_float(v[1] & 0xFFFF0000u);
    }
  }
  template <typename O>
  __device__ __forceinline__ void add(const O& x) {
#pragma unroll
    for (int i = 0; i < W; ++i) a[i] += x.a[i];
  }
  // dst row = (acc ? dst row : 0) + scale * this
  __device__ __forceinline__ void store(float* row, int E, float scale, bool acc) const {
    const int c = col();
    if (c >= E) return;
    if constexpr (W == 1) {
      row[c] = (acc ? row[c] : 0.f) + a[0] * scale;
    } else {
      const int at = min(c, E - 4);
      if (acc && at < c) {
#pragma unroll
        for (int i = 1; i < W; ++i)
          if (at + i >= c) row[at + i] += a[i] * scale;
        return;
      }
      f32x4_a4 v{0.f, 0.f, 0.f, 0.f};
      if (acc) v = *reinterpret_cast<const f32x4_a4*>(row + at);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] += a[i] * scale;
      *reinterpret_cast<f32x4_a4*>(row + at) = v;
    }
  }
};

__device__ __forceinline__ unsigned uniform(unsigned x) { return __builtin_amdgcn_readfirstlane(x); }

// Sum over the N + 1 waves of a workgroup in wave order, into wave 0's x
template <typename X, int W, int N>
__device__ __forceinline__ void join_waves(X& x, float (&sh)[N][W][64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave)
#pragma unroll
    for (int i = 0; i < W; ++i) sh[wave - 1][i][lane] = x.a[i];
  __syncthreads();
  if (wave == 0)
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int w = 0; w < N; ++w) x.a[i] += sh[w][i][lane];
}

// Few tokens.  Workgroup b < T: token b, which writes its id's row if it is the id's first token
// (every wave adds the rows of one quarter of the tokens).  Workgroups behind: zeros for the rows
// without a token.
template <typename TG, int W>
__global__ __launch_bounds__(256) void small_grad_kernel(Ids ids, const TG* __restrict__ g, float* __restrict__ dW,
                                                         int T, long V, int E, long pad, float scale, int acc) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x < T) {
    __shared__ float sh[3][W][64];
    const int t = blockIdx.x;
    const unsigned v = ids.key(t, V, pad);
    if (v == (unsigned)V) return;
    int before = 0;
    for (int u = threadIdx.x; u < t; u += 256) before |= ids.key(u, V, pad) == v;
    if (__syncthreads_or(before)) return;
    const int q = (T - t + 3) / 4, u0 = t + wave * q, u1 = min(T, u0 + q);
    Cols<TG, W> sum;
    sum.zero();
    for (int u = u0; u < u1; u += 64) {
      unsigned long long hit = __ballot(u + lane < u1 && ids.key(min(u + lane, T - 1), V, pad) == v);
      while (hit) {  // four rows on their way at once, added in token order
        Cols<TG, W> row[4];
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = hit ? __builtin_ctzll(hit) : 0;
          n += hit != 0ull;
          row[i].load(g + (size_t)(u + k) * E, E);
          hit &= hit - 1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) sum.add(row[i]);
      }
    }
    join_waves<Cols<TG, W>, W, 3>(sum, sh);
    if (wave == 0) sum.store(dW + (size_t)v * E, E, scale, acc);
    return;
  }
  __shared__ int has[ZROWS];
  if (blockIdx.y) return;  // the zeroing workgroups take whole rows
  for (long r0 = (long)(blockIdx.x - T) * ZROWS; r0 < V; r0 += (long)(gridDim.x - T) * ZROWS) {
    __syncthreads();
    if (threadIdx.x < ZROWS) has[threadIdx.x] = 0;
    __syncthreads();
    for (int u = threadIdx.x; u < T; u += 256) {
      const long k = (long)ids.key(u, V, pad) - r0;
      if (k >= 0 && k < ZROWS) has[k] = 1;
    }
    __syncthreads();
    const int n = (int)min((long)ZROWS, V - r0);
    for (int r = wave; r < n; r += 4) {
      if (has[r]) continue;
      float* row = dW + (r0 + r) * E;
      const int whole = W == 4 ? E / 4 * 4 : 0;
      for (int c = lane * 4; c < whole; c += 256) *reinterpret_cast<f32x4_a4*>(row + c) = f32x4_a4{0.f, 0.f, 0.f, 0.f};
      for (int c = whole + lane; c < E; c += 64) row[c] = 0.f;
    }
  }
}

// ---- sort by id: 8 bits at a time, least significant first, stable
// The tokens lie in at most PARTS parts of whole tiles, one per workgroup.  count_kernel: how many tokens of each
// part have which digit.  place_kernel: every workgroup adds up that table for itself (a part's digit starts
// behind the smaller digits of all parts and its own digit in the parts before; no launch for the sums) and moves its tokens.
// Few workgroups and short ones, bound by latency; the zeroing of the gradient is spread over these launches as further
// workgroups, whose writes run meanwhile.  At 73728 tokens, 30522 rows of 768: 30 us, where a launch that zeroes
// and the general sort's six launches took 46.
constexpr int TILE = 1024;   // threads of a workgroup, a token each
constexpr int PARTS = 128;
constexpr int ZFILL = 512;   // zeroing workgroups per launch, at most

template <typename KT>
struct Tokens {  // keys and token numbers; from the ids themselves if keys is null
  Ids ids;
  long V, pad;
  const KT* keys;
  const unsigned* slot;
  __device__ __forceinline__ unsigned key(long t) const { return keys ? (unsigned)keys[t] : ids.key(t, V, pad); }
};

struct Fill {  // n floats at p, this launch's share of the gradient
  float* p;
  long n;
  __device__ __forceinline__ void run(int wg, int wgs) const {
    const long i0 = (long)wg * TILE + threadIdx.x, step = (long)wgs * TILE;
    const long n4 = (reinterpret_cast<size_t>(p) & 15) == 0 ? n / 4 : 0;
    for (long i = i0; i < n4; i += step) reinterpret_cast<f32x4*>(p)[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (long i = n4 * 4 + i0; i < n; i += step) p[i] = 0.f;
  }
};

// the wave's lanes that hold a token of the same digit as this one
__device__ __forceinline__ unsigned long long same_digit(unsigned digit, bool here) {
  unsigned long long m = __ballot(here);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const unsigned long long one = __ballot((digit >> b) & 1u);
    m &= (digit >> b) & 1u ? one : ~one;
  }
  return m;
}

template <typename KT>
__global__ __launch_bounds__(TILE) void count_kernel(Tokens<KT> src, long T, long part, int parts, int shift,
                                                     unsigned* __restrict__ table, Fill fill) {
  if ((int)blockIdx.x >= parts) return fill.run((int)blockIdx.x - parts, (int)gridDim.x - parts);
  __shared__ unsigned n[256];
  if (threadIdx.x < 256) n[threadIdx.x] = 0;
  __syncthreads();
  const long b = (long)blockIdx.x * part, e = min(T, b + part);
  for (long t0 = b; t0 < e; t0 += TILE) {
    const long t = t0 + threadIdx.x;
    const bool here = t < e;
    const unsigned digit = here ? (src.key(t) >> shift) & 255u : 0u;
    const unsigned long long m = same_digit(digit, here);
    if (here && (threadIdx.x & 63) == (unsigned)__builtin_ctzll(m)) atomicAdd(&n[digit], (unsigned)__popcll(m));
  }
  __syncthreads();
  if (threadIdx.x < 256) table[(size_t)blockIdx.x * 256 + threadIdx.x] = n[threadIdx.x];
}

template <typename KT>
__global__ __launch_bounds__(TILE) void place_kernel(Tokens<KT> src, long T, long part, int parts, int shift,
                                                     const unsigned* __restrict__ table, KT* __restrict__ keys,
                                                     unsigned* __restrict__ slot, Fill fill) {
  if ((int)blockIdx.x >= parts) return fill.run((int)blockIdx.x - parts, (int)gridDim.x - parts);
  __shared__ unsigned base[256], before[4][256], all[4][256], waves[4];
  __shared__ unsigned short in[TILE / 64][256];  // tokens of the tile per wave and digit, then those of the waves before
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = threadIdx.x & 255, quarter = threadIdx.x >> 8;
  {
    unsigned x = 0, y = 0;
#pragma unroll 8
    for (int p = quarter; p < parts; p += 4) {
      const unsigned n = table[(size_t)p * 256 + d];
      y += n;
      x += p < (int)blockIdx.x ? n : 0u;
    }
    before[quarter][d] = x;
    all[quarter][d] = y;
  }
  __syncthreads();
  unsigned sum = 0, own = 0;
  if (quarter == 0) {  // running sum over the digits: within each of four waves, then over them
    own = all[0][d] + all[1][d] + all[2][d] + all[3][d];
    sum = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned v = __shfl_up(sum, o);
      sum += lane >= o ? v : 0u;
    }
    if (lane == 63) waves[wave] = sum;
  }
  __syncthreads();
  if (quarter == 0) {
    sum -= own;
    for (int w = 0; w < wave; ++w) sum += waves[w];
    base[d] = sum + before[0][d] + before[1][d] + before[2][d] + before[3][d];
  }
  const long b = (long)blockIdx.x * part, e = min(T, b + part);
  for (long t0 = b; t0 < e; t0 += TILE) {
    const long t = t0 + threadIdx.x;
    const bool here = t < e;
    const unsigned key = here ? src.key(t) : 0u, tok = here ? (src.keys ? src.slot[t] : (unsigned)t) : 0u;
    const unsigned digit = (key >> shift) & 255u;
#pragma unroll
    for (int u = 0; u < TILE / 64 / 4; ++u) in[4 * u + quarter][d] = 0;
    __syncthreads();
    const unsigned long long m = same_digit(digit, here);
    const int rank = __popcll(m & ((1ull << lane) - 1ull));
    if (here && rank == 0) in[wave][digit] = (unsigned short)__popcll(m);
    __syncthreads();
    unsigned n = 0;
    if (quarter == 0)
#pragma unroll
      for (int w = 0; w < TILE / 64; ++w) {
        const unsigned x = in[w][d];
        in[w][d] = (unsigned short)n;
        n += x;
      }
    __syncthreads();
    if (here) {
      const unsigned to = base[digit] + in[wave][digit] + (unsigned)rank;
      keys[to] = (KT)key;
      slot[to] = tok;
    }
    __syncthreads();
    if (quarter == 0) base[d] += n;
  }
}

// A wave adds the rows of its chunk of the sorted tokens, run by run (bound by the rows' reads, 512 bytes each at
// their tokens' places: 42 us at 73728 tokens x 768, 84 at 256000 x 512; chunks of 16 tokens 137 and 251 us instead of 125
// and 217 for the whole, of 64 tokens 149 and 221).  Partial rows: slot 2 c = the
// part of a run that began before chunk c, slot 2 c + 1 = the part of a run that begins in chunk c
// and goes on behind it.
template <typename TG, typename KT, int W>
__global__ __launch_bounds__(256) void walk_kernel(const KT* __restrict__ keys, const unsigned* __restrict__ slot,
                                                   const TG* __restrict__ g, float* __restrict__ part,
                                                   float* __restrict__ dW, long T, long V, int E, float scale,
                                                   int acc) {
  const int lane = threadIdx.x & 63;
  const long c = (long)blockIdx.x * 4 + (threadIdx.x >> 6), b = c * CHUNK, e = min(T, b + CHUNK);
  if (b >= T) return;
  const unsigned none = (unsigned)V;
  unsigned mykey = none, mypos = 0;
  if (lane < CHUNK && b + lane < e) {
    mykey = keys[b + lane];
    mypos = slot[b + lane];
  }
  unsigned cur = uniform(mykey);
  if (cur == none) return;  // padding sorts last
  const bool from_before = b > 0 && keys[b - 1] == (KT)cur;
  const unsigned behind = e < T ? (unsigned)keys[e] : none;
  bool first = true;
  Cols<TG, W> sum;
  sum.zero();
  auto flush = [&](unsigned key, bool goes_on) {
    if (first && from_before) sum.store(part + (2 * c) * E, E, 1.f, false);
    else if (goes_on) sum.store(part + (2 * c + 1) * E, E, 1.f, false);
    else sum.store(dW + (size_t)key * E, E, scale, acc);
    first = false;
    sum.zero();
  };
  const int n = (int)(e - b);
  constexpr int U = 8;  // rows on their way at once (16: 103 instead of 83 us at 256000 tokens x 512)
  for (int k0 = 0; k0 < n; k0 += U) {
    Cols<TG, W> row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned p = __builtin_amdgcn_readlane(mypos, min(k0 + u, n - 1));
      row[u].load(g + (size_t)p * E, E);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u >= n) break;
      const unsigned k = __builtin_amdgcn_readlane(mykey, k0 + u);
      if (k != cur) {
        flush(cur, false);
        cur = k;
      }
      if (cur == none) return;
      sum.add(row[u]);
    }
  }
  flush(cur, behind == cur);
}

// Where a run begins in chunk c and goes on behind it: the sum of its partial rows.  A wave per chunk; runs over
// many chunks (frequent ids) are added by the workgroup's four waves together, a quarter each (sixteen waves: 30 us
// instead of 20 at 256000 tokens x 512).
constexpr int ALONE = 16;  // partial rows that a wave adds by itself
constexpr int JOIN = 4;   // waves per workgroup
template <typename TG, typename KT, int W>
__global__ __launch_bounds__(64 * JOIN) void join_kernel(const KT* __restrict__ keys, const float* __restrict__ part,
                                                   float* __restrict__ dW, long T, long V, int E, float scale,
                                                   int acc) {
  __shared__ float sh[JOIN - 1][W][64];
  __shared__ long many[JOIN];
  const int wave = threadIdx.x >> 6;
  auto total = [&](long c, long x0, long x1) {  // partial rows x0 .. of the run that begins in chunk c
    Cols<float, W> sum, row;
    sum.zero();
#pragma unroll 8
    for (long x = x0; x < x1; ++x) {
      row.load(part + (x == 0 ? 2 * c + 1 : 2 * (c + x)) * E, E);
      sum.add(row);
    }
    return sum;
  };
  {
    const long c = (long)blockIdx.x * JOIN + wave, b = c * CHUNK, e = b + CHUNK;
    long m = 0;
    if (e < T) {
      const KT key = keys[e - 1];
      if ((unsigned)key != (unsigned)V && keys[e] == key && !(keys[b] == key && b > 0 && keys[b - 1] == key)) {
        long lo = e, hi = T;  // first position behind the run
        while (lo < hi) {
          const long mid = (lo + hi) >> 1;
          if (keys[mid] == key) lo = mid + 1;
          else hi = mid;
        }
        m = (lo - 1) / CHUNK - c + 1;  // slot 2c+1, then 2(c+1), 2(c+2), ..
        if (m <= ALONE) total(c, 0, m).store(dW + (size_t)key * E, E, scale, acc);
      }
    }
    if ((threadIdx.x & 63) == 0) many[wave] = m > ALONE ? m : 0;
  }
  __syncthreads();
  for (int w = 0; w < JOIN; ++w) {
    const long m = many[w], c = (long)blockIdx.x * JOIN + w;
    if (!m) continue;
    const long q = (m + JOIN - 1) / JOIN, x0 = wave * q;
    Cols<float, W> sum = total(c, x0, min(m, x0 + q));
    join_waves<Cols<float, W>, W, JOIN - 1>(sum, sh);
    if (wave == 0) sum.store(dW + (size_t)keys[c * CHUNK + CHUNK - 1] * E, E, scale, acc);
    __syncthreads();
  }
}

// workgroups of a launch: fewer than 2^32 threads along an axis
__host__ inline long grid_limit(int threads) { return ((1L << 32) - 1) / threads; }

__host__ inline size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

struct Layout {
  size_t keys[2], slot[2], part, table, bytes;
  long chunks, per;  // tokens per part of the sort
  int kb, passes, parts;
};

__host__ inline Layout layout(long T, long V, int E) {
  Layout l{};
  if (T <= SMALL_T) return l;
  l.kb = V < 65536 ? 2 : 4;
  l.passes = 1;
  while ((1L << (8 * l.passes)) <= V) ++l.passes;  // keys 0 .. V
  l.chunks = (T + CHUNK - 1) / CHUNK;
  l.per = ((T + PARTS - 1) / PARTS + TILE - 1) / TILE * TILE;
  l.parts = (int)((T + l.per - 1) / l.per);
  size_t o = 0;
  for (int i = 0; i < (l.passes > 1 ? 2 : 1); ++i) {
    l.keys[i] = o;
    o = up(o + (size_t)T * l.kb);
    l.slot[i] = o;
    o = up(o + (size_t)T * 4);
  }
  l.part = o;
  o = up(o + (size_t)l.chunks * 2 * E * 4);
  l.table = o;
  l.bytes = up(o + (size_t)l.parts * 256 * 4);
  return l;
}

template <typename TG, typename KT, int W>
int sorted_grad(const Ids& ids, const TG* g, float* dW, long T, long V, int E, long pad, float scale, int acc,
                char* ws, const Layout& l, hipStream_t st) {
  float* part = (float*)(ws + l.part);
  unsigned* table = (unsigned*)(ws + l.table);
  const long z = acc ? 0 : V * E, share = (z / (2 * l.passes) + 3) & ~3L;
  Tokens<KT> src{ids, V, pad, nullptr, nullptr};
  for (int k = 0; k < 2 * l.passes; ++k) {
    const long z0 = min(z, k * share), z1 = k + 1 == 2 * l.passes ? z : min(z, z0 + share);
    const Fill fill{dW + z0, z1 - z0};
    const dim3 grid((unsigned)(l.parts + min((fill.n + 4 * TILE - 1) / (4 * TILE), (long)ZFILL)));
    KT* keys = (KT*)(ws + l.keys[k / 2 & 1]);
    unsigned* slot = (unsigned*)(ws + l.slot[k / 2 & 1]);
    if (k % 2 == 0) {
      hipLaunchKernelGGL((count_kernel<KT>), grid, dim3(TILE), 0, st, src, T, l.per, l.parts, 4 * k, table, fill);
    } else {
      hipLaunchKernelGGL((place_kernel<KT>), grid, dim3(TILE), 0, st, src, T, l.per, l.parts, 4 * (k - 1),
                         (const unsigned*)table, keys, slot, fill);
      src.keys = keys;
      src.slot = slot;
    }
    PV_LAUNCH_CHECK();
  }
  const KT* sk = src.keys;
  const unsigned* slot = src.slot;
  const int slabs = (E + 64 * W - 1) / (64 * W);
  hipLaunchKernelGGL((walk_kernel<TG, KT, W>), dim3((unsigned)((l.chunks + 3) / 4), slabs), dim3(256), 0, st,
                     sk, slot, g, part, dW, T, V, E, scale, acc);
  PV_LAUNCH_CHECK();
  hipLaunchKernelGGL((join_kernel<TG, KT, W>), dim3((unsigned)((l.chunks + JOIN - 1) / JOIN), slabs), dim3(64 * JOIN), 0, st, sk,
                     (const float*)part, dW, T, V, E, scale, acc);
  PV_LAUNCH_CHECK();
  return 0;
}

template <typename TG, int W>
int grad(const Ids& ids, const TG* g, float* dW, long T, long V, int E, long pad, float scale, int acc, char* ws,
         long ws_bytes, hipStream_t st) {
  if (T <= SMALL_T) {
    const int slabs = (E + 64 * W - 1) / (64 * W);
    const long z = acc ? 0 : min(grid_limit(256) - T, (V + ZROWS - 1) / ZROWS);
    if (T + z == 0) return 0;
    hipLaunchKernelGGL((small_grad_kernel<TG, W>), dim3((unsigned)(T + z), slabs), dim3(256), 0, st, ids, g, dW,
                       (int)T, V, E, pad, scale, acc);
    PV_LAUNCH_CHECK();
    return 0;
  }
  const Layout l = layout(T, V, E);
  if (!ws || (size_t)ws_bytes < l.bytes) return -5;
  return l.kb == 2 ? sorted_grad<TG, unsigned short, W>(ids, g, dW, T, V, E, pad, scale, acc, ws, l, st)
                   : sorted_grad<TG, unsigned, W>(ids, g, dW, T, V, E, pad, scale, acc, ws, l, st);
}

template <typename TG>
int grad_w(const Ids& ids, const TG* g, float* dW, long T, long V, int E, long pad, float scale, int acc, char* ws,
           long ws_bytes, hipStream_t st) {
  return E < 4 ? grad<TG, 1>(ids, g, dW, T, V, E, pad, scale, acc, ws, ws_bytes, st)
               : grad<TG, 4>(ids, g, dW, T, V, E, pad, scale, acc, ws, ws_bytes, st);
}

template <typename TW, typename TO>
int lookup(const Ids& ids, const TW* W, TO* out, long T, long V, int E, float scale, const float* pos,
           const float* typ, const Groups& gr, hipStream_t st) {
  const bool vec = E >= 8;
  const int per = vec ? (E + 7) / 8 : E;
  // about four pieces per thread; more where there are so many tokens that the grid could not hold them
  const int rows = (int)max(T / grid_limit(256) + 1, (long)max(1, min(64, 1024 / per)));
  const dim3 grid((unsigned)((T + rows - 1) / rows));
  if (vec)
    hipLaunchKernelGGL((lookup_kernel<TW, TO, 8>), grid, dim3(256), 0, st, ids, W, out, T, V, E, scale, rows, pos, typ, gr);
  else
    hipLaunchKernelGGL((lookup_kernel<TW, TO, 1>), grid, dim3(256), 0, st, ids, W, out, T, V, E, scale, rows, pos, typ, gr);
  PV_LAUNCH_CHECK();
  return 0;
}

}  // namespace temb
}  // namespace pv

using namespace pv;
using namespace pv::temb;

namespace {
inline int temb_sizes(long T, long V, long E) {
  if (T < 0 || V <= 0 || E <= 0) return -1;
  if (T > MAX_T || V >= 0x7FFFFFFFL || E > (1L << 20)) return -2;
  return 0;
}
}  // namespace

// ids (T) int32 / int64; W (V, E) fp32 (w16 = 0) or bf16; out (T, E) bf16 (o16 = 1) or fp32.  pos (Lmax, E) and
// typ (E) fp32, both or none; groups: ng <= 4 (first token, length) pairs, first tokens ascending from 0.  An
// id outside [0, V) gives a row of NaN.
PV_API int pv_temb_fwd(const void* ids, int is64, const void* W, int w16, void* out, int o16, long T, long V, int E,
                       float scale, const float* pos, const float* typ, const int* goff, const int* glen, int ng,
                       void* stream) {
  if (const int rc = temb_sizes(T, V, E)) return rc;
  if (T == 0) return 0;
  Groups gr{};
  if (pos) {
    if (!typ || ng < 1 || ng > 4) return -3;
    gr.n = ng;
    for (int i = 0; i < ng; ++i) gr.off[i] = goff[i], gr.L[i] = glen[i];
  }
  const Ids id{ids, is64};
  hipStream_t st = (hipStream_t)stream;
  if (w16 && o16) return lookup(id, (const unsigned short*)W, (unsigned short*)out, T, V, E, scale, pos, typ, gr, st);
  if (w16) return lookup(id, (const unsigned short*)W, (float*)out, T, V, E, scale, pos, typ, gr, st);
  if (o16) return lookup(id, (const float*)W, (unsigned short*)out, T, V, E, scale, pos, typ, gr, st);
  return lookup(id, (const float*)W, (float*)out, T, V, E, scale, pos, typ, gr, st);
}

// workspace bytes of pv_temb_grad
PV_API long pv_temb_grad_ws(long T, long V, int E) { return temb_sizes(T, V, E) ? 0 : (long)layout(T, V, E).bytes; }

// g (T, E) bf16 (g16 = 1) or fp32; dW (V, E) fp32: every row written (acc = 0) or the rows of the tokens added
// to (acc = 1).  pad: the id whose row gets no gradient, -1 for none.
PV_API int pv_temb_grad(const void* ids, int is64, const void* g, int g16, float* dW, long T, long V, int E, long pad,
                        float scale, int acc, void* ws, long ws_bytes, void* stream) {
  if (const int rc = temb_sizes(T, V, E)) return rc;
  const Ids id{ids, is64};
  hipStream_t st = (hipStream_t)stream;
  return g16 ? grad_w(id, (const unsigned short*)g, dW, T, V, E, pad, scale, acc, (char*)ws, ws_bytes, st)
             : grad_w(id, (const float*)g, dW, T, V, E, pad, scale, acc, (char*)ws, ws_bytes, st);
}
