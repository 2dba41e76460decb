// Layer norm over runs of n columns (a row is `groups` runs), forward and backward.
//
// A run is held by LANES threads of a warp (several runs a warp where they are short) or by a whole CTA, EPT elements a thread in
// registers, so that x is read once: mean first, then the sum of squared distances from it.  A CTA has SPC places, each with a
// group of its own that it keeps over all its rows: weight and bias stay in registers, and the backward adds up its share
// of d_weight and d_bias there; places are joined in shared memory in their order, CTAs by a second kernel in theirs.
// Bound by HBM: x (and d_y) read once, y (d_x) written once.  Forward / backward, us, with the share of a copy's 6.4 TB/s: 65536 x 1024 fp16 in 16 groups
// 52 / 78 (80 %), in one 50 / 80; bf16, 16384 x 4096 54 / 86, 8192 x 8192 56 / 90, 4096 x 16384 64 / -; rows of odd lengths, which take the same loads with
// their ends picked out, 20000 x 2002 bf16 59 / 65 (42 / 57 %: the picking).  The kernel that joins the CTAs' sums takes 5 to 10.  A second row under way
// ahead, forward: no faster (65536 x 1024 52, 16384 x 4096 56), short rows slower (200000 x 128 bf16 25.5 against 23.9: registers).
#pragma once
#include "common.cuh"

namespace fnb {

constexpr int kNormThreads = 256;         // of a CTA that holds several runs
constexpr int kNormMaxCols = 16384;       // of a run: 512 threads with 32 elements each

struct NormParams {
  const void *x, *dy, *w, *b;
  void* y;                    // y, or d_x (may be null)
  int64_t xs, dys, ys;        // row strides, elements
  float *mean, *rstd;
  float* part;                // backward: [CTA][2][span] sums of this CTA, or null
  int64_t rows;
  int n, groups;
  float eps;
  int lanes;                  // threads of a run
  int places, per_row;        // places a CTA uses; how many of them one row takes
  int gblocks;                // blocks of groups (more than one where a row has more groups than a CTA places)
  int span;                   // columns whose sums a CTA has: places of distinct groups x n
  int stride_left, base_left; // SHIFT: elements by which rows lie apart and the first begins, past whole loads
};

// SHIFT, rows of a length that whole loads do not divide: a run's first load is the one that its first element lies in, `off` elements into it.  The rows of a
// place lie a multiple of VEC rows apart (the host sees to it), so that this is the same for all of them.
struct NormPlace {
  int lane, place, group;
  int64_t row, step;
  bool active;
};
template <int VEC> __device__ __forceinline__ int norm_shift(const NormParams& p, const NormPlace& t) {
  return (int)((p.base_left + t.row % VEC * p.stride_left + (int64_t)t.group * p.n) % VEC);
}

// element type of weight and bias: F32 or T
template <class T, bool PF32> struct NormParam { using type = T; };
template <class T> struct NormParam<T, true> { using type = float; };

template <class T, int VEC>
__device__ __forceinline__ void norm_load(const T* p, float* v) {
  if (VEC == 1) {
    v[0] = to_f<T>(*p);
  } else if (VEC * sizeof(T) == 16) {
    load16<T>(p, v);
  } else {      // eight floats beside eight 16-bit values
#pragma unroll
    for (int j = 0; j < VEC; j += 4) load16<T>(p + j, v + j);
  }
}
template <class P, int VEC, bool SHIFT>
__device__ __forceinline__ void norm_param(const P* p, int c, int n, float* v) {
  if (!SHIFT) {
    norm_load<P, VEC>(p + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (c + j >= 0 && c + j < n) v[j] = to_f<P>(p[c + j]);
  }
}
template <class T, int VEC, bool SHIFT>
__device__ __forceinline__ void norm_store(T* p, const float* v, int c, int n) {
  if (VEC == 1) {
    *p = from_f<T>(v[0]);
  } else if (SHIFT && (c < 0 || c + VEC > n)) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (c + j >= 0 && c + j < n) p[j] = from_f<T>(v[j]);
  } else {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = from_f<T>(v[j]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
}

// VEC elements as they lie in memory
template <class T, int VEC> struct NormRaw { uint4 v; };
template <class T> struct NormRaw<T, 1> { T v; };
template <class T, int VEC> __device__ __forceinline__ NormRaw<T, VEC> norm_nothing() {
  NormRaw<T, VEC> r;
  if constexpr (VEC == 1) r.v = from_f<T>(0.f);
  else r.v = make_uint4(0u, 0u, 0u, 0u);
  return r;
}
// Columns c .. c + VEC - 1 of a run.  At a run's ends a load has elements beside it, which norm_inside takes out again: a load of 16 bytes from a multiple of 16 that
// has one of the tensor's elements lies in the tensor's allocation.
template <class T, int VEC> __device__ __forceinline__ NormRaw<T, VEC> norm_raw(const T* run, int c, int n) {
  return c < n ? *reinterpret_cast<const NormRaw<T, VEC>*>(run + c) : norm_nothing<T, VEC>();
}
template <int VEC, bool SHIFT> __device__ __forceinline__ void norm_inside(float* v, int c, int n) {
  if (SHIFT) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = c + j >= 0 && c + j < n ? v[j] : 0.f;
  }
}
template <class T, int VEC> __device__ __forceinline__ void norm_floats(const NormRaw<T, VEC>& r, float* v) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int j = 0; j < VEC; ++j) v[j] = to_f<T>(e[j]);
}

// Sum over `lanes` neighbouring threads of a warp.
__device__ __forceinline__ float norm_lanes(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Two values of every warp of the CTA to all its threads, added up by f(first, second) in the warps' order.  `red`: two sets of 32 floats, used in turn, so
// that one barrier is enough.
template <class F>
__device__ __forceinline__ void norm_block(float a, float b, float* red, int& turn, F&& f) {
  float* r = red + 32 * turn;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) {
    r[threadIdx.x >> 5] = a;
    r[16 + (threadIdx.x >> 5)] = b;
  }
  __syncthreads();
  const int warps = blockDim.x >> 5;
  for (int i = 0; i < warps; ++i) f(r[i], r[16 + i], i);
}
// Columns that a warp of a CTA-wide run holds.
template <int VEC, int ITEMS>
__device__ __forceinline__ int norm_warp_cols(int n, int off, int warp, int threads) {
  int cols = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = (i * threads + 32 * warp) * VEC - off;
    cols += max(0, min(c + 32 * VEC, n) - max(c, 0));
  }
  return cols;
}

template <bool BLOCK>
__device__ __forceinline__ NormPlace norm_place(const NormParams& p) {
  NormPlace t;
  t.lane = BLOCK ? threadIdx.x : threadIdx.x & (p.lanes - 1);
  t.place = BLOCK ? 0 : threadIdx.x / p.lanes;
  const int gb = blockIdx.x % p.gblocks, rb = blockIdx.x / p.gblocks, nrb = gridDim.x / p.gblocks;
  const int rows_at_once = p.places / p.per_row;
  t.group = gb * p.places + t.place % p.per_row;
  t.active = t.place < p.places && t.group < p.groups;
  t.row = (int64_t)rb * rows_at_once + t.place / p.per_row;
  t.step = (int64_t)nrb * rows_at_once;
  return t;
}

// copies of the sums in a CTA of several runs, each of 2 x span <= 2 x 512 floats where there are several
__host__ __device__ constexpr int norm_copies(int lanes, int per_row) { return per_row <= 32 / lanes ? kNormThreads / 32 : 1; }
// threads that an SM should hold at once, by elements a thread: what keeps enough loads under way, and what their registers allow
__host__ __device__ constexpr int norm_resident(bool backward, int elements) {
  return elements <= 8 ? 1024 : elements <= 16 && !backward ? 768 : 512;
}
template <class T, bool PF32, int VEC, int ITEMS, bool BLOCK, bool SHIFT>
__global__ void __launch_bounds__(BLOCK ? 512 : kNormThreads, BLOCK ? norm_resident(false, VEC * ITEMS) / 512 : norm_resident(false, VEC * ITEMS) / kNormThreads) norm_fwd_kernel(NormParams p) {
  using P = typename NormParam<T, PF32>::type;
  constexpr int EPT = VEC * ITEMS;
  __shared__ float red[64];
  int turn = 0;
  const NormPlace t = norm_place<BLOCK>(p);
  const int threads = BLOCK ? blockDim.x : p.lanes, lanes = BLOCK ? 32 : p.lanes;
  const int off = SHIFT ? norm_shift<VEC>(p, t) : 0;
  float w[EPT], b[EPT];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = (i * threads + t.lane) * VEC - off;
#pragma unroll
    for (int j = 0; j < VEC; ++j) { w[i * VEC + j] = 1.f; b[i * VEC + j] = 0.f; }
    if (t.active && c < p.n) {
      if (p.w) norm_param<P, VEC, SHIFT>(static_cast<const P*>(p.w) + (int64_t)t.group * p.n, c, p.n, w + i * VEC);
      if (p.b) norm_param<P, VEC, SHIFT>(static_cast<const P*>(p.b) + (int64_t)t.group * p.n, c, p.n, b + i * VEC);
    }
  }
  __shared__ float warp_cols[16], warp_inv[16];
  if (BLOCK) {
    if (threadIdx.x < (blockDim.x >> 5)) {
      const int cols = norm_warp_cols<VEC, ITEMS>(p.n, off, threadIdx.x, threads);
      warp_cols[threadIdx.x] = (float)cols;
      warp_inv[threadIdx.x] = cols ? 1.f / (float)cols : 0.f;
    }
    __syncthreads();
  }
  const float inv_n = 1.f / (float)p.n;
  // (every thread of a warp goes round as often as the others: the sums are shuffles of whole warps)
  const int64_t first = BLOCK ? t.row : (int64_t)(blockIdx.x / p.gblocks) * (p.places / p.per_row);
  const int apart = BLOCK ? 0 : t.place / p.per_row;
  // the next row's loads are under way while one is worked on
  NormRaw<T, VEC> next[ITEMS];
  const auto fetch = [&](int64_t row) {
    const T* x = static_cast<const T*>(p.x) + row * p.xs + (int64_t)t.group * p.n;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * threads + t.lane) * VEC - off;
      next[i] = t.active && row < p.rows ? norm_raw<T, VEC>(x, c, p.n) : norm_nothing<T, VEC>();
    }
  };
  fetch(first + apart);
  for (int64_t base = first; base < p.rows; base += t.step) {
    const int64_t row = base + apart;
    const bool on = t.active && row < p.rows;
    float v[EPT];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      norm_floats<T, VEC>(next[i], v + i * VEC);
      norm_inside<VEC, SHIFT>(v + i * VEC, (i * threads + t.lane) * VEC - off, p.n);
    }
    fetch(row + t.step);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < EPT; ++j) s += v[j];
    s = norm_lanes(s, lanes);
    // (a warp of a CTA-wide run: about its own mean first; the warps' sums of squares are then moved to the mean of all)
    float mean = s * (BLOCK ? warp_inv[threadIdx.x >> 5] : inv_n), q = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * threads + t.lane) * VEC - off;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const bool in = SHIFT ? c + j >= 0 && c + j < p.n : c < p.n;
        v[i * VEC + j] = in ? v[i * VEC + j] - mean : 0.f;
        q = fmaf(v[i * VEC + j], v[i * VEC + j], q);
      }
    }
    q = norm_lanes(q, lanes);
    if (BLOCK) {
      const float own = mean;
      float all = 0.f, squares = 0.f;
      norm_block(s, q, red, turn, [&](float a, float b, int) { all += a; squares += b; });
      mean = all * inv_n;
      const float* r = red + 32 * (turn ^ 1);
      for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
        const float off = r[w] * warp_inv[w] - mean;
        squares = fmaf(warp_cols[w] * off, off, squares);
      }
      q = squares;
#pragma unroll
      for (int j = 0; j < EPT; ++j) v[j] += own - mean;
    }
    const float r = 1.f / sqrtf(q * inv_n + p.eps);
    if (!on) continue;
    T* y = static_cast<T*>(p.y) + row * p.ys + (int64_t)t.group * p.n;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * threads + t.lane) * VEC - off;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i * VEC + j] = fmaf(v[i * VEC + j] * r, w[i * VEC + j], b[i * VEC + j]);
      if (c < p.n) norm_store<T, VEC, SHIFT>(y + c, v + i * VEC, c, p.n);
    }
    if (t.lane == 0) {
      if (p.mean) p.mean[row * p.groups + t.group] = mean;
      if (p.rstd) p.rstd[row * p.groups + t.group] = r;
    }
  }
}

// With u = d_y w and xh = (x - mean) rstd:  d_x = rstd (u - mean(u) - xh mean(u xh)).
template <class T, bool PF32, int VEC, int ITEMS, bool BLOCK, bool SHIFT>
__global__ void __launch_bounds__(BLOCK ? 512 : kNormThreads, BLOCK ? norm_resident(true, VEC * ITEMS) / 512 : norm_resident(true, VEC * ITEMS) / kNormThreads) norm_bwd_kernel(NormParams p) {
  using P = typename NormParam<T, PF32>::type;
  constexpr int EPT = VEC * ITEMS;
  __shared__ float red[64];
  extern __shared__ float sums[];      // [2][span]
  int turn = 0;
  const NormPlace t = norm_place<BLOCK>(p);
  const int threads = BLOCK ? blockDim.x : p.lanes, lanes = BLOCK ? 32 : p.lanes;
  const int off = SHIFT ? norm_shift<VEC>(p, t) : 0;
  pdl_trigger();
  float w[EPT], dw[EPT], db[EPT];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = (i * threads + t.lane) * VEC - off;
#pragma unroll
    for (int j = 0; j < VEC; ++j) { w[i * VEC + j] = 1.f; dw[i * VEC + j] = db[i * VEC + j] = 0.f; }
    if (p.w && t.active && c < p.n) norm_param<P, VEC, SHIFT>(static_cast<const P*>(p.w) + (int64_t)t.group * p.n, c, p.n, w + i * VEC);
  }
  const float inv_n = 1.f / (float)p.n;
  const int64_t first = BLOCK ? t.row : (int64_t)(blockIdx.x / p.gblocks) * (p.places / p.per_row);
  const int apart = BLOCK ? 0 : t.place / p.per_row;
  NormRaw<T, VEC> next_x[ITEMS], next_d[ITEMS];
  float next_mean, next_r;
  const auto fetch = [&](int64_t row) {
    const bool on = t.active && row < p.rows;
    const T* x = static_cast<const T*>(p.x) + row * p.xs + (int64_t)t.group * p.n;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dys + (int64_t)t.group * p.n;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * threads + t.lane) * VEC - off;
      next_x[i] = on ? norm_raw<T, VEC>(x, c, p.n) : norm_nothing<T, VEC>();
      next_d[i] = on ? norm_raw<T, VEC>(dy, c, p.n) : norm_nothing<T, VEC>();
    }
    next_mean = on ? p.mean[row * p.groups + t.group] : 0.f;
    next_r = on ? p.rstd[row * p.groups + t.group] : 0.f;
  };
  fetch(first + apart);
  for (int64_t base = first; base < p.rows; base += t.step) {
    const int64_t row = base + apart;
    const bool on = t.active && row < p.rows;
    float v[EPT], d[EPT];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      norm_floats<T, VEC>(next_x[i], v + i * VEC);
      norm_floats<T, VEC>(next_d[i], d + i * VEC);
      norm_inside<VEC, SHIFT>(d + i * VEC, (i * threads + t.lane) * VEC - off, p.n);
    }
    const float mean = next_mean, r = next_r;
    fetch(row + t.step);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * threads + t.lane) * VEC - off;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e = i * VEC + j;
        const bool in = on && (SHIFT ? c + j >= 0 && c + j < p.n : c < p.n);
        v[e] = in ? (v[e] - mean) * r : 0.f;
        dw[e] = fmaf(d[e], v[e], dw[e]);
        db[e] += d[e];
        d[e] *= w[e];
        s1 += d[e];
        s2 = fmaf(d[e], v[e], s2);
      }
    }
    if (!p.y) continue;      // (the same for all threads)
    s1 = norm_lanes(s1, lanes);
    s2 = norm_lanes(s2, lanes);
    if (BLOCK) {
      float a1 = 0.f, a2 = 0.f;
      norm_block(s1, s2, red, turn, [&](float a, float b, int) { a1 += a; a2 += b; });
      s1 = a1;
      s2 = a2;
    }
    s1 *= inv_n;
    s2 *= inv_n;
    if (!on) continue;
    T* dx = static_cast<T*>(p.y) + row * p.ys + (int64_t)t.group * p.n;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * threads + t.lane) * VEC - off;
#pragma unroll
      for (int j = 0; j < VEC; ++j) d[i * VEC + j] = r * (d[i * VEC + j] - s1 - v[i * VEC + j] * s2);
      if (c < p.n) norm_store<T, VEC, SHIFT>(dx + c, d + i * VEC, c, p.n);
    }
  }
  if (!p.part) return;
  float* part = p.part + (size_t)blockIdx.x * 2 * p.span;
  if constexpr (BLOCK) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = (i * threads + t.lane) * VEC - off;
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c + j < p.n && (!SHIFT || c + j >= 0)) {
          part[c + j] = dw[i * VEC + j];
          part[p.span + c + j] = db[i * VEC + j];
        }
    }
  } else {
    // Places of one group add to its columns in turn.  Where a warp has every group of a row the warps have a copy of the sums each, and only its own places wait
    // for one another (60000 x 64 bf16: 49 us with one copy, a CTA-wide barrier a place).
    const int copies = norm_copies(p.lanes, p.per_row), in_warp = 32 / p.lanes, warp = threadIdx.x >> 5, size = 2 * p.span;
    for (int c = threadIdx.x; c < copies * size; c += kNormThreads) sums[c] = 0.f;
    __syncthreads();
    const auto add = [&] {
      float* to = sums + (copies > 1 ? warp * size : 0) + (t.place % p.per_row) * p.n;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = (i * threads + t.lane) * VEC - off;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (c + j < p.n && (!SHIFT || c + j >= 0)) {
            to[c + j] += dw[i * VEC + j];
            to[p.span + c + j] += db[i * VEC + j];
          }
      }
    };
    const int turn_of = t.place < p.places ? t.place / p.per_row : -1;
    if (copies > 1) {
      const int last = (warp * in_warp + in_warp - 1) / p.per_row;
      for (int k = warp * in_warp / p.per_row; k <= last; ++k) {
        if (turn_of == k) add();
        __syncwarp();
      }
      __syncthreads();
    } else {
      for (int k = 0; k < p.places / p.per_row; ++k) {
        if (turn_of == k) add();
        __syncthreads();
      }
    }
    for (int c = threadIdx.x; c < size; c += kNormThreads) {
      float a = sums[c];
      for (int i = 1; i < copies; ++i) a += sums[i * size + c];
      part[c] = a;
    }
  }
}

// d_weight (blockIdx.y 0) or d_bias (1): the CTAs' sums of a column.  32 columns a CTA, 32 threads a column, each a run of CTAs in ascending order.
template <class P>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* __restrict__ part, P* __restrict__ dw, P* __restrict__ db, int cols, int n,
                                                           int places, int gblocks, int ctas, int span) {
  __shared__ float s[32][33];
  pdl_wait();
  const int l = threadIdx.x % 32, k = threadIdx.x / 32, c = blockIdx.x * 32 + l;
  P* to = blockIdx.y ? db : dw;
  if (!to) return;
  float a = 0.f;
  if (c < cols) {
    const int gb = gblocks == 1 ? 0 : c / n / places, col = c - gb * places * n, nrb = ctas / gblocks;
    const int r0 = (int)((int64_t)nrb * k / 32), r1 = (int)((int64_t)nrb * (k + 1) / 32);
#pragma unroll 8
    for (int r = r0; r < r1; ++r) a += part[((size_t)(r * gblocks + gb) * 2 + blockIdx.y) * span + col];
  }
  s[k][l] = a;
  __syncthreads();
  if (k == 0 && c < cols) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += s[i][l];
    to[c] = from_f<P>(t);
  }
}

}  // namespace fnb
