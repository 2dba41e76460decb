// Causal attention with a decay for each head, on the CUDA cores: the chunked form for sequences, the sum of states over the
// cuts of a sequence, and the step for single tokens.
//
// Output and all three gradients are one form, taken forwards or backwards in time:
//     A(x, y, z)_s  = sum over t <= s of  exp(g (s - t)) (x_s . y_t) z_t          o = A(q, k, v),  dq = A(do, v, k)
//     A'(x, y, z)_s = sum over t >= s of  exp(g (t - s)) (x_s . y_t) z_t          dk = A'(v, do, q),  dv = A'(k, q, do)
// A chunk of C rows takes the pairs inside it from the C x C product x y^T, masked and weighted, and everything before it from
// the D x D state S = sum exp(..) y z^T, which goes on from chunk to chunk.  Exponents are never negative distances:
// nothing is divided by a power of exp(g), so that no decay, however strong, leaves the range.
#pragma once
#include "common.cuh"

namespace fnb {

struct DecayRows {
  const void* p;
  int64_t sb, sh, sn;
};
struct DecayParams {
  DecayRows x, y, z, out;
  const float* log_decay;     // [H]
  const int32_t* seq_lens;    // [B] or null
  const float* state_in;      // [BH][ncut][D][D] or null (zeros): the state that enters each run of rows
  float* state_out;           // (without outputs) [BH][ncut][D][D]: the sum of each run alone
  int64_t N;
  int H, ncut;                // runs of rows per slice
  int cut0, nrun;             // the runs of this launch: nrun of them from cut0 on
  int64_t seg_rows;           // rows of a segment (a multiple of the chunk)
  int sub;                    // runs per segment
  int64_t sub_rows;           // rows of a run but the last of its segment
  float scale;                // of the output's part from the run's own chunks
  float inter;                // of its part from the state: scale, or 1 where the state has it already (gradients of states)
  float sum_scale;            // of the state's own sums: 1, or scale there
  int transposed;             // the state is read as its transpose
  int vec;                    // every pointer and stride is a multiple of 16 bytes
};

__host__ __device__ inline int64_t decay_cut_begin(int64_t seg_rows, int sub, int64_t sub_rows, int i) {
  return (int64_t)(i / sub) * seg_rows + (int64_t)(i % sub) * sub_rows;
}
// rows [begin, end) of run i, before the sequence's own length is taken into account
__host__ __device__ inline int64_t decay_cut_end(int64_t seg_rows, int sub, int64_t sub_rows, int64_t N, int i) {
  const int64_t seg = (int64_t)(i / sub + 1) * seg_rows;
  int64_t e = i % sub == sub - 1 ? seg : decay_cut_begin(seg_rows, sub, sub_rows, i + 1);
  if (e > seg) e = seg;
  return e < N ? e : N;
}

__device__ __forceinline__ int64_t decay_len(const int32_t* seq_lens, int64_t b, int64_t N) {
  if (!seq_lens) return N;
  const int64_t n = seq_lens[b];
  return n < 0 ? 0 : n > N ? N : n;
}
// -inf stands for "nothing of the past": a finite exponent that gives zero at every distance but 0 (-inf * 0 would be NaN)
__device__ __forceinline__ double decay_log(float g) { return g == -INFINITY ? -1e30 : (double)g; }
// exp(g n) as the sum of two floats.  The state is multiplied by it once a chunk: a factor rounded to one float would be off by
// 2^-24 each time in the same direction, 1e-5 over a few hundred chunks of a slow decay.
struct DecayPair { float hi, lo; };
__device__ __forceinline__ DecayPair decay_pair(double g, int64_t n) {
  const double w = exp(g * (double)n);
  DecayPair p;
  p.hi = (float)w;
  p.lo = p.hi < INFINITY ? (float)(w - (double)p.hi) : 0.f;
  return p;
}
__device__ __forceinline__ float decay_by(const DecayPair& p, float s) { return s == 0.f ? 0.f : fmaf(s, p.hi, s * p.lo); }
// A weight of zero takes what it is given with it, infinities and NaN too.  (Asked once where the weight is the same for all of a state, so not in decay_by.)
__device__ __forceinline__ bool leaves_something(const DecayPair& p) { return p.hi != 0.f; }

// two FP32 values in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}

// ---- chunked form ------------------------------------------------------------------------------------------
// A CTA walks one run of rows, C at a time; tiles in shared memory as FP32.  Thread (ty, tx) of a 16 x 16 grid holds rows
// ty + 16 i of the score and output tiles and a (D / 16)^2 piece of the state.  Bound by the shared-memory loads of its FP32 products (4 x 4 outputs a
// thread: two values loaded for four products; with 128 registers a thread there is no room for more).  fp32, 2 x 8 x 5001 x 64, a pass with outputs / the sums:
// 79 / 29 us; 4 x 8 x 4096 x 128: 329 / 97.  Before tiles were fetched ahead and y' formed once a chunk: 115 / 46 and 532 / 166.  FP32 units at about half their
// rate.  Three-term products on the tensor cores, as the landmark passes have for fp32, are not built.
constexpr int kDecayC = 64;
template <int D> struct DecaySmem {
  static constexpr int LD = D + 4, LP = kDecayC + 4;      // (padded rows: 16 rows read at once fall on different banks)
  static constexpr int kTile = kDecayC * LD, kPowers = 80;
  static constexpr int bytes(bool out) { return (4 * kTile + kPowers + (out ? kDecayC * LP + D * LD : 0)) * 4; }
};

template <class T, int D>
__device__ __forceinline__ void decay_load_tile(float* dst, const DecayRows& t, int64_t base, int64_t row0, int nv, int vec) {
  constexpr int V = Vec16<T>::n, CH = D / V, LD = DecaySmem<D>::LD;
  const T* src = static_cast<const T*>(t.p) + base + row0 * t.sn;
  for (int i = threadIdx.x; i < kDecayC * CH; i += kThreads) {
    const int r = i / CH, c = (i % CH) * V;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
    if (r < nv) {
      const T* p = src + (int64_t)r * t.sn + c;
      if (vec) {
        load16<T>(p, v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_f<T>(p[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; j += 4) *reinterpret_cast<float4*>(dst + r * LD + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  }
}

// The same under way while the CTA goes on, where rows can be copied as they are; a group of its own for decay_arrived.
template <class T, int D>
__device__ __forceinline__ void decay_fetch_tile(float* dst, const DecayRows& t, int64_t base, int64_t row0, int nv, int vec) {
  if (sizeof(T) == 4 && vec) {
    constexpr int CH = D / 4, LD = DecaySmem<D>::LD;
    const float* src = static_cast<const float*>(t.p) + base + row0 * t.sn;
    for (int i = threadIdx.x; i < kDecayC * CH; i += kThreads) {
      const int r = i / CH, c = (i % CH) * 4;
      float* to = dst + r * LD + c;
      if (r < nv) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(src + (int64_t)r * t.sn + c) : "memory");
      else *reinterpret_cast<float4*>(to) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else if (nv > 0) {
    decay_load_tile<T, D>(dst, t, base, row0, nv, vec);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// y' in y's place: row t times exp(g (rows behind it, or before it backwards in time)).  (The CTA meets before and behind it.)
template <int D, bool REV> __device__ __forceinline__ void decay_weigh_tile(float* y, const float* pw, int nv, float scale) {
  for (int i = threadIdx.x; i < nv * (D / 4); i += kThreads) {
    const int t = i / (D / 4);
    const float w = scale * pw[REV ? t + 1 : nv - 1 - t];
    float4* at = reinterpret_cast<float4*>(y + t * DecaySmem<D>::LD + i % (D / 4) * 4);
    float4 v = *at;
    v.x *= w; v.y *= w; v.z *= w; v.w *= w;
    *at = w == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : v;
  }
}
// all but the last PENDING tiles are there
template <int PENDING> __device__ __forceinline__ void decay_arrived() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
  __syncthreads();
}

// CW consecutive floats from shared memory (CW = 1, 2, 4)
template <int CW> __device__ __forceinline__ void decay_lds(const float* p, float* v) {
  if (CW == 4) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x; v[1 % CW] = x.y; v[2 % CW] = x.z; v[3 % CW] = x.w;
  } else {
#pragma unroll
    for (int j = 0; j < CW; ++j) v[j] = p[j];
  }
}

// o += a z, CW values
template <int CW> __device__ __forceinline__ void decay_axpy(float a, const float* z, float* o) {
  if (CW == 1) {
    o[0] = fmaf(a, z[0], o[0]);
  } else {
#pragma unroll
    for (int j = 0; j + 1 < CW; j += 2)
      *reinterpret_cast<float2*>(o + j) = fma2(make_float2(a, a), *reinterpret_cast<const float2*>(z + j), *reinterpret_cast<const float2*>(o + j));
  }
}
template <class T, int D, bool REV, bool OUT>
__global__ void __launch_bounds__(kThreads, D <= 64 ? 2 : 1) decay_chunk_kernel(DecayParams p) {
  using L = DecaySmem<D>;
  constexpr int LD = L::LD, LP = L::LP, C = kDecayC;
  constexpr int CW = D / 16 < 4 ? D / 16 : 4, CG = D / 16 / CW;      // a thread's columns (and state rows): CG groups of CW
  extern __shared__ float4 smem4[];
  // Four tiles take turns.  With outputs: y, x and z of a chunk and the next y; the next x takes x's place and the next z y's as soon as those are done with.
  float* ys = reinterpret_cast<float*>(smem4);
  float* xs = ys + L::kTile;
  float* zs = xs + L::kTile;
  float* spare = zs + L::kTile;
  float* pw = spare + L::kTile;      // exp(g n), n = 0 .. C
  float* ps = pw + L::kPowers;
  float* ss = ps + C * LP;

  const int bh = blockIdx.x / p.nrun, cut = p.cut0 + blockIdx.x % p.nrun;
  const int b = bh / p.H, h = bh % p.H;
  const int64_t len = decay_len(p.seq_lens, b, p.N);
  const int64_t r0 = decay_cut_begin(p.seg_rows, p.sub, p.sub_rows, cut);
  const int64_t r1 = decay_cut_end(p.seg_rows, p.sub, p.sub_rows, p.N, cut);
  const int64_t end = r1 < len ? r1 : len;            // rows that count
  if (!OUT && r0 >= end) return;                       // (what joins the runs knows that there is nothing)
  const double g = decay_log(p.log_decay[h]);
  // (a warp's threads 8 x 4: the 16 bytes that they load for their columns are 128 together)
  const int tx = (threadIdx.x & 7) + (threadIdx.x >> 2 & 8), ty = (threadIdx.x >> 3 & 3) + (threadIdx.x >> 6) * 4;
  for (int i = threadIdx.x; i <= C; i += kThreads) pw[i] = (float)exp(g * i);
  const DecayPair full = decay_pair(g, C);

  T* out = OUT ? static_cast<T*>(const_cast<void*>(p.out.p)) + b * p.out.sb + h * p.out.sh : nullptr;
  if (OUT) {
    const int64_t z0 = r0 > end ? r0 : end;
    for (int64_t i = threadIdx.x; i < (r1 - z0) * D; i += kThreads) out[(z0 + i / D) * p.out.sn + i % D] = from_f<T>(0.f);
  }
  __align__(8) float S[CG][CW][CG][CW];
#pragma unroll
  for (int a = 0; a < CG; ++a)
#pragma unroll
    for (int i = 0; i < CW; ++i)
#pragma unroll
      for (int c = 0; c < CG; ++c)
#pragma unroll
        for (int j = 0; j < CW; ++j) {
          float s = 0.f;
          if (OUT && p.state_in) {
            const int si = a * 64 + ty * CW + i, sj = c * 64 + tx * CW + j;
            s = p.state_in[((size_t)bh * p.ncut + cut) * D * D + (p.transposed ? sj * D + si : si * D + sj)];
          }
          S[a][i][c][j] = s;
        }
  const int64_t bx = b * p.x.sb + h * p.x.sh, by = b * p.y.sb + h * p.y.sh, bz = b * p.z.sb + h * p.z.sh;
  const int chunks = r0 < end ? (int)((end - r0 + C - 1) / C) : 0;
  struct Rows { int64_t at; int n; };
  const auto chunk = [&](int ci) -> Rows {      // (no rows behind the last)
    if (ci >= chunks) return {r0, 0};
    const int64_t c0 = r0 + (int64_t)(REV ? chunks - 1 - ci : ci) * C;
    return {c0, end - c0 < C ? (int)(end - c0) : C};
  };
  const auto fetch = [&](float* to, const DecayRows& t, int64_t base, int ci) {
    const Rows c = chunk(ci);
    if (c.n > 0) decay_fetch_tile<T, D>(to, t, base, c.at, c.n, p.vec);
    else asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(ys, p.y, by, 0);
  if (OUT) fetch(xs, p.x, bx, 0);
  fetch(zs, p.z, bz, 0);
  for (int ci = 0; ci < chunks; ++ci) {
    const Rows rows = chunk(ci);
    const int64_t c0 = rows.at;
    const int nv = rows.n;
    const bool more = ci + 1 < chunks;
    __align__(8) float o[4][CG][CW];
    if (OUT) {
#pragma unroll
      for (int a = 0; a < CG; ++a)
#pragma unroll
        for (int i = 0; i < CW; ++i)
#pragma unroll
          for (int c = 0; c < CG; ++c)
#pragma unroll
            for (int j = 0; j < CW; ++j) ss[(a * 64 + ty * CW + i) * LD + c * 64 + tx * CW + j] = S[a][i][c][j];
      decay_arrived<1>();      // (y and x)
      fetch(spare, p.y, by, ci + 1);
      float2 acc[4][4];      // even and odd columns
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
      for (int k = 0; k < D; k += 4) {
        float4 xv[4], yv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xv[i] = *reinterpret_cast<const float4*>(xs + (ty + 16 * i) * LD + k);
          yv[i] = *reinterpret_cast<const float4*>(ys + (tx + 16 * i) * LD + k);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[i][j] = fma2(make_float2(xv[i].x, xv[i].y), make_float2(yv[j].x, yv[j].y), acc[i][j]);
            acc[i][j] = fma2(make_float2(xv[i].z, xv[i].w), make_float2(yv[j].z, yv[j].w), acc[i][j]);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int s = ty + 16 * i, t = tx + 16 * j, d = REV ? t - s : s - t;
          ps[s * LP + t] = d >= 0 ? (acc[i][j].x + acc[i][j].y) * pw[d] * p.scale : 0.f;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < CG; ++c)
#pragma unroll
          for (int j = 0; j < CW; ++j) o[i][c][j] = 0.f;
      for (int k = 0; k < D; k += 4) {
        float xv[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) decay_lds<4>(xs + (ty + 16 * i) * LD + k, xv[i]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < CG; ++c) {
            __align__(8) float sv[CW];
            decay_lds<CW>(ss + (k + u) * LD + c * 64 + tx * CW, sv);
#pragma unroll
            for (int i = 0; i < 4; ++i) decay_axpy<CW>(xv[i][u], sv, o[i][c]);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = ty + 16 * i;
        const float w = s < nv ? p.inter * pw[REV ? nv - 1 - s : s + 1] : 0.f;
#pragma unroll
        for (int c = 0; c < CG; ++c)
#pragma unroll
          for (int j = 0; j < CW; ++j) o[i][c][j] = w == 0.f ? 0.f : w * o[i][c][j];
      }
      decay_arrived<1>();      // (z; scores are written, x is done with)
      fetch(xs, p.x, bx, ci + 1);
    } else {
      decay_arrived<0>();
      fetch(xs, p.y, by, ci + 1);
      fetch(spare, p.z, bz, ci + 1);
    }
    // the state: U = sum over the chunk's rows, then S = exp(g nv) S + U (nothing needs the one behind the last chunk of a run with outputs)
    if (!OUT || more) {
      decay_weigh_tile<D, REV>(ys, pw, nv, p.sum_scale);
      __syncthreads();
      __align__(8) float U[CG][CW][CG][CW];
#pragma unroll
      for (int a = 0; a < CG; ++a)
#pragma unroll
        for (int i = 0; i < CW; ++i)
#pragma unroll
          for (int c = 0; c < CG; ++c)
#pragma unroll
            for (int j = 0; j < CW; ++j) U[a][i][c][j] = 0.f;
#pragma unroll 4
      for (int t = 0; t < nv; ++t) {
        __align__(8) float yv[CG][CW], zv[CG][CW];
#pragma unroll
        for (int a = 0; a < CG; ++a) {
          decay_lds<CW>(ys + t * LD + a * 64 + ty * CW, yv[a]);
          decay_lds<CW>(zs + t * LD + a * 64 + tx * CW, zv[a]);
        }
#pragma unroll
        for (int a = 0; a < CG; ++a)
#pragma unroll
          for (int i = 0; i < CW; ++i)
#pragma unroll
            for (int c = 0; c < CG; ++c) decay_axpy<CW>(yv[a][i], zv[c], U[a][i][c]);
      }
      const DecayPair by_nv = nv == C ? full : decay_pair(g, nv);
      const bool past = leaves_something(by_nv);
#pragma unroll
      for (int a = 0; a < CG; ++a)
#pragma unroll
        for (int i = 0; i < CW; ++i)
#pragma unroll
          for (int c = 0; c < CG; ++c)
#pragma unroll
            for (int j = 0; j < CW; ++j) S[a][i][c][j] = (past ? decay_by(by_nv, S[a][i][c][j]) : 0.f) + U[a][i][c][j];
    }
    if (OUT) {
      if (more) __syncthreads();      // (y is done with)
      fetch(ys, p.z, bz, ci + 1);
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
        for (int t = tb * 16; t < tb * 16 + 16; t += 4) {
          float pv[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (REV ? i <= tb : i >= tb) decay_lds<4>(ps + (ty + 16 * i) * LP + t, pv[i]);
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < CG; ++c) {
              __align__(8) float zv[CW];
              decay_lds<CW>(zs + (t + u) * LD + c * 64 + tx * CW, zv);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (REV ? i <= tb : i >= tb) decay_axpy<CW>(pv[i][u], zv, o[i][c]);
            }
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = ty + 16 * i;
        if (s >= nv) continue;
        T* to = out + (c0 + s) * p.out.sn;
#pragma unroll
        for (int c = 0; c < CG; ++c) {
          T v[CW];
#pragma unroll
          for (int j = 0; j < CW; ++j) v[j] = from_f<T>(o[i][c][j]);
          if (CW == 4 && p.vec) {
            if (sizeof(T) == 4) *reinterpret_cast<uint4*>(to + c * 64 + tx * CW) = *reinterpret_cast<uint4*>(v);
            else *reinterpret_cast<uint2*>(to + c * 64 + tx * CW) = *reinterpret_cast<uint2*>(v);
          } else {
#pragma unroll
            for (int j = 0; j < CW; ++j) to[c * 64 + tx * CW + j] = v[j];
          }
        }
      }
      float* const was = zs;
      zs = ys; ys = spare; spare = was;
    } else {
      float* const y = ys; float* const z = zs;
      ys = xs; zs = spare; xs = y; spare = z;
    }
  }
  if (OUT) return;
  float* to = p.state_out + ((size_t)bh * p.ncut + cut) * D * D;
#pragma unroll
  for (int a = 0; a < CG; ++a)
#pragma unroll
    for (int i = 0; i < CW; ++i)
#pragma unroll
      for (int c = 0; c < CG; ++c)
#pragma unroll
        for (int j = 0; j < CW; ++j) to[(a * 64 + ty * CW + i) * D + c * 64 + tx * CW + j] = S[a][i][c][j];
}

// ---- the runs of a slice joined -----------------------------------------------------------------------------
// One thread per element of the state of a slice goes through the runs in the order of time: before the first run of a segment
// the state so far is what enters that segment.  What depends on the run alone is formed once a CTA.  A chain over the runs, its loads fetched ahead:
// 9 us for 16 slices in 9 segments of two runs (19 MB), 17 us for 64 slices with heads of 128 in two segments.
struct DecayJoinParams {
  const float* sums;          // [BH][ncut][D][D]: each run alone
  const float* state_in;      // [BH][D][D] or null
  float* seg_states;          // [BH][nseg][D][D] or null
  float* state_out;           // [BH][D][D] or null
  const float* log_decay;
  const int32_t* seq_lens;
  int64_t N;
  int H, D, nseg, sub;
  int64_t seg_rows, sub_rows;
  int count;                  // runs with a sum, in the order of time; with fewer than all of them there is no state_out
};
struct DecayJoinRun { float hi, lo; int rows, seg; };      // exp(g rows); rows that count; the segment that begins (in time) with it, or -1
template <bool REV>
__global__ void __launch_bounds__(kThreads) decay_join_kernel(DecayJoinParams p) {
  extern __shared__ float4 smem4[];
  DecayJoinRun* runs = reinterpret_cast<DecayJoinRun*>(smem4);
  pdl_trigger();
  pdl_wait();
  const int bh = blockIdx.y, e = blockIdx.x * kThreads + threadIdx.x, DD = p.D * p.D, ncut = p.nseg * p.sub;
  const int walk = min(ncut, p.count + 1);
  const double g = decay_log(p.log_decay[bh % p.H]);
  const int64_t len = decay_len(p.seq_lens, bh / p.H, p.N);
  for (int k = threadIdx.x; k < walk; k += kThreads) {
    const int i = REV ? ncut - 1 - k : k;
    int64_t n = decay_cut_end(p.seg_rows, p.sub, p.sub_rows, p.N, i);
    n = (n < len ? n : len) - decay_cut_begin(p.seg_rows, p.sub, p.sub_rows, i);
    if (n < 0 || k >= p.count) n = 0;
    const DecayPair w = decay_pair(g, n);
    runs[k] = {w.hi, w.lo, (int)n, i % p.sub == (REV ? p.sub - 1 : 0) ? i / p.sub : -1};
  }
  __syncthreads();
  if (e >= DD) return;
  float s = p.state_in ? p.state_in[(size_t)bh * DD + e] : 0.f;
  const float* from = p.sums + (size_t)bh * ncut * DD + e;
  float* to = p.seg_states ? p.seg_states + (size_t)bh * p.nseg * DD + e : nullptr;
  constexpr int kAhead = 8;      // sums fetched ahead: the walk is a chain, its loads are not
  for (int k0 = 0; k0 < walk; k0 += kAhead) {
    float u[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      u[k] = k0 + k < walk && runs[k0 + k].rows > 0 ? from[(size_t)(REV ? ncut - 1 - (k0 + k) : k0 + k) * DD] : 0.f;
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k0 + k < walk) {
        const DecayJoinRun run = runs[k0 + k];
        if (to && run.seg >= 0) to[(size_t)run.seg * DD] = s;
        const DecayPair w{run.hi, run.lo};
        if (run.rows > 0) s = (leaves_something(w) ? decay_by(w, s) : 0.f) + u[k];
      }
  }
  if (p.state_out) p.state_out[(size_t)bh * DD + e] = s;
}

// ---- one token ----------------------------------------------------------------------------------------------
// A CTA takes W columns of one head's state: LPR = W / 4 threads hold a row's columns as float4, the rows are spread over the CTA.
// Columns are independent of one another, the sum over the rows ends in shared memory.  Bound by the state,
// read and written once: 4096 heads of 128 (541 MB) 83 us, 6.5 TB/s, which is the rate of a copy.
struct DecayStepParams {
  const void *q, *k, *v;
  void* out;
  int64_t qb, qh, kb, kh, vb, vh, ob, oh;
  const float* log_decay;
  float* states;
  const int32_t* slots;
  int64_t num_states;
  int B, H;
  float scale;
};
template <class T, int D, int W>
__global__ void __launch_bounds__(D * W / 4 < 256 ? D * W / 4 : 256) decay_step_kernel(DecayStepParams p) {
  constexpr int NT = D * W / 4 < 256 ? D * W / 4 : 256, LPR = W / 4, RPI = NT / LPR, ITERS = D / RPI;
  __shared__ float s_q[D], s_k[D], s_sum[RPI][W];
  __shared__ int s_next, s_early;
  const int b0 = blockIdx.x / p.H, h = blockIdx.x % p.H, col = blockIdx.y * W + (threadIdx.x % LPR) * 4, row = threadIdx.x / LPR;
  T* out = static_cast<T*>(p.out);
  int64_t slot = b0;
  if (p.slots) {
    slot = p.slots[b0];
    if (slot < 0 || slot >= p.num_states) {
      if (threadIdx.x < W) out[b0 * p.ob + h * p.oh + blockIdx.y * W + threadIdx.x] = from_f<T>(0.f);
      return;
    }
  }
  float4* S = reinterpret_cast<float4*>(p.states + ((size_t)slot * p.H + h) * D * D + col);
  float4 s[ITERS];
#pragma unroll
  for (int i = 0; i < ITERS; ++i) s[i] = S[(size_t)(row + i * RPI) * (D / 4)];
  // (two floats: one alone is off by up to 2^-25 each token in the same direction, 1e-4 of the state with a memory of 4096 tokens)
  const DecayPair decay = decay_pair(decay_log(p.log_decay[h]), 1);
  int b = b0;
  if (p.slots) {
    // rows of the batch that name one state are tokens in a row: the first of them takes all, the others leave
    if (threadIdx.x == 0) { s_early = 0; s_next = p.B; }
    __syncthreads();
    for (int i = threadIdx.x; i < p.B; i += NT)
      if (i != b0 && p.slots[i] == slot) {
        if (i < b0) s_early = 1;
        else atomicMin(&s_next, i);
      }
    __syncthreads();
    if (s_early) return;
  }
  for (;;) {
    const T* q = static_cast<const T*>(p.q) + b * p.qb + h * p.qh;
    const T* k = static_cast<const T*>(p.k) + b * p.kb + h * p.kh;
    const T* v = static_cast<const T*>(p.v) + b * p.vb + h * p.vh + col;
    for (int i = threadIdx.x; i < D; i += NT) { s_q[i] = to_f<T>(q[i]); s_k[i] = to_f<T>(k[i]); }
    const float v0 = to_f<T>(v[0]), v1 = to_f<T>(v[1]), v2 = to_f<T>(v[2]), v3 = to_f<T>(v[3]);
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      const float kr = s_k[row + i * RPI], qr = s_q[row + i * RPI];
      float4& x = s[i];
      if (!leaves_something(decay)) x = make_float4(0.f, 0.f, 0.f, 0.f);
      // (the token joins the low part: what is added to the state is rounded once, and not the decay before it)
      x.x = fmaf(x.x, decay.hi, fmaf(kr, v0, x.x * decay.lo)); x.y = fmaf(x.y, decay.hi, fmaf(kr, v1, x.y * decay.lo));
      x.z = fmaf(x.z, decay.hi, fmaf(kr, v2, x.z * decay.lo)); x.w = fmaf(x.w, decay.hi, fmaf(kr, v3, x.w * decay.lo));
      o.x = fmaf(qr, x.x, o.x); o.y = fmaf(qr, x.y, o.y); o.z = fmaf(qr, x.z, o.z); o.w = fmaf(qr, x.w, o.w);
    }
    *reinterpret_cast<float4*>(&s_sum[row][(threadIdx.x % LPR) * 4]) = o;
    const int next = p.slots ? s_next : p.B;
    __syncthreads();
    if (threadIdx.x < W) {
      float t = 0.f;
#pragma unroll
      for (int r = 0; r < RPI; ++r) t += s_sum[r][threadIdx.x];
      out[b * p.ob + h * p.oh + blockIdx.y * W + threadIdx.x] = from_f<T>(t * p.scale);
    }
    if (next >= p.B) break;
    b = next;                       // (rare: further tokens for the same state)
    if (threadIdx.x == 0) s_next = p.B;
    __syncthreads();
    for (int i = b + 1 + threadIdx.x; i < p.B; i += NT)
      if (p.slots[i] == slot) atomicMin(&s_next, i);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < ITERS; ++i) S[(size_t)(row + i * RPI) * (D / 4)] = s[i];
}

}  // namespace fnb
