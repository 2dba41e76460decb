// Causal attention with a decay on the tensor cores (fp16 / bf16): out = A(x, y, z) of decay_kernels.cuh, C rows at a time, and the
// sums of y z^T over runs of rows that join the segments of a sequence.
//
// Per chunk, with S the state that enters it (FP32):
//     P = x y^T (C x C)             -> times exp(g |s - t|) and the mask, rounded to 16 bits
//     out = P z + exp(g (s + 1)) x S
//     S = exp(g C) S + y'^T z,      y' = exp(g (C - 1 - t)) y, as one 16-bit term for the outputs, as two or three
//                                                                 for the state that is handed out
// S takes part in x S as the sum of two 16-bit terms.  So each term of an output is rounded once on its way to 16 bits (its score inside a chunk, its y'
// outside), and the output once.
#pragma once
#include "common.cuh"
#include "decay_kernels.cuh"
#include "tc_common.cuh"

namespace fnb {
namespace dtc {

using namespace tc;

constexpr int kGroup = 256;                                   // threads of a group of eight warps
__device__ __forceinline__ uint8_t* at1024(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~(uintptr_t)1023);
}
// operands staged as blocks of [rows x 64] with the 128-byte swizzle: K along the rows' 128 bytes, or K along the rows
__device__ __forceinline__ uint64_t along_row(uint32_t base, int k, int rows) {
  return smem_desc_sw128(base + (k >> 2) * (rows * 128) + (k & 3) * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t along_rows(uint32_t base, int k, int rows) {
  return smem_desc_sw128(base + k * 2048, rows * 128, 1024);
}
struct DecayTcParams {
  const float* log_decay;
  const int32_t* seq_lens;
  const float* state_in;      // main kernel: [BH][nseg][Dr][Dr] or null
  float* sums;                // sums kernel: [BH][ncut][Dr][Dr]
  int64_t N, seg_rows, sub_rows;
  int H, Dr, sub, ncut, cut0, nrun;
  float scale, inter, sum_scale;
  int* status;
};
// One form of a launch of the main kernel.
struct DecayTcForm {
  CUtensorMap x, y, z, o;
  void* out;                  // rows that do not count are cleared by plain stores
  int64_t ob, oh, on;
  int transposed;             // the state is read as its transpose
};
// Two forms that read mostly the same rows (dv and dk: q and do in both, k or v) run side by side, the same segment of both in neighbouring CTAs: what one
// reads the other finds in L2 (1 x 16 x 65536 x 64 bf16: 246 us one after the other, 231 together; 4 x 16 x 16384 x 128: 425 and 430).
template <int FORMS> struct DecayTcForms { DecayTcForm f[FORMS]; };

template <class T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
// 16 values, TERMS of them 16-bit: term t holds what the terms before it leave
template <class T, int TERMS, int N>
__device__ __forceinline__ void split_terms(float2* f, uint32_t (*terms)[N]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      terms[t][j] = pack2<T>(f[j].x, f[j].y);
      if (t + 1 < TERMS) f[j] = fma2(unpack2<T>(terms[t][j]), make_float2(-1.f, -1.f), f[j]);
    }
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
               "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

// y' for 16 bytes (eight elements) of one row, as TERMS 16-bit terms
template <class T, int TERMS>
__device__ __forceinline__ void scaled_terms(uint4 raw, float w, uint4* terms) {
  const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
  float2 f[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = mul2(unpack2<T>(u[j]), make_float2(w, w));
  uint32_t t[TERMS][4];
  split_terms<T, TERMS, 4>(f, t);
#pragma unroll
  for (int k = 0; k < TERMS; ++k) terms[k] = make_uint4(t[k][0], t[k][1], t[k][2], t[k][3]);
}

// Powers of two that take values of up to m into fp16's range and back: m * down lies in 2^14 .. 2^15, so that what is rounded below the normal numbers is 2^-39 of m
// at most.  1 where m is infinite or nothing.
__device__ __forceinline__ void into_range(float m, float& up, float& down) {
  int e = (int)(__float_as_uint(m) >> 23) - 127;
  e = e == 128 || e == -127 ? 14 : min(max(e, -100), 100);
  down = __uint_as_float((uint32_t)(14 - e + 127) << 23);
  up = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
}

// y' of a tile gets a power of two in fp16 where all of y is below 2^-7 (rare): down to there what y' = y e^(..) loses below the normal numbers is 2^-18 of y's largest at
// most.  Whether it is so shows in two bits of the exponents, so that the bits of all values together tell; the exponent that they have together is at most three
// above the largest.  That goes to 14 by the factor, or the factor is 2^24, which leaves a state that is multiplied by it in FP32's range.
__device__ __forceinline__ uint32_t bits_of(uint4 v) { return v.x | v.y | v.z | v.w; }
__device__ __forceinline__ bool not_small(uint32_t bits) { return bits & 0x60006000u; }
__device__ __forceinline__ float factor_of(uint32_t bits) {
  const float m = __half2float(__ushort_as_half((unsigned short)((bits | bits >> 16) & 0x7fffu)));
  const int e = (int)(__float_as_uint(m) >> 23) - 127;
  return e == -127 ? 1.f : __uint_as_float((uint32_t)(min(14 - e, 24) + 127) << 23);
}
// The same for the sums over runs.  Where they are to have FP32's bits y below 2 gets 2^13 already, so that what is lost is 2^-25 of y's largest at most.  Nothing but zeros
// may have any.
template <bool EXACT> __device__ __forceinline__ float sums_factor_of(uint32_t bits) {
  if (bits & (EXACT ? 0x40004000u : 0x60006000u)) return 1.f;
  return bits & 0x20002000u ? 8192.f : bits & 0x7fff7fffu ? factor_of(bits) : 16777216.f;
}
// (of a power of two, exactly)
__device__ __forceinline__ float inverse_of(float power) { return __uint_as_float(0x7f000000u - __float_as_uint(power)); }

// ---- sums over runs ------------------------------------------------------------------------------------------
// One CTA a run, two CTAs an SM: a group of eight warps forms the terms of y', double-buffered, one thread issues the products, which add up in
// tensor memory over kSpan rows (weights reach back that far) before the group takes them out and decays what it has.
// EXACT: two terms of fp16, three of bf16, 22 and 24 bits: the sums are FP32 sums, as a state that is handed out has to be.  Where the sums only join
// segments, one term, as the chunks inside a segment have it: what an output gets from before its segment is then rounded once, like the rest.  In fp16 y' may have a power
// of two in it (sums_factor_of), so that small keys keep these bits.
// Bound by what the eight warps do (a value into terms, two swizzled stores).  1 x 16 x 65536 x 64, 268 MB read: 58 us with one term (4.6 TB/s) in bf16 and 74 in fp16 (58 before
// it looked at y's size), 86 with two (fp16, 74), 80 with three (bf16); 4 x 16 x 16384 x 128, 537 MB, one term, half of the rows (what the first of two segments needs): 68 us.
template <class T, int D, bool EXACT> struct SumsCfg {
  static constexpr int C = D == 64 ? 64 : 32, kStages = 3, kTerms = !EXACT ? 1 : UmmaFmt<T>::v == 0 ? 2 : 3;
  static constexpr int kSpan = 256;
  static constexpr int kTile = C * D * 2;
  static constexpr int kThreads = kGroup + 64;
  static constexpr int kBytes = 1024 + kStages * 2 * kTile + 2 * kTerms * kTile + (kSpan + 1) * 4 + 16 + 256;
};

template <class T, int D, bool EXACT, bool REV>
__global__ void __launch_bounds__((SumsCfg<T, D, EXACT>::kThreads), 2)
decay_tc_sums_kernel(const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_z, DecayTcParams p) {
  using L = SumsCfg<T, D, EXACT>;
  constexpr int C = L::C, NST = L::kStages, KB = D / 64, PER = L::kSpan / C;
  extern __shared__ uint8_t smem_raw[];
  pdl_trigger();
  uint8_t* s_in = at1024(smem_raw);                      // stages of [y | z]
  uint8_t* s_y = s_in + NST * 2 * L::kTile;               // two buffers of kTerms tiles
  float* pw = reinterpret_cast<float*>(s_y + 2 * L::kTerms * L::kTile);
  uint64_t* bars = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(pw + L::kSpan + 1 + 4) + 15) & ~(uintptr_t)15);
  uint64_t* full = bars;             // [3]
  uint64_t* empty = bars + 3;        // [3]
  uint64_t* y_ready = bars + 6;      // [2]
  uint64_t* y_free = bars + 8;       // [2]
  uint64_t* fin = bars + 10;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11);
  int* abort_word = reinterpret_cast<int*>(tmem_slot + 1);
  uint32_t* s_seen = reinterpret_cast<uint32_t*>((reinterpret_cast<uintptr_t>(abort_word + 1) + 15) & ~(uintptr_t)15);      // fp16: [2][8], by chunk parity, bits of y by warp
  constexpr bool F16 = UmmaFmt<T>::v == 0;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bh = blockIdx.x / p.nrun, cut = p.cut0 + blockIdx.x % p.nrun, b = bh / p.H, h = bh % p.H;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NST; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(y_ready + i, kGroup / 32); mbar_init(y_free + i, 1); }
    mbar_init(fin, 1);
    *abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 0) { tmem_alloc(tmem_slot, 2 * D); tmem_relinquish(); }      // the products' sums, and what was taken out of them so far
  tc_fence_before();
  pdl_wait();
  const int64_t len = decay_len(p.seq_lens, b, p.N);
  const int64_t r0 = decay_cut_begin(p.seg_rows, p.sub, p.sub_rows, cut);
  const int64_t r1 = decay_cut_end(p.seg_rows, p.sub, p.sub_rows, p.N, cut);
  const int64_t end = r1 < len ? r1 : len;
  const double g = decay_log(p.log_decay[h]);
  const int count = r0 < end ? (int)((end - r0 + C - 1) / C) : 0;
  for (int i = threadIdx.x; i <= L::kSpan; i += L::kThreads) pw[i] = (float)exp(g * i);
  // what a span decays the sums before it by: a whole one, and (forwards) the last, which may end with the sequence; backwards that one is the first
  DecayPair* s_pair = reinterpret_cast<DecayPair*>(pw + L::kSpan + 1);
  if (threadIdx.x >= L::kThreads - 2)
    s_pair[threadIdx.x - (L::kThreads - 2)] = decay_pair(g, threadIdx.x == L::kThreads - 2 ? L::kSpan : count > 0 ? (end - r0) - (int64_t)(count - PER) * C : 0);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Abort ab{abort_word, p.status};
  // Chunks are taken in the order of time; a span is PER chunks of it, the last one (backwards: the first) may be shorter.
  const auto row_of = [&](int i) { return r0 + (int64_t)(REV ? count - 1 - i : i) * C; };
  // spans are aligned to the end of the run in time, so that each but the first is whole
  const int first_span = count % PER == 0 ? PER : count % PER;
  const auto last_of_span = [&](int i) { return (i + 1 - first_span) % PER == 0 && i + 1 >= first_span; };
  const auto first_of_span = [&](int i) { return i == 0 || last_of_span(i - 1); };

  if (warp == 8) {
    if (lane == 0 && count > 0) {
      tma_prefetch_desc(&tm_y);
      tma_prefetch_desc(&tm_z);
      int armed = 0;
      for (int i = 0; i < count; ++i) {
        const int st = i % NST;
        if (!mbar_wait(empty + st, ((i / NST) & 1) ^ 1, ab, 0x7100 + i)) break;
        mbar_expect_tx(full + st, 2 * L::kTile);
        uint8_t* to = s_in + st * 2 * L::kTile;
        for (int kb = 0; kb < KB; ++kb) {
          tma_load_4d_h(to + kb * (C * 128), &tm_y, full + st, kb * 64, (int)row_of(i), h, b, 0);
          tma_load_4d_h(to + L::kTile + kb * (C * 128), &tm_z, full + st, kb * 64, (int)row_of(i), h, b, 0);
        }
        armed = i + 1;
      }
      if (ab.raised())
        for (int i = max(0, armed - NST); i < armed; ++i) mbar_drain(full + i % NST, (i / NST) & 1);
    }
  } else if (warp == 9) {
    // (the whole warp walks this code and one lane issues: descriptors stay in uniform registers)
    if (count > 0) {
      constexpr uint32_t idesc = make_idesc<T>(D, D, true, true);
      for (int i = 0; i < count; ++i) {
        const int st = i % NST, u = i & 1;
        const bool ok = mbar_wait(full + st, (i / NST) & 1, ab, 0x7280 + i) && mbar_wait(y_ready + u, (i >> 1) & 1, ab, 0x7200 + i);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        // (what was added up before a new sum has been taken out by the time y' is ready)
        const bool fresh = first_of_span(i);
        const uint32_t a_z = smem_u32(s_in + st * 2 * L::kTile + L::kTile), a_y = smem_u32(s_y + u * L::kTerms * L::kTile);
#pragma unroll 1
        for (int t = L::kTerms - 1; t >= 0; --t)
#pragma unroll 2
          for (int k = 0; k < C / 16; ++k)
            umma_elect(tmem, along_rows(a_y + t * L::kTile, k, C), along_rows(a_z, k, C), idesc, !(fresh && t == L::kTerms - 1 && k == 0));
        umma_commit_elect(empty + st);
        umma_commit_elect(y_free + u);
      }
      umma_commit_elect(fin);          // nothing of the CTA is given back while a product runs
      mbar_drain(fin, 0);
    }
  } else {
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int row = D == 64 ? quarter * 16 + lane : quarter * 32 + lane;
    const uint32_t t_sum = tmem + lane_base + half * (D / 2), t_state = t_sum + D;
    // (a wait that gave up does not leave the loop: the warps meet at barriers, and the status word has it)
    const DecayPair whole = s_pair[0], last = s_pair[1];
    constexpr int PIECES = L::kTile / 16 / kGroup;
    const bool grows = pw[L::kSpan] > 1.f;      // (a decay above 0: y' may be larger than y, so no factor)
    int in_span = 0;
    int64_t span_end = 0;        // forwards: the row behind the span; backwards: its first row
    float factor = 1.f;          // fp16: of y' in the sums that are in tensor memory now
    bool some = false;           // there is something in what was taken out so far
    bool decayed = false;        // fp16: and that has been decayed by the span's rows (something of this span has been taken out)
    // Iteration i takes out the sums that chunk i - 1 ended, a span's or (fp16) those that chunk i is too large for, and forms y' of chunk i.
    for (int i = 0; i <= count; ++i) {
      const int st = i % NST, u = i & 1;
      const bool any = i < count, ends = i > 0 && last_of_span(i - 1), first = i == 0 || ends;
      uint8_t* src = s_in + st * 2 * L::kTile;
      uint8_t* dst = s_y + u * L::kTerms * L::kTile;
      const int64_t c0 = row_of(i);
      const int nv = end - c0 < C ? (int)(end - c0) : C;
      // fp16: sums share a factor of y'.  A span begins with that of its first chunk, and does not look at others where that is 1 (the usual).
      const bool looks = F16 && any && !grows && (first || factor != 1.f);
      if (warp == 0) {      // (one warp asks for all)
        if (any) mbar_wait(full + st, (i / NST) & 1, ab, 0x7400 + i);
        if (ends) mbar_wait(y_free + (u ^ 1), ((i - 1) >> 1) & 1, ab, 0x7600 + i);      // (the products of the chunk before)
        else if (i >= 2) mbar_wait(y_free + u, ((i >> 1) & 1) ^ 1, ab, 0x7500 + i);
      }
      if (looks) {
        mbar_wait(full + st, (i / NST) & 1, ab, 0x7480 + i);
        uint32_t bits = 0;
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
          const int idx = threadIdx.x + q * kGroup;
          if (((idx >> 3) & (C - 1)) < nv) bits |= bits_of(*reinterpret_cast<const uint4*>(src + idx * 16));
        }
        bits = __reduce_or_sync(0xffffffffu, bits);
        if (lane == 0) s_seen[u * 8 + warp] = bits;
      }
      named_barrier(1, kGroup);
      float own = 1.f;
      bool less = false;
      if (looks) {
        const uint4 a = *reinterpret_cast<const uint4*>(s_seen + u * 8), b = *reinterpret_cast<const uint4*>(s_seen + u * 8 + 4);
        own = sums_factor_of<EXACT>(bits_of(a) | bits_of(b));
        less = !first && own < factor;
        if (less) {
          if (warp == 0) mbar_wait(y_free + (u ^ 1), ((i - 1) >> 1) & 1, ab, 0x7580 + i);
          named_barrier(1, kGroup);
        }
      }
      if (ends || less) {
        tc_fence_after();
        const DecayPair w = in_span == L::kSpan ? whole : last;
        const bool past = some && (decayed || leaves_something(w));
        const float mul = F16 ? p.sum_scale * inverse_of(factor) : p.sum_scale;
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          float U[16], S[16];
          tmem_ld16(t_sum + q * 16, U);
          if (past) tmem_ld16(t_state + q * 16, S);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) S[j] = (past ? decayed ? S[j] : decay_by(w, S[j]) : 0.f) + mul * U[j];
          tmem_st16(t_state + q * 16, S);
          if (less) {      // (the span's sum goes on from nothing)
#pragma unroll
            for (int j = 0; j < 16; ++j) U[j] = 0.f;
            tmem_st16(t_sum + q * 16, U);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        some = true;
        decayed = less;
      }
      if (!any) break;
      if (first) {
        const int n = i == 0 ? first_span : PER;
        span_end = REV ? row_of(i + n - 1) : row_of(i + n - 1) + C;
        if (!REV && span_end > end) span_end = end;
        in_span = REV ? (int)((i == 0 ? end : row_of(i) + C) - span_end) : (int)(span_end - row_of(i));
      }
      if (F16 && (first || less)) factor = own;
#pragma unroll
      for (int q = 0; q < PIECES; ++q) {
        const int idx = threadIdx.x + q * kGroup, r = (idx >> 3) & (C - 1);
        uint4 terms[L::kTerms];
#pragma unroll
        for (int t = 0; t < L::kTerms; ++t) terms[t] = make_uint4(0, 0, 0, 0);
        // weights: forwards exp(g (rows of the span behind this one)), backwards exp(g (rows of the span up to and with this one))
        if (r < nv) {
          const float w = pw[REV ? (int)(c0 + r - span_end) + 1 : (int)(span_end - 1 - c0 - r)];
          scaled_terms<T, L::kTerms>(*reinterpret_cast<const uint4*>(src + idx * 16), F16 ? factor * w : w, terms);
        } else {
          *reinterpret_cast<uint4*>(src + L::kTile + idx * 16) = make_uint4(0, 0, 0, 0);      // (z's row too: it may hold anything)
        }
#pragma unroll
        for (int t = 0; t < L::kTerms; ++t) *reinterpret_cast<uint4*>(dst + t * L::kTile + idx * 16) = terms[t];
      }
      fence_proxy_async();
      mbar_arrive_warp(y_ready + u);
    }
    if (count > 0) {
      float* to = p.sums + ((size_t)bh * p.ncut + cut) * p.Dr * p.Dr + row * p.Dr;
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        float S[16];
        const int col = half * (D / 2) + q * 16;
        tmem_ld16(t_state + q * 16, S);
        tmem_ld_wait();
        if ((D == 128 || lane < 16) && row < p.Dr && col < p.Dr)
#pragma unroll
          for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(to + col + j) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 2 * D);
}

// ---- outputs -------------------------------------------------------------------------------------------------
// One CTA a segment, one CTA an SM, 28 warps with heads of 64 and 20 with heads of 128, chunks of 128 rows: group A (eight warps; with heads of 64 there are
// two, which take the chunks in turn) turns P into its 16-bit operand and takes the output tile out, group B (eight) forms y' and carries the state, one warp loads, one issues the products of A, one those of B, one
// stores.  The two groups meet only in what the products need: while A works on the scores of a chunk, B is at the state behind it.
//
// Shared memory is what there is least of, its bandwidth (every operand of a product passes it) and, with heads of 128, its room: so P goes to its product
// through tensor memory, the output tile takes x's place, and with heads of 128 y' takes y's.  The state stays in tensor memory: B takes it out to form
// its two 16-bit terms, puts it back decayed, and the products add y'^T z to it.
//
// Measured: 1 x 16 x 65536 x 64, a pass of 537 MB, 144 CTAs: bf16 123 us (4.4 TB/s), fp16 151 (scores, y' and the state are taken into its range by powers of two); 4 x 16 x
// 16384 x 128, 1.07 GB, 128 CTAs: 220 us (4.9 TB/s; 193 is what 128 of 148 SMs move), fp16 250.  Bound with heads of 64 by the warps' arithmetic in turn: of 127 us, 8 go
// without forming y', 10 without the state, 16 without weighing the scores, 6 without the output tile.  What decides it is code that stays in the instruction
// cache: loops over 16 columns that are not unrolled took 131 us where pieces of 32 columns, unrolled, took 150 (fp16 152 and 187).
// Sixteen warps in group B: no change with heads of 64, 238 in place of 216 with 128.  Outputs stored from registers: 195 in place of 162 at the time.
constexpr int kC = 128;      // rows of a chunk
template <int D> struct MainCfg {
  static constexpr int kTile = kC * D * 2;
  static constexpr int kS = D * D * 2;                                   // one term of the state
  static constexpr int kSlots = D == 64 ? 10 : 5;                        // tiles in flight, in the order y, x, z of the chunks
  static constexpr int kTerms = D == 64 ? 2 : 0;                         // tiles for y' (none: in y's place)
  static constexpr int kGroupsA = D == 64 ? 2 : 1;                       // groups A, which take the chunks in turn: as many as there is tensor memory for
  static constexpr int kWarpB = 8 * kGroupsA;                            // first warp of group B, then single warps
  static constexpr int kLoad = kWarpB + 8, kProductsA = kLoad + 1, kProductsB = kLoad + 2, kStore = kLoad + 3;
  static constexpr int kThreads = (kGroupsA + 1) * kGroup + 128;
  // (relies on the dynamic shared window being 1024-byte aligned, which is checked)
  static constexpr int kBytes = (kSlots + kTerms) * kTile + 2 * kS + 32 * 16 * 4 + (kC + 4) * 4 + 128 + (2 * kSlots + 26) * 8 + 16;
  static_assert(kBytes <= 232448, "shared memory of one CTA");
  // Tensor-memory columns.  Packed scores take the place of the scores that they come from, each half of a row in its own: of columns 0-63 from kScores on,
  // of 64-127 from kPackedHalf on behind.  Scores and P z are there for each group A.
  static constexpr int kScores = 0, kPackedHalf = 64, kIntra = kGroupsA * 128, kInter = kIntra + kGroupsA * D, kState = kInter + D;
  static_assert(kState + D <= 512, "tensor memory");
};
// D[tmem] (+)= A[tmem] * B[smem], from warp-uniform code as umma_elect
__device__ __forceinline__ void umma_ta_elect(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <class T, int D, bool REV, int FORMS>
__global__ void __launch_bounds__(MainCfg<D>::kThreads, 1) decay_tc_kernel(const __grid_constant__ DecayTcForms<FORMS> forms, DecayTcParams p) {
  using L = MainCfg<D>;
  constexpr int C = kC, NS = L::kSlots, KB = D / 64, NA = L::kGroupsA;
  constexpr bool F16 = UmmaFmt<T>::v == 0;
  extern __shared__ uint8_t smem_raw[];
  pdl_trigger();
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, (kStatusSmemAlign << 24) | 0x8000);
    return;
  }
  uint8_t* s_in = smem_raw;
  uint8_t* s_y = s_in + NS * L::kTile;                // y' of even and odd chunks
  uint8_t* s_s = s_y + L::kTerms * L::kTile;          // two terms of S
  float* s_diag = reinterpret_cast<float*>(s_s + 2 * L::kS);      // [32][16]: weights beside the diagonal, see below
  float* s_pow = s_diag + 32 * 16;                    // powers of exp(g): forwards that of C - k at k, backwards that of k
  float* s_mul = s_pow + C + 4;                       // [4]: what x S of chunk i is to be multiplied by, in s_mul[i & 3] (B may be ahead)
  float* s_max = s_mul + 4;                           // [8], one a warp of group B: the largest of the state; then [8]: bits of a tile of y; [8] not used
  DecayPair* s_pair = reinterpret_cast<DecayPair*>(s_max + 24);      // [2]: what a chunk decays the state by, a whole one and the first
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_pair + 2);
  uint64_t* full = bars;             // [NS]
  uint64_t* empty = full + NS;       // [NS]
  uint64_t* p_full = empty + NS;     // [4]: scores of chunk i in p_full[i & 3]; B waits for them too and may be two chunks behind
  uint64_t* u_full = p_full + 4;
  uint64_t* s_ready = u_full + 1;
  uint64_t* s_done = u_full + 2;
  uint64_t* clean = u_full + 3;
  uint64_t* i_free = u_full + 4;
  uint64_t* y_ready = u_full + 5;    // [2], by chunk parity: B is a chunk ahead with it
  uint64_t* fin = u_full + 7;        // [2]
  uint64_t* p_ready = u_full + 9;   // [2], by group A
  uint64_t* o_full = u_full + 11;    // [2]
  uint64_t* o_free = u_full + 13;    // [2]
  uint64_t* i_full = u_full + 15;    // [2]
  uint64_t* t_ready = u_full + 17;   // [4]: the output tile of chunk i in t_ready[i & 3]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(u_full + 21);
  int* abort_word = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const DecayTcForm& form = forms.f[FORMS == 1 ? 0 : blockIdx.x % FORMS];
  const int segment = blockIdx.x / FORMS, bh = segment / p.ncut, cut = segment % p.ncut, b = bh / p.H, h = bh % p.H;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 2); }
    for (int i = 0; i < 4; ++i) { mbar_init(p_full + i, 1); mbar_init(t_ready + i, kGroup / 32); }
    mbar_init(u_full, 1); mbar_init(s_ready, kGroup / 32); mbar_init(s_done, 1); mbar_init(clean, kGroup / 32);
    mbar_init(i_free, kGroup / 32);
    for (int i = 0; i < 2; ++i) {
      mbar_init(fin + i, 1); mbar_init(y_ready + i, kGroup / 32); mbar_init(p_ready + i, kGroup / 32); mbar_init(o_full + i, 1);
      mbar_init(o_free + i, kGroup / 32); mbar_init(i_full + i, 1);
    }
    *abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 0) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  pdl_wait();
  const int64_t len = decay_len(p.seq_lens, b, p.N);
  const int64_t r0 = (int64_t)cut * p.seg_rows;
  const int64_t r1 = r0 + p.seg_rows < p.N ? r0 + p.seg_rows : p.N;
  const int64_t end = r1 < len ? r1 : len;
  const double g = decay_log(p.log_decay[h]);
  const int count = r0 < end ? (int)((end - r0 + C - 1) / C) : 0;
  const auto row_of = [&](int i) { return r0 + (int64_t)(REV ? count - 1 - i : i) * C; };
  if (threadIdx.x <= C) s_pow[REV ? threadIdx.x : C - threadIdx.x] = (float)exp(g * threadIdx.x);
  // (only the last chunk in space is not whole: backwards in time the first, forwards one whose state nobody needs)
  if (threadIdx.x >= L::kThreads - 2) s_pair[threadIdx.x - (L::kThreads - 2)] = decay_pair(g, REV && count > 0 && threadIdx.x == L::kThreads - 1 ? end - row_of(0) : C);
  const auto power = [&](int n) { return s_pow[REV ? n : C - n]; };
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Abort ab{abort_word, p.status};
  // Row r of a 32 x 32 block on the diagonal: forwards the weight of column j < 16 is s_diag[r][j], of column 16 + j s_diag[r - 16][j]; backwards of
  // column 16 + j s_diag[r][j], of column j < 16 s_diag[r + 16][j]; what such an index would leave the table with is behind the mask.
  // (16-byte pieces of a row are stored at piece ^ (row / 2) % 4: eight rows read at once fall on different banks)
  if (warp < L::kWarpB) {
    for (int i = threadIdx.x & (kGroup - 1); i < 32 * 16; i += kGroup) {      // (both groups A the same)
      const int row = i / 16, j = i % 16, d = REV ? 16 + j - row : row - j;
      s_diag[row * 16 + ((j / 4) ^ (row / 2 % 4)) * 4 + j % 4] = d >= 0 ? p.scale * power(d) : 0.f;
    }
  }
  // The last rows of a tile lie past the sequence's length, but not past the tensor: they hold anything, and are cleared.
  const int dirty = end == len && len < p.N && (end - r0) % C != 0 ? (REV ? 0 : count - 1) : -1;
  const auto tile = [&](int n) { return s_in + (n % NS) * L::kTile; };      // n = 3 i + 0, 1, 2: y, x, z of chunk i
  const auto landed = [&](int n, int where) { return mbar_wait(full + n % NS, (n / NS) & 1, ab, where + n); };

  if (warp == L::kStore) {
    // ---- output tiles, from x's place to their rows; the place is then free
    if (lane == 0 && count > 0) {
      tma_prefetch_desc(&form.o);
      for (int i = 0; i < count; ++i) {
        if (!mbar_wait(t_ready + (i & 3), (i >> 2) & 1, ab, 0x8080 + i)) break;
        for (int kb = 0; kb < KB; ++kb) tma_store_4d_h(&form.o, tile(3 * i + 1) + kb * (C * 128), kb * 64, (int)row_of(i), h, b, 0);
        tma_store_commit();
        tma_store_wait_read();
        mbar_arrive(empty + (3 * i + 1) % NS);
        mbar_arrive(empty + (3 * i + 1) % NS);
      }
      tma_store_wait_all();
    }
  } else if (warp == L::kLoad) {
    if (lane == 0 && count > 0) {
      tma_prefetch_desc(&form.x);
      tma_prefetch_desc(&form.y);
      tma_prefetch_desc(&form.z);
      int armed = 0;
      for (int n = 0; n < 3 * count; ++n) {
        if (!mbar_wait(empty + n % NS, ((n / NS) & 1) ^ 1, ab, 0x8100 + n)) break;
        mbar_expect_tx(full + n % NS, L::kTile);
        const CUtensorMap* m = n % 3 == 0 ? &form.y : n % 3 == 1 ? &form.x : &form.z;
        for (int kb = 0; kb < KB; ++kb) tma_load_4d_h(tile(n) + kb * (C * 128), m, full + n % NS, kb * 64, (int)row_of(n / 3), h, b, 0);
        armed = n + 1;
      }
      if (ab.raised())
        for (int n = max(0, armed - NS); n < armed; ++n) mbar_drain(full + n % NS, (n / NS) & 1);
    }
  } else if (warp == L::kProductsA) {
    // ---- products of the groups A: the scores of a chunk, and P z of the one before
    // (the whole warp walks this code and the next branch's, and one lane issues: descriptors stay in uniform registers, 70 to 100 cycles a product less)
    if (count > 0) {
      constexpr uint32_t i_p = make_idesc<T>(C, C, false, false), i_o = make_idesc<T>(C, D, false, true);
      const auto scores = [&](int i) -> bool {
        bool ok = landed(3 * i, 0x8200) && landed(3 * i + 1, 0x8280);
        if (i == dirty) ok = ok && mbar_wait(clean, 0, ab, 0x8300 + i);
        // (the product that reads the packed scores among those of NA chunks before has to be done)
        if (i >= NA) ok = ok && mbar_wait(o_full + i % NA, (i / NA - 1) & 1, ab, 0x8400 + i);
        if (!__all_sync(0xffffffffu, ok)) return false;
        tc_fence_after();
        const uint32_t a_y = smem_u32(tile(3 * i)), a_x = smem_u32(tile(3 * i + 1));
#pragma unroll 2
        for (int k = 0; k < D / 16; ++k) umma_elect(tmem + L::kScores + i % NA * 128, along_row(a_x, k, C), along_row(a_y, k, C), i_p, k > 0);
        umma_commit_elect(p_full + (i & 3));
        if (D == 64) umma_commit_elect(empty + (3 * i) % NS);
        return true;
      };
      bool go = scores(0);
      for (int i = 0; go && i < count; ++i) {
        const int ga = i % NA;
        if (NA == 2 && i + 1 < count) go = scores(i + 1);
        if (!go) break;
        bool ok = landed(3 * i + 2, 0x8880) && mbar_wait(p_ready + ga, (i / NA) & 1, ab, 0x8800 + i);
        if (i >= NA) ok = ok && mbar_wait(o_free + ga, (i / NA - 1) & 1, ab, 0x8700 + i);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint32_t a_z = smem_u32(tile(3 * i + 2));
#pragma unroll 2
        for (int k = 0; k < C / 16; ++k)
          umma_ta_elect(tmem + L::kIntra + ga * D, tmem + L::kScores + ga * 128 + (k >> 2) * L::kPackedHalf + 8 * (k & 3), along_rows(a_z, k, C), i_o, k > 0);
        umma_commit_elect(o_full + ga);
        umma_commit_elect(empty + (3 * i + 2) % NS);
        if (NA == 1 && i + 1 < count) go = scores(i + 1);
      }
      umma_commit_elect(fin);          // nothing of the CTA is given back while a product runs
      mbar_drain(fin, 0);
    }
  } else if (warp == L::kProductsB) {
    // ---- products of group B: x S, then the state's own
    if (count > 0) {
      constexpr uint32_t i_o = make_idesc<T>(C, D, false, true), i_u = make_idesc<T>(D, D, true, true);
      const uint32_t a_s = smem_u32(s_s);
      for (int i = 0; i < count; ++i) {
        bool ok = landed(3 * i + 1, 0x8580);
        if (i == dirty) ok = ok && mbar_wait(clean, 0, ab, 0x8590 + i);
        ok = ok && mbar_wait(s_ready, i & 1, ab, 0x8600 + i);
        if (i > 0) ok = ok && mbar_wait(i_free, (i - 1) & 1, ab, 0x8780 + i);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        const uint32_t a_x = smem_u32(tile(3 * i + 1));
#pragma unroll 1
        for (int t = 1; t >= 0; --t)
#pragma unroll 2
          for (int k = 0; k < D / 16; ++k)
            umma_elect(tmem + L::kInter, along_row(a_x, k, C), along_rows(a_s + t * L::kS, k, D), i_o, !(t == 1 && k == 0));
        umma_commit_elect(s_done);
        umma_commit_elect(i_full + i % NA);
        if (i + 1 < count) {
          // (the state in tensor memory has been decayed by the time its 16-bit terms are ready)
          ok = landed(3 * i + 2, 0x8590) && mbar_wait(y_ready + (i & 1), (i >> 1) & 1, ab, 0x8500 + i);
          if (!__all_sync(0xffffffffu, ok)) break;
          tc_fence_after();
          const uint32_t a_y = smem_u32(D == 64 ? s_y + (i & 1) * L::kTile : tile(3 * i)), a_z = smem_u32(tile(3 * i + 2));
#pragma unroll 2
          for (int k = 0; k < C / 16; ++k) umma_elect(tmem + L::kState, along_rows(a_y, k, C), along_rows(a_z, k, C), i_u, 1);
          umma_commit_elect(u_full);
          umma_commit_elect(empty + (3 * i) % NS);      // (with heads of 64 y' has been formed: y_ready)
          if (D == 128) umma_commit_elect(empty + (3 * i) % NS);
          umma_commit_elect(empty + (3 * i + 2) % NS);
        }
      }
      umma_commit_elect(fin + 1);
      mbar_drain(fin + 1, 0);
    }
  } else if (warp < L::kWarpB) {
    // ---- group A: scores and outputs of every NA-th chunk
    // (Here and in group B one warp asks the mbarriers for all, the others wait at a barrier.  A wait that gave up does not leave the loop: the warps meet at barriers, and the status word has it.)
    const int ga = warp >> 3, quarter = warp & 3, half = warp >> 2 & 1, bar = 1 + 2 * ga;
    const bool asks = (warp & 7) == 0;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int w0 = quarter * 32, s = w0 + lane;
    const float largest = fabsf(p.scale) * fmaxf(1.f, power(C - 1));      // of a score's factors
    const float row_factor = p.scale * power(REV ? 32 - lane : lane);
    // rows of the segment past the sequence's length
    {
      const int64_t z0 = r0 + (int64_t)count * C;
      T* out = static_cast<T*>(form.out) + b * form.ob + h * form.oh;
      const int per = p.Dr / 8;
      for (int64_t i = threadIdx.x; i < (r1 - z0) * per; i += NA * kGroup)
        *reinterpret_cast<uint4*>(out + (z0 + i / per) * form.on + (i % per) * 8) = make_uint4(0, 0, 0, 0);
    }
    for (int i = ga; i < count; i += NA) {
      const int nv = end - row_of(i) < C ? (int)(end - row_of(i)) : C;
      if (asks) mbar_wait(p_full + (i & 3), (i >> 2) & 1, ab, 0x8900 + i);
      named_barrier(bar, kGroup);
      tc_fence_after();
      // Scores, weighted and packed, 16 columns at a time.  In fp16 a row's are taken into that type's range by a power of two, its largest (of the blocks that are not
      // masked, unweighted) to 2^14 and more: neither large nor small ones lose more than their rounding.  Each half of a row is looked at by both of its warps, so
      // these meet before either packs.  (Loops are not unrolled: the warps' ways through this kernel have to share the instruction cache.)
      const uint32_t t_row = tmem + L::kScores + ga * 128 + lane_base, t_scores = t_row + half * 64, t_packed = t_scores;
      float up = 1.f, down = 1.f;
      if (F16) {
        float most = 0.f;
#pragma unroll 1
        for (int n = 0; n < 4; ++n) {
          if (REV ? 32 * n < w0 : 32 * n > w0) continue;
          float v[32];
          tmem_ld32(t_row + n * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) most = fmaxf(most, fabsf(v[j]));
        }
        into_range(most * largest, up, down);
        tc_fence_before();
        named_barrier(bar, kGroup);
        tc_fence_after();
      }
#pragma unroll 1
      for (int n = 0; n < 4; ++n) {
        const int t0 = half * 64 + n * 16, part = n & 1, d0 = t0 - 16 * part - w0;      // d0: of the 32-column block, from the diagonal
        float2 v[8];
        uint32_t pk[8];
        if (REV ? d0 < 0 : d0 > 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) pk[j] = 0u;
        } else {
          tmem_ld16(t_scores + n * 16, reinterpret_cast<float*>(v));
          const int from = REV ? lane + 16 - 16 * part : lane - 16 * part;
          const float4* c = reinterpret_cast<const float4*>(d0 == 0 ? s_diag + (from & 31) * 16 : s_pow + (REV ? d0 - 32 : C + d0) + 16 * part);
          const int turn = d0 == 0 ? from / 2 & 3 : 0;
          // on the diagonal the table has it all; behind it exp(g |s - t|) is the row's distance to a block's edge, and the column's
          float row = d0 == 0 ? 1.f : row_factor;
          if (F16) row *= down;
          const bool none = d0 == 0 && (REV ? from >= 32 : from < 0);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 f = c[j ^ turn];
            v[2 * j] = mul2(mul2(v[2 * j], make_float2(row, row)), make_float2(f.x, f.y));
            v[2 * j + 1] = mul2(mul2(v[2 * j + 1], make_float2(row, row)), make_float2(f.z, f.w));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) pk[j] = none ? 0u : pack2<T>(v[j].x, v[j].y);
        }
        tmem_st8(t_packed + n * 8, reinterpret_cast<const float*>(pk));
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive_warp(p_ready + ga);
      float wi = 0.f;
      if (REV ? s < nv : true) wi = p.inter * p.sum_scale * power(REV ? nv - 1 - s : s + 1);
      if (asks) {
        mbar_wait(o_full + ga, (i / NA) & 1, ab, 0x8a00 + i);
        mbar_wait(i_full + ga, (i / NA) & 1, ab, 0x8a80 + i);
      }
      named_barrier(bar, kGroup);
      tc_fence_after();
      if (F16) wi *= s_mul[i & 3];
      uint8_t* to = tile(3 * i + 1);
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        const int col = half * (D / 2) + q * 16;
        float2 a[8], e[8];
        tmem_ld16(tmem + L::kIntra + ga * D + lane_base + col, reinterpret_cast<float*>(a));
        tmem_ld16(tmem + L::kInter + lane_base + col, reinterpret_cast<float*>(e));
        tmem_ld_wait();
        if (q == D / 32 - 1) {
          tc_fence_before();
          mbar_arrive_warp(o_free + ga);
          mbar_arrive_warp(i_free);
        }
        uint32_t u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (F16) a[j] = mul2(a[j], make_float2(up, up));
          if (wi != 0.f) a[j] = fma2(e[j], make_float2(wi, wi), a[j]);
          u[j] = pack2<T>(a[j].x, a[j].y);
        }
        if (s >= nv)      // (cleared rows times an infinity or NaN of one that counts are not zero)
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = 0u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int cc = (col >> 3) + j;
          *reinterpret_cast<uint4*>(to + (cc >> 3) * (C * 128) + sw128_offset(s, cc & 7)) = make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
        }
      }
      fence_proxy_async();
      mbar_arrive_warp(t_ready + (i & 3));
    }
  } else {
    // ---- group B: the state
    const int tid = threadIdx.x - 32 * L::kWarpB, quarter = warp & 3, half = (warp - L::kWarpB) >> 2;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int row = D == 64 ? quarter * 16 + lane : quarter * 32 + lane;
    const bool owner = D == 128 || lane < 16;
    constexpr int HC = D / 2;
    const DecayPair full_chunk = s_pair[0], first_chunk = s_pair[1];
    const uint32_t t_state = tmem + L::kState + lane_base + half * HC;
    // the state that enters the segment, without the factor of the sums, to tensor memory
    if (count > 0) {
      const float mul = 1.f / p.sum_scale;
      const float* from = p.state_in ? p.state_in + ((size_t)bh * p.ncut + cut) * p.Dr * p.Dr + (form.transposed ? row : row * p.Dr) : nullptr;
      const int step = form.transposed ? p.Dr : 1;
#pragma unroll 1
      for (int q = 0; q < HC / 16; ++q) {
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int col = half * HC + q * 16 + j;
          f[j] = from && owner && row < p.Dr && col < p.Dr ? mul * from[col * step] : 0.f;
        }
        tmem_st16(t_state + q * 16, f);
      }
      tmem_st_wait();
    }
    // In fp16 y' of a chunk may have a power of two in it (factor_of); the state that it is added to is put back times that.  (With what finds it 1.5 to 4 % of a call:
    // 1 x 16 x 65536 x 64 forward 237 us, 228 without; 4 x 16 x 16384 x 128 479 and 472.)
    float y_factor = 1.f, held = 1.f;      // of the chunk that put_state is at; the one that the state in tensor memory has
    uint32_t seen = 0;                     // the bits of y that this thread has seen
    const bool grows = power(C - 1) > 1.f;      // (a decay above 0: y' may be larger than y, so no factor)
    constexpr int PIECES = L::kTile / 16 / kGroup;
    const auto rows_in = [&](int i) { const int64_t n = end - row_of(i); return n < C ? (int)n : C; };
    // the factor by what all threads have seen of a small y
    const auto find_factor = [&] {
      uint32_t* s_seen = reinterpret_cast<uint32_t*>(s_max + 8);
      uint32_t bits = __reduce_or_sync(0xffffffffu, seen);
      if (lane == 0) s_seen[warp - L::kWarpB] = bits;
      named_barrier(2, kGroup);
      for (int k = 0; k < 8; ++k) bits |= s_seen[k];
      named_barrier(2, kGroup);
      return factor_of(bits);
    };
    // The state as two 16-bit terms for x S (in fp16 taken into range by a power of two), and, decayed by the chunk's
    // rows, back to tensor memory, where y'^T z is added to it.
    const auto put_state = [&](int i) {
      float down = 1.f;
      if (F16) {
        float most = 0.f, up;
#pragma unroll 1
        for (int q = 0; q < HC / 32; ++q) {
          float f[32];
          tmem_ld32(t_state + q * 32, f);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) most = fmaxf(most, fabsf(f[j]));
        }
        const unsigned w = __reduce_max_sync(0xffffffffu, owner && most < INFINITY ? __float_as_uint(most) : 0u);
        if (lane == 0) s_max[warp - L::kWarpB] = __uint_as_float(w);
        named_barrier(2, kGroup);
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, s_max[k]);
        const float unheld = inverse_of(held);
        into_range(m * unheld, up, down);
        down *= unheld;
        if (tid == 0) s_mul[i & 3] = up;
      }
      DecayPair w = i == 0 ? first_chunk : full_chunk;
      const bool past = leaves_something(w);
      if (F16) {
        const float change = y_factor * inverse_of(held);
        w = {w.hi * change, w.lo * change};
        held = y_factor;
      }
#pragma unroll 1
      for (int q = 0; q < HC / 16; ++q) {
        float2 f[8];
        tmem_ld16(t_state + q * 16, reinterpret_cast<float*>(f));
        tmem_ld_wait();
        if (i + 1 < count) {
          float2 d[8];
          if (past) {
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = fma2(f[j], make_float2(w.hi, w.hi), mul2(f[j], make_float2(w.lo, w.lo)));
            tmem_st16(t_state + q * 16, reinterpret_cast<const float*>(d));
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = make_float2(0.f, 0.f);
            tmem_st16(t_state + q * 16, reinterpret_cast<const float*>(d));
          }
        }
        if (F16)
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = mul2(f[j], make_float2(down, down));
        uint32_t t[2][8];
        split_terms<T, 2, 8>(f, t);
        if (owner) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int cc = (half * HC >> 3) + 2 * q + k;
            const uint32_t off = (cc >> 3) * (D * 128) + sw128_offset(row, cc & 7);
            *reinterpret_cast<uint4*>(s_s + off) = make_uint4(t[0][4 * k], t[0][4 * k + 1], t[0][4 * k + 2], t[0][4 * k + 3]);
            *reinterpret_cast<uint4*>(s_s + L::kS + off) = make_uint4(t[1][4 * k], t[1][4 * k + 1], t[1][4 * k + 2], t[1][4 * k + 3]);
          }
        }
      }
      tmem_st_wait();
      tc_fence_before();
      fence_proxy_async();
      mbar_arrive_warp(s_ready);
    };
    // the state again, times a power of two that it has not got yet (the first chunk's, found while its state is on the way)
    const auto scale_state = [&](float factor) {
#pragma unroll 1
      for (int q = 0; q < HC / 16; ++q) {
        float f[16];
        tmem_ld16(t_state + q * 16, f);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] *= factor;
        tmem_st16(t_state + q * 16, f);
      }
      tmem_st_wait();
      tc_fence_before();
      held = factor;
    };
    // rows of chunk i that do not count, before anything reads them
    const auto clear_rows = [&](int i) {
      const int nv = rows_in(i);
      for (int j = 0; j < 3; ++j) {
        landed(3 * i + j, 0x8b00);
        for (int idx = tid; idx < L::kTile / 16; idx += kGroup)
          if (((idx >> 3) & (C - 1)) >= nv) *reinterpret_cast<uint4*>(tile(3 * i + j) + idx * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async();
      mbar_arrive_warp(clean);
      named_barrier(2, kGroup);
    };
    // y' of chunk i (in y's place: once the scores have been formed from it)
    const auto form_y = [&](int i, float factor) {
      const int nv = rows_in(i);
      const uint8_t* src = tile(3 * i);
      uint8_t* dst = D == 64 ? s_y + (i & 1) * L::kTile : tile(3 * i);
      uint32_t bits = 0;
#pragma unroll 1
      for (int q = 0; q < PIECES; ++q) {
        const int idx = tid + q * kGroup, r = (idx >> 3) & (C - 1);
        const uint4 raw = *reinterpret_cast<const uint4*>(src + idx * 16);
        float w = r < nv ? power(REV ? r + 1 : nv - 1 - r) : 0.f;
        if (F16) w *= factor;
        uint4 term;
        scaled_terms<T, 1>(raw, w, &term);
        *reinterpret_cast<uint4*>(dst + idx * 16) = term;
        if (F16 && D == 64) bits |= bits_of(raw);
      }
      if (F16 && D == 64) seen = bits;
      fence_proxy_async();
    };
    const auto await_y = [&](int i) {
      if (warp == L::kWarpB) {
        landed(3 * i, 0x8c80);
        if (D == 128) mbar_wait(p_full + (i & 3), (i >> 2) & 1, ab, 0x8c00 + i);
      }
      named_barrier(2, kGroup);
    };
    const auto await_products = [&](int i) {      // those of chunk i that the state takes part in
      if (warp == L::kWarpB) {
        mbar_wait(s_done, i & 1, ab, 0x8e00 + i);
        mbar_wait(u_full, i & 1, ab, 0x8d00 + i);
      }
    };
    if constexpr (!F16) {
      const auto put_y = [&](int i) {
        if (i == dirty) clear_rows(i);
        if (i + 1 >= count) return;
        await_y(i);
        form_y(i, 1.f);
        mbar_arrive_warp(y_ready + (i & 1));
      };
      if (count > 0) {
        put_state(0);
        put_y(0);
      }
      // (heads of 64: y' a chunk ahead, while the products that end this one run; its tile is free since u_full of the chunk before)
      for (int i = 0; i + 1 < count; ++i) {
        if (D == 64) put_y(i + 1);
        await_products(i);
        named_barrier(2, kGroup);
        tc_fence_after();
        put_state(i + 1);
        if (D == 128) put_y(i + 1);
      }
    } else if constexpr (D == 64) {
      // the same order; y' is formed without a factor, and again where the barrier behind the products tells that y is small (y is still there)
      for (int c = 0; c < count; ++c) {
        put_state(c);
        for (int i = c ? c + 1 : 0; i <= c + 1 && i < count; ++i) {
          const bool forms = i + 1 < count;
          if (i == dirty) clear_rows(i);
          if (forms) {
            await_y(i);
            form_y(i, 1.f);
          }
          if (i > 0) await_products(i - 1);
          const bool small = !named_barrier_or(2, kGroup, grows || not_small(seen));
          tc_fence_after();
          if (forms) {
            y_factor = 1.f;
            if (small) {
              y_factor = find_factor();
              if (i == 0) scale_state(y_factor);
              if (y_factor != 1.f) form_y(i, y_factor);
            }
            mbar_arrive_warp(y_ready + (i & 1));
          }
        }
      }
    } else {
      // y' takes y's place: y is looked at before the state is put, while products run
      for (int c = 0; c < count; ++c) {
        if (c == dirty) clear_rows(c);
        const bool forms = c + 1 < count;
        if (forms) {
          landed(3 * c, 0x8c90);
          uint32_t bits = 0;
#pragma unroll 4
          for (int q = 0; q < PIECES; ++q) bits |= bits_of(*reinterpret_cast<const uint4*>(tile(3 * c) + (tid + q * kGroup) * 16));
          seen = bits;
        }
        if (c > 0) await_products(c - 1);
        const bool small = !named_barrier_or(2, kGroup, grows || not_small(seen));
        tc_fence_after();
        y_factor = small && forms ? find_factor() : 1.f;
        put_state(c);
        if (forms) {
          await_y(c);
          form_y(c, y_factor);
          mbar_arrive_warp(y_ready + (c & 1));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

}  // namespace dtc
}  // namespace fnb
