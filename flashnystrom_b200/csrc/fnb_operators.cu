// C ABI of the causal attention with a decay and of the layer norm: argument checks, the split of sequences over SMs, launches.
// See include/flashnystrom_b200.h for the contract of every entry point.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "host.cuh"
#include "decay_kernels.cuh"
#include "decay_tc.cuh"
#include "norm_kernels.cuh"
#include "tma_host.cuh"

namespace fnb {

cudaError_t set_operators_wait_limit(unsigned long long ns) { return cudaMemcpyToSymbol(tc::g_wait_limit_ns, &ns, sizeof(ns)); }

// ---- how a sequence is split ----------------------------------------------------------------------------------
// A slice (b, h) is cut into segments of whole 128-row units, one CTA each; the states that enter the segments come from a pass over
// y and z alone, in runs of `sub` to a segment, and one over the D x D sums (decay_join_kernel).  Nothing here depends on pointers, so
// that forward and backward of one call agree.
struct DecayPlan {
  int nseg, sub;
  int64_t seg_rows, sub_rows;
  int runs() const { return nseg * sub; }
};

static DecayPlan decay_plan(const fnb_decay_shape& s) {
  const int64_t unit = s.dtype == FNB_F32 ? 64 : 128;      // rows of a chunk
  const int64_t BH = s.batch * s.heads, units = (s.seq_len + unit - 1) / unit;
  const int sms = current_sm_count();
  // Estimated time of a split, in units that one CTA takes in turn: rounds of CTAs x units of the longest, and, where there is more
  // than one segment, half of that for the pass over the states and about four units' time for two more launches.
  const int slots = s.dtype == FNB_F32 && s.head_dim <= 64 ? 2 * sms : sms;
  int64_t best = 1;
  double least = 1e300;
  const int64_t most = std::min<int64_t>(units, std::max<int64_t>(1, 2 * slots / std::min<int64_t>(BH, 2 * slots)));
  for (int64_t n = 1; n <= most; ++n) {
    const double per = (double)((units + n - 1) / n);
    double t = (double)((BH * n + slots - 1) / slots) * per;
    if (n > 1) t += 0.5 * (double)(BH * (n - 1)) / slots * per + 4.0;
    if (t < least) { least = t; best = n; }
  }
  DecayPlan p;
  p.seg_rows = (units + best - 1) / best * unit;
  p.nseg = (int)((s.seq_len + p.seg_rows - 1) / p.seg_rows);
  // two CTAs of the pass over the states fit on an SM
  int64_t sub = std::max<int64_t>(1, std::min<int64_t>(2 * (int64_t)sms / std::max<int64_t>(1, BH * std::max(1, p.nseg - 1)), p.seg_rows / unit));
  p.sub_rows = (p.seg_rows / unit + sub - 1) / sub * unit;
  p.sub = (int)((p.seg_rows + p.sub_rows - 1) / p.sub_rows);
  return p;
}

static int check_decay_shape(const fnb_decay_shape* s) {
  if (!s) return fail(FNB_ERR_INVALID_ARGUMENT, "shape is NULL");
  if (s->batch <= 0 || s->heads <= 0 || s->seq_len <= 0)
    return fail(FNB_ERR_INVALID_ARGUMENT, "batch, heads and seq_len must be positive (got %lld, %lld, %lld)", (long long)s->batch,
                (long long)s->heads, (long long)s->seq_len);
  if (s->batch > 65535 || s->heads > 65535 || s->batch * s->heads > 65535)
    return fail(FNB_ERR_INVALID_ARGUMENT, "batch * heads (%lld * %lld) exceeds 65535", (long long)s->batch, (long long)s->heads);
  if (s->seq_len > ((int64_t)1 << 30)) return fail(FNB_ERR_INVALID_ARGUMENT, "seq_len (%lld) exceeds 2^30", (long long)s->seq_len);
  if (s->dtype != FNB_F32 && s->dtype != FNB_F16 && s->dtype != FNB_BF16)
    return fail(FNB_ERR_INVALID_ARGUMENT, "Supported dtypes: float32, float16, bfloat16 (got code %d)", s->dtype);
  if (!(s->head_dim == 16 || s->head_dim == 32 || s->head_dim == 64 || s->head_dim == 128))
    return fail(FNB_ERR_INVALID_ARGUMENT, "head_dim must be 16, 32, 64 or 128, got %d", s->head_dim);
  // (gradients of states have the scale in them, and their share of a product is divided by it)
  if (!(std::fabs(s->scale) >= 0x1p-64f && std::fabs(s->scale) <= 0x1p64f))
    return fail(FNB_ERR_INVALID_ARGUMENT, "scale must be finite and not 0, between 2^-64 and 2^64 in magnitude (got %g)", (double)s->scale);
  if (s->flags & ~FNB_FLAG_FORCE_GENERIC) return fail(FNB_ERR_INVALID_ARGUMENT, "unknown flags 0x%x", s->flags);
  return 0;
}

static size_t elem_bytes(int dtype) { return dtype == FNB_F32 ? 4 : 2; }
static int check_rows(const fnb_rows& t, const char* name, int dtype) {
  if (!t.data) return fail(FNB_ERR_INVALID_ARGUMENT, "%s must not be NULL", name);
  if (reinterpret_cast<uintptr_t>(t.data) % elem_bytes(dtype)) return fail(FNB_ERR_INVALID_ARGUMENT, "%s is not aligned to its type", name);
  if (t.stride_b < 0 || t.stride_h < 0 || t.stride_n < 0) return fail(FNB_ERR_INVALID_ARGUMENT, "%s has a negative stride", name);
  return 0;
}
// FP32 and int32 arrays of the caller are read and written element by element: at their type's alignment, or not at all
template <class... P>
static int check_words(const P*... p) {
  if (((reinterpret_cast<uintptr_t>(p) & 3u) | ...)) return fail(FNB_ERR_INVALID_ARGUMENT, "a float or int32 array is not aligned to its type");
  return 0;
}
static bool vec_rows(const fnb_rows& t, int dtype) {
  const int64_t v = 16 / (int64_t)elem_bytes(dtype);
  return aligned16(t.data) && t.stride_b % v == 0 && t.stride_h % v == 0 && t.stride_n % v == 0;
}
static DecayRows rows_of(const fnb_rows& t) { return {t.data, t.stride_b, t.stride_h, t.stride_n}; }

// f(T{}, D as an integral constant)
template <class F>
static int dispatch_decay(int dtype, int D, F&& f) {
  auto by_d = [&](auto tag) -> int {
    switch (D) {
      case 16: return f(tag, std::integral_constant<int, 16>{});
      case 32: return f(tag, std::integral_constant<int, 32>{});
      case 64: return f(tag, std::integral_constant<int, 64>{});
      default: return f(tag, std::integral_constant<int, 128>{});
    }
  };
  switch (dtype) {
    case FNB_F32: return by_d(float{});
    case FNB_F16: return by_d(__half{});
    default: return by_d(__nv_bfloat16{});
  }
}

// What all launches of a call share.
struct DecayCall {
  fnb_decay_shape s;
  DecayPlan plan;
  int64_t BH;
  const float* log_decay;
  const int32_t* seq_lens;
  float* sums;               // [BH][runs][D][D]
  int max_smem;
  cudaStream_t stream;
  int32_t* status;
};
// One A(x, y, z): see decay_kernels.cuh.
struct DecayForm {
  fnb_rows x, y, z, out;
  bool reversed, transposed;
};

static size_t slice_floats(const fnb_decay_shape& s) { return (size_t)s.batch * s.heads * s.head_dim * s.head_dim; }
static size_t segment_floats(const fnb_decay_shape& s, const DecayPlan& p) { return p.nseg > 1 ? slice_floats(s) * p.nseg : 0; }
static size_t decay_ws_bytes(const fnb_decay_shape& s, const DecayPlan& p) {
  return align256(slice_floats(s) * p.runs() * sizeof(float)) + align256(segment_floats(s, p) * sizeof(float));
}

static DecayParams decay_params(const DecayCall& c, const fnb_rows& y, const fnb_rows& z) {
  DecayParams p{};
  p.y = rows_of(y); p.z = rows_of(z);
  p.log_decay = c.log_decay; p.seq_lens = c.seq_lens;
  p.N = c.s.seq_len; p.H = (int)c.s.heads;
  p.seg_rows = c.plan.seg_rows; p.scale = c.s.scale;
  p.vec = vec_rows(y, c.s.dtype) && vec_rows(z, c.s.dtype);
  return p;
}

template <bool REV, bool OUT>
static int launch_chunks(const DecayCall& c, const DecayParams& p, Launcher& L, const char* name) {
  return dispatch_decay(c.s.dtype, c.s.head_dim, [&](auto tag, auto d) -> int {
    using T = decltype(tag);
    constexpr int D = decltype(d)::value;
    auto kern = decay_chunk_kernel<T, D, REV, OUT>;
    constexpr int smem = DecaySmem<D>::bytes(OUT);
    if (int rc = set_smem(kern, smem, c.max_smem, name)) return rc;
    L.begin();
    kern<<<(unsigned)(c.BH * p.nrun), kThreads, smem, c.stream>>>(p);
    return L.end(name);
  });
}

// ---- tensor cores ---------------------------------------------------------------------------------------------
// 16-bit rows that TMA can address: whole 16 bytes everywhere, no dimension spread out of one element.
static bool tma_rows(const fnb_rows& t, const fnb_decay_shape& s) {
  const int64_t size[3] = {s.batch, s.heads, s.seq_len}, stride[3] = {t.stride_b, t.stride_h, t.stride_n};
  for (int i = 0; i < 3; ++i)
    if (size[i] > 1 && (stride[i] <= 0 || stride[i] >= ((int64_t)1 << 38))) return false;
  return vec_rows(t, s.dtype);
}
// (D, N, H, B) map of it, box 64 columns x `rows` rows of one slice: rows past N and columns past D read as zero and are not stored.
static bool make_rows_map(CUtensorMap* map, const fnb_rows& t, const fnb_decay_shape& s, int rows) {
  tc::EncodeTiledFn fn = tc::encode_fn();
  if (!fn) return false;
  const auto stride = [](int64_t size, int64_t st) { return (cuuint64_t)(size > 1 ? st : 128) * 2; };
  cuuint64_t dims[4] = {(cuuint64_t)s.head_dim, (cuuint64_t)s.seq_len, (cuuint64_t)s.heads, (cuuint64_t)s.batch};
  cuuint64_t strides[3] = {stride(s.seq_len, t.stride_n), stride(s.heads, t.stride_h), stride(s.batch, t.stride_b)};
  cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, each[4] = {1, 1, 1, 1};
  return fn(map, tc::map_dtype(s.dtype), 4, t.data, dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// f(T{}, D of the kernel): heads narrower than 64 are padded by the maps
template <class F>
static int dispatch_decay_tc(const fnb_decay_shape& s, F&& f) {
  const auto by_d = [&](auto tag) -> int {
    return s.head_dim <= 64 ? f(tag, std::integral_constant<int, 64>{}) : f(tag, std::integral_constant<int, 128>{});
  };
  return s.dtype == FNB_F16 ? by_d(__half{}) : by_d(__nv_bfloat16{});
}
static dtc::DecayTcParams decay_tc_params(const DecayCall& c, bool reversed) {
  dtc::DecayTcParams p{};
  p.log_decay = c.log_decay; p.seq_lens = c.seq_lens; p.N = c.s.seq_len; p.H = (int)c.s.heads; p.Dr = c.s.head_dim;
  p.seg_rows = c.plan.seg_rows; p.scale = c.s.scale; p.inter = reversed ? 1.f : c.s.scale; p.sum_scale = reversed ? c.s.scale : 1.f;
  p.status = c.status;
  return p;
}
template <bool REV>
static int launch_tc_sums(const DecayCall& c, const fnb_rows& y, const fnb_rows& z, int cut0, int nrun, bool exact, Launcher& L) {
  const auto go = [&](auto tag, auto d, auto ex) -> int {
    using T = decltype(tag);
    constexpr int D = decltype(d)::value;
    constexpr bool EXACT = decltype(ex)::value;
    using Cfg = dtc::SumsCfg<T, D, EXACT>;
    CUtensorMap my, mz;
    if (!make_rows_map(&my, y, c.s, Cfg::C) || !make_rows_map(&mz, z, c.s, Cfg::C)) return fail(FNB_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    dtc::DecayTcParams p = decay_tc_params(c, REV);
    p.sums = c.sums; p.sub = c.plan.sub; p.sub_rows = c.plan.sub_rows; p.ncut = c.plan.runs(); p.cut0 = cut0; p.nrun = nrun;
    auto kern = dtc::decay_tc_sums_kernel<T, D, EXACT, REV>;
    if (int rc = set_smem(kern, Cfg::kBytes, c.max_smem, "decay_sums")) return rc;
    L.begin();
    FNB_CUDA(launch_pdl(kern, dim3((unsigned)(c.BH * nrun)), dim3(Cfg::kThreads), Cfg::kBytes, c.stream, my, mz, p));
    return L.end("decay_sums");
  };
  return dispatch_decay_tc(c.s, [&](auto tag, auto d) -> int { return exact ? go(tag, d, std::true_type{}) : go(tag, d, std::false_type{}); });
}
template <bool REV, int FORMS>
static int launch_tc_forms(const DecayCall& c, const DecayForm* const (&f)[FORMS], const float* state_in, Launcher& L, const char* name) {
  return dispatch_decay_tc(c.s, [&](auto tag, auto d) -> int {
    using T = decltype(tag);
    constexpr int D = decltype(d)::value;
    using Cfg = dtc::MainCfg<D>;
    dtc::DecayTcForms<FORMS> forms;
    for (int i = 0; i < FORMS; ++i) {
      dtc::DecayTcForm& t = forms.f[i];
      if (!make_rows_map(&t.x, f[i]->x, c.s, dtc::kC) || !make_rows_map(&t.y, f[i]->y, c.s, dtc::kC) || !make_rows_map(&t.z, f[i]->z, c.s, dtc::kC) ||
          !make_rows_map(&t.o, f[i]->out, c.s, dtc::kC))
        return fail(FNB_ERR_CUDA, "cuTensorMapEncodeTiled failed");
      t.out = f[i]->out.data; t.ob = f[i]->out.stride_b; t.oh = f[i]->out.stride_h; t.on = f[i]->out.stride_n;
      t.transposed = f[i]->transposed;
    }
    dtc::DecayTcParams p = decay_tc_params(c, REV);
    p.state_in = state_in; p.ncut = c.plan.nseg;
    auto kern = dtc::decay_tc_kernel<T, D, REV, FORMS>;
    if (int rc = set_smem(kern, Cfg::kBytes, c.max_smem, name)) return rc;
    L.begin();
    FNB_CUDA(launch_pdl(kern, dim3((unsigned)(c.BH * c.plan.nseg * FORMS)), dim3(Cfg::kThreads), Cfg::kBytes, c.stream, forms, p));
    return L.end(name);
  });
}
static bool decay_on_tensor_cores(const fnb_decay_shape& s) { return s.dtype != FNB_F32 && !(s.flags & FNB_FLAG_FORCE_GENERIC); }

// The states that enter the segments of a slice -> seg_states (none with one segment), and what leaves the slice -> state_out, where
// that is wanted of this pass.  state_in: what enters the slice.
static int decay_states(const DecayCall& c, const fnb_rows& y, const fnb_rows& z, bool reversed, const float* state_in, float* seg_states,
                        float* state_out, Launcher& L) {
  const bool cut = c.plan.nseg > 1;
  if (!cut && !state_out) return 0;
  // (without state_out nothing needs the sums of the last segment in time)
  const int runs = c.plan.runs(), nrun = state_out ? runs : runs - c.plan.sub, cut0 = state_out || !reversed ? 0 : c.plan.sub;
  if (decay_on_tensor_cores(c.s) && tma_rows(y, c.s) && tma_rows(z, c.s)) {
    if (int rc = reversed ? launch_tc_sums<true>(c, y, z, cut0, nrun, state_out, L) : launch_tc_sums<false>(c, y, z, cut0, nrun, state_out, L)) return rc;
  } else {
    DecayParams p = decay_params(c, y, z);
    p.sum_scale = reversed ? c.s.scale : 1.f;
    p.state_out = c.sums;
    p.ncut = runs; p.sub = c.plan.sub; p.sub_rows = c.plan.sub_rows; p.nrun = nrun; p.cut0 = cut0;
    if (int rc = reversed ? launch_chunks<true, false>(c, p, L, "decay_sums") : launch_chunks<false, false>(c, p, L, "decay_sums")) return rc;
  }
  DecayJoinParams j{};
  j.sums = c.sums; j.state_in = state_in; j.seg_states = cut ? seg_states : nullptr; j.state_out = state_out; j.log_decay = c.log_decay;
  j.seq_lens = c.seq_lens; j.N = c.s.seq_len; j.H = (int)c.s.heads; j.D = c.s.head_dim; j.nseg = c.plan.nseg; j.sub = c.plan.sub;
  j.seg_rows = c.plan.seg_rows; j.sub_rows = c.plan.sub_rows; j.count = nrun;
  const dim3 grid((unsigned)((j.D * j.D + kThreads - 1) / kThreads), (unsigned)c.BH);
  L.begin();
  FNB_CUDA(launch_pdl(reversed ? decay_join_kernel<true> : decay_join_kernel<false>, grid, dim3(kThreads), runs * sizeof(DecayJoinRun), c.stream, j));
  return L.end("decay_join");
}

static bool tma_form(const DecayCall& c, const DecayForm& f) {
  return decay_on_tensor_cores(c.s) && tma_rows(f.x, c.s) && tma_rows(f.y, c.s) && tma_rows(f.z, c.s) && tma_rows(f.out, c.s);
}
// out = scale A(x, y, z) with the states that enter each segment.  Backwards in time the state is dL/dS, which has the scale in it.
static int decay_form(const DecayCall& c, const DecayForm& f, const float* state_in, Launcher& L, const char* name) {
  if (tma_form(c, f)) return f.reversed ? launch_tc_forms<true, 1>(c, {&f}, state_in, L, name) : launch_tc_forms<false, 1>(c, {&f}, state_in, L, name);
  DecayParams p = decay_params(c, f.y, f.z);
  p.x = rows_of(f.x); p.out = rows_of(f.out);
  p.vec = p.vec && vec_rows(f.x, c.s.dtype) && vec_rows(f.out, c.s.dtype);
  p.state_in = state_in;
  p.inter = f.reversed ? 1.f : c.s.scale;
  p.sum_scale = f.reversed ? c.s.scale : 1.f;
  p.ncut = p.nrun = c.plan.nseg; p.sub = 1; p.sub_rows = p.seg_rows; p.transposed = f.transposed;
  return f.reversed ? launch_chunks<true, true>(c, p, L, name) : launch_chunks<false, true>(c, p, L, name);
}

static int check_decay_common(const DecayCall& c, const float* segment_states, const void* ws, size_t ws_bytes) {
  if (!c.log_decay) return fail(FNB_ERR_INVALID_ARGUMENT, "log_decay must not be NULL");
  if (c.plan.nseg > 1 && !segment_states) return fail(FNB_ERR_INVALID_ARGUMENT, "segment_states must not be NULL for this shape");
  const size_t need = decay_ws_bytes(c.s, c.plan);
  if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u))
    return fail(FNB_ERR_WORKSPACE, "workspace must be 256-byte aligned and >= %zu bytes (got %zu)", need, ws_bytes);
  return 0;
}

static int check_norm_shape(const fnb_norm_shape* s) {
  if (!s) return fail(FNB_ERR_INVALID_ARGUMENT, "shape is NULL");
  if (s->rows <= 0 || s->cols <= 0) return fail(FNB_ERR_INVALID_ARGUMENT, "rows and cols must be positive (got %lld, %d)", (long long)s->rows, s->cols);
  if (s->groups <= 0 || s->cols % s->groups)
    return fail(FNB_ERR_INVALID_ARGUMENT, "cols (%d) must be a multiple of groups (%d)", s->cols, s->groups);
  if (s->cols / s->groups > kNormMaxCols)
    return fail(FNB_ERR_INVALID_ARGUMENT, "at most %d columns are normalised together, got %d", kNormMaxCols, s->cols / s->groups);
  if (s->rows > ((int64_t)1 << 40)) return fail(FNB_ERR_INVALID_ARGUMENT, "rows (%lld) exceeds 2^40", (long long)s->rows);
  if (s->dtype != FNB_F32 && s->dtype != FNB_F16 && s->dtype != FNB_BF16)
    return fail(FNB_ERR_INVALID_ARGUMENT, "Supported dtypes: float32, float16, bfloat16 (got code %d)", s->dtype);
  if (s->param_dtype != FNB_F32 && s->param_dtype != s->dtype)
    return fail(FNB_ERR_INVALID_ARGUMENT, "weight and bias must be float32 or of x's dtype");
  if (!std::isfinite(s->eps) || s->eps < 0.f) return fail(FNB_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0 (got %g)", (double)s->eps);
  return 0;
}

// How a norm is spread over threads and CTAs: by the shape, the SM count and how rows can be read.  The workspace has room for any of the three ways.
struct NormPlan {
  int how;                   // NormLoads
  int vec, items;            // elements of a load; loads of a thread
  bool block;                // a run is a CTA's
  int threads, lanes, places, per_row, gblocks, span, ctas;
};
// How rows are read: loads of 16 bytes that their starts and lengths are multiples of; such loads with the rows' ends picked out of them, where x, y (and the gradients)
// lie alike; one element at a time.
enum NormLoads { kNormWhole, kNormShifted, kNormSingle };
static NormPlan norm_plan(const fnb_norm_shape& s, NormLoads how, bool backward, int sms) {
  NormPlan p;
  const int n = s.cols / s.groups, V = 16 / (int)elem_bytes(s.dtype);
  p.how = how;
  p.vec = how == kNormSingle ? 1 : V;
  // Up to 512 columns a warp (or a part of one) holds a run, 16 elements a thread and two loads where there are as many; above that a CTA, 16 elements a
  // thread while it has threads (65536 x 1024 fp16, backward: 95 us, with a warp a run 168).  The forward keeps to warps up to 1024 columns of 16 bits
  // (56 us, a CTA a run 76), and to 32 elements a thread above: fewer warps meet once a row, and an SM has several CTAs, which wait for their own row alone
  // (bf16, 16384 x 4096: 54 us, with 16 elements 77; 8192 x 8192: 56 and 79; not where ends are picked out, which takes registers: fp32, 3000 x 7001, 55 and 41).
  p.block = n > (!backward && how == kNormWhole && V == 8 ? 1024 : 512);
  const int loads = how == kNormShifted ? (n + 2 * V - 2) / V : (n + p.vec - 1) / p.vec;
  if (!p.block) {
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes * (p.vec > 1 ? 2 : 1) < loads) p.lanes *= 2;
    p.items = (loads + p.lanes - 1) / p.lanes;
    p.threads = kNormThreads;
    const int spc = kNormThreads / p.lanes;
    p.per_row = std::min(s.groups, spc);
    p.places = spc / p.per_row * p.per_row;
    p.gblocks = (s.groups + p.per_row - 1) / p.per_row;
    if (p.gblocks > 1) p.places = p.per_row;
  } else {
    p.lanes = 32;
    p.threads = 64;
    const bool few = !backward && how == kNormWhole;
    const int each = few ? 32 : 16, most = few && n <= 8192 ? 256 : 512;
    while (p.threads < most && loads * p.vec > p.threads * each) p.threads *= 2;
    p.items = (loads + p.threads - 1) / p.threads;
    p.per_row = p.places = 1;
    p.gblocks = s.groups;
  }
  p.span = p.per_row * n;
  const int64_t at_once = p.places / p.per_row;
  const int64_t row_blocks = (s.rows + at_once - 1) / at_once;
  const int64_t slots = (int64_t)sms * std::max(1, norm_resident(backward, p.vec * p.items) / p.threads);
  int64_t nrb = std::max<int64_t>(1, std::min<int64_t>(row_blocks, slots / p.gblocks));
  if (how == kNormShifted && nrb < row_blocks) nrb = std::min<int64_t>(row_blocks, std::max<int64_t>(1, nrb / V) * V);      // (see norm_shift)
  p.ctas = p.gblocks * (int)nrb;
  return p;
}
static size_t norm_ws_bytes(const fnb_norm_shape& s) {
  const int sms = current_sm_count();
  size_t most = 0;
  for (NormLoads how : {kNormWhole, kNormShifted, kNormSingle}) {
    const NormPlan p = norm_plan(s, how, true, sms);
    most = std::max(most, (size_t)p.ctas * 2 * p.span);
  }
  return align256(most * sizeof(float));
}

// f(T{}, PF32, VEC, ITEMS, BLOCK, SHIFT)
template <class F>
static int dispatch_norm(const fnb_norm_shape& s, const NormPlan& p, F&& f) {
  auto by_items = [&](auto tag, auto pf, auto block) -> int {
    constexpr int V = 16 / sizeof(tag);
    using I = std::integral_constant<int, V>;
    using One = std::integral_constant<int, 1>;
    const auto vectors = [&](auto shift) -> int {
      if (p.items <= 1) return f(tag, pf, I{}, std::integral_constant<int, 1>{}, block, shift);
      if (p.items <= 2) return f(tag, pf, I{}, std::integral_constant<int, 2>{}, block, shift);
      if (V == 8 || p.items <= 4) return f(tag, pf, I{}, std::integral_constant<int, 4>{}, block, shift);
      return f(tag, pf, I{}, std::integral_constant<int, 32 / V>{}, block, shift);
    };
    if (p.how == kNormWhole) return vectors(std::false_type{});
    if (p.how == kNormShifted) return vectors(std::true_type{});
    if (p.items <= 8) return f(tag, pf, One{}, std::integral_constant<int, 8>{}, block, std::false_type{});
    if (p.items <= 16) return f(tag, pf, One{}, std::integral_constant<int, 16>{}, block, std::false_type{});
    return f(tag, pf, One{}, std::integral_constant<int, 32>{}, block, std::false_type{});
  };
  auto by_block = [&](auto tag, auto pf) -> int {
    return p.block ? by_items(tag, pf, std::true_type{}) : by_items(tag, pf, std::false_type{});
  };
  auto by_param = [&](auto tag) -> int {
    return s.param_dtype == FNB_F32 ? by_block(tag, std::true_type{}) : by_block(tag, std::false_type{});
  };
  switch (s.dtype) {
    case FNB_F32: return by_block(float{}, std::true_type{});
    case FNB_F16: return by_param(__half{});
    default: return by_param(__nv_bfloat16{});
  }
}
static NormParams norm_params(const fnb_norm_shape& s, const NormPlan& n) {
  NormParams p{};
  p.rows = s.rows; p.n = s.cols / s.groups; p.groups = s.groups; p.eps = s.eps;
  p.lanes = n.lanes; p.places = n.places; p.per_row = n.per_row; p.gblocks = n.gblocks; p.span = n.span;
  return p;
}
static bool typed(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % elem_bytes(dtype) == 0; }
// How far into 16 bytes a tensor's first row begins, and rows lie apart past whole ones, in elements.
struct NormAlign { int base, stride; };
static NormAlign norm_align(const void* p, int64_t stride, int dtype) {
  const int64_t e = (int64_t)elem_bytes(dtype), V = 16 / e;
  return {(int)(reinterpret_cast<uintptr_t>(p) / e % V), (int)((stride % V + V) % V)};
}
static NormLoads norm_loads(const fnb_norm_shape& s, const NormAlign* t, int count, bool params_wide) {
  const int V = 16 / (int)elem_bytes(s.dtype);
  bool alike = true;
  for (int i = 1; i < count; ++i) alike = alike && t[i].base == t[0].base && t[i].stride == t[0].stride;
  const int n = s.cols / s.groups;
  if (alike && t[0].base == 0 && t[0].stride == 0 && n % V == 0 && params_wide) return kNormWhole;
  return alike && n + V - 1 <= kNormMaxCols ? kNormShifted : kNormSingle;
}

}  // namespace fnb

using namespace fnb;

extern "C" {

int fnb_check_decay_shape(const fnb_decay_shape* shape) { return check_decay_shape(shape); }
size_t fnb_decay_segment_floats(const fnb_decay_shape* shape) {
  return check_decay_shape(shape) ? 0 : segment_floats(*shape, decay_plan(*shape));
}
size_t fnb_decay_workspace_bytes(const fnb_decay_shape* shape) {
  return check_decay_shape(shape) ? 0 : decay_ws_bytes(*shape, decay_plan(*shape));
}

int fnb_decay_forward(const fnb_decay_fwd_args* a) {
  if (!a) return fail(FNB_ERR_INVALID_ARGUMENT, "args is NULL");
  if (int rc = check_decay_shape(&a->shape)) return rc;
  const struct { const fnb_rows* t; const char* name; } big[] = {{&a->q, "q"}, {&a->k, "k"}, {&a->v, "v"}, {&a->out, "out"}};
  for (const auto& e : big)
    if (int rc = check_rows(*e.t, e.name, a->shape.dtype)) return rc;
  if (int rc = check_words(a->log_decay, a->seq_lens, a->initial_state, a->final_state, a->segment_states)) return rc;
  DeviceGuard g(a->device);
  if (!g.ok) return fail(FNB_ERR_CUDA, "cannot select CUDA device %d", a->device);
  int max_smem = 0, cc = 0, sms = 0;
  if (int rc = device_limits(a->device, &max_smem, &cc, &sms)) return rc;
  DecayCall c{a->shape, decay_plan(a->shape), a->shape.batch * a->shape.heads, a->log_decay, a->seq_lens, (float*)a->workspace, max_smem,
              (cudaStream_t)a->stream, a->device_status};
  if (int rc = check_decay_common(c, a->segment_states, a->workspace, a->workspace_bytes)) return rc;
  Launcher L(c.stream, a->device);
  const bool cut = c.plan.nseg > 1;
  const DecayForm out{a->q, a->k, a->v, a->out, false, false};
  // (one segment: its outputs read initial_state itself, which final_state may be, so they come before the sums)
  if (!cut)
    if (int rc = decay_form(c, out, a->initial_state, L, "decay_fwd")) return rc;
  if (int rc = decay_states(c, a->k, a->v, false, a->initial_state, a->segment_states, a->final_state, L)) return rc;
  return cut ? decay_form(c, out, a->segment_states, L, "decay_fwd") : 0;
}

int fnb_decay_backward(const fnb_decay_bwd_args* a) {
  if (!a) return fail(FNB_ERR_INVALID_ARGUMENT, "args is NULL");
  if (int rc = check_decay_shape(&a->shape)) return rc;
  const struct { const fnb_rows* t; const char* name; } big[] = {{&a->q, "q"}, {&a->k, "k"}, {&a->v, "v"}, {&a->d_out, "d_out"},
                                                                 {&a->dq, "dq"}, {&a->dk, "dk"}, {&a->dv, "dv"}};
  for (const auto& e : big)
    if (int rc = check_rows(*e.t, e.name, a->shape.dtype)) return rc;
  if (int rc = check_words(a->log_decay, a->seq_lens, a->initial_state, a->d_final_state, a->d_initial_state, a->segment_states)) return rc;
  DeviceGuard g(a->device);
  if (!g.ok) return fail(FNB_ERR_CUDA, "cannot select CUDA device %d", a->device);
  int max_smem = 0, cc = 0, sms = 0;
  if (int rc = device_limits(a->device, &max_smem, &cc, &sms)) return rc;
  DecayCall c{a->shape, decay_plan(a->shape), a->shape.batch * a->shape.heads, a->log_decay, a->seq_lens, (float*)a->workspace, max_smem,
              (cudaStream_t)a->stream, a->device_status};
  if (int rc = check_decay_common(c, a->segment_states, a->workspace, a->workspace_bytes)) return rc;
  Launcher L(c.stream, a->device);
  const bool cut = c.plan.nseg > 1;
  // E = dL/dS runs backwards in time; its states at the cuts lie behind the sums in the workspace
  float* e_states = (float*)((char*)a->workspace + align256(slice_floats(c.s) * c.plan.runs() * sizeof(float)));
  const auto states = [&] { return decay_states(c, a->q, a->d_out, true, a->d_final_state, e_states, a->d_initial_state, L); };
  if (cut)
    if (int rc = states()) return rc;
  const float* e_in = cut ? e_states : a->d_final_state;
  if (int rc = decay_form(c, {a->d_out, a->v, a->k, a->dq, false, true}, cut ? a->segment_states : a->initial_state, L, "decay_dq")) return rc;
  const DecayForm dv{a->k, a->q, a->d_out, a->dv, true, false}, dk{a->v, a->d_out, a->q, a->dk, true, true};
  if (tma_form(c, dv) && tma_form(c, dk)) {
    if (int rc = launch_tc_forms<true, 2>(c, {&dv, &dk}, e_in, L, "decay_dv_dk")) return rc;
  } else {
    if (int rc = decay_form(c, dv, e_in, L, "decay_dv")) return rc;
    if (int rc = decay_form(c, dk, e_in, L, "decay_dk")) return rc;
  }
  return cut ? 0 : states();      // (one segment: d_initial_state may be the memory of a state that the gradients read)
}

int fnb_decay_step(const fnb_decay_step_args* a) {
  if (!a) return fail(FNB_ERR_INVALID_ARGUMENT, "args is NULL");
  fnb_decay_shape s{a->batch, a->heads, 1, a->head_dim, a->dtype, a->scale, 0};
  if (s.batch > 65535) return fail(FNB_ERR_INVALID_ARGUMENT, "batch (%lld) exceeds 65535", (long long)s.batch);
  if (s.heads > 0 && s.heads <= 65535 && s.batch * s.heads > INT32_MAX)
    return fail(FNB_ERR_INVALID_ARGUMENT, "batch * heads (%lld * %lld) exceeds 2^31 - 1", (long long)s.batch, (long long)s.heads);
  if (s.heads > 0 && s.heads <= 65535 && s.batch * s.heads > 65535) s.batch = 1;      // (one CTA a head: more of them are taken here)
  if (int rc = check_decay_shape(&s)) return rc;
  const struct { const fnb_rows* t; const char* name; } big[] = {{&a->q, "q"}, {&a->k, "k"}, {&a->v, "v"}, {&a->out, "out"}};
  for (const auto& e : big)
    if (int rc = check_rows(*e.t, e.name, a->dtype)) return rc;
  if (!a->log_decay || !a->states) return fail(FNB_ERR_INVALID_ARGUMENT, "log_decay and states must not be NULL");
  if (int rc = check_words(a->log_decay, a->slots)) return rc;
  if (!aligned16(a->states)) return fail(FNB_ERR_INVALID_ARGUMENT, "states must be 16-byte aligned");
  if (a->num_states <= 0 || (!a->slots && a->num_states < a->batch))
    return fail(FNB_ERR_INVALID_ARGUMENT, "%lld states for %lld rows", (long long)a->num_states, (long long)a->batch);
  DeviceGuard g(a->device);
  if (!g.ok) return fail(FNB_ERR_CUDA, "cannot select CUDA device %d", a->device);
  int max_smem = 0, cc = 0, sms = 0;
  if (int rc = device_limits(a->device, &max_smem, &cc, &sms)) return rc;
  DecayStepParams p{a->q.data, a->k.data, a->v.data, a->out.data, a->q.stride_b, a->q.stride_h, a->k.stride_b, a->k.stride_h, a->v.stride_b,
                    a->v.stride_h, a->out.stride_b, a->out.stride_h, a->log_decay, a->states, a->slots, a->num_states, (int)a->batch,
                    (int)a->heads, a->scale};
  const int64_t BH = a->batch * a->heads;
  // a head's columns are split over CTAs (32 each) while that leaves SMs without work
  const bool narrow = a->head_dim > 32 && BH < 2 * sms;
  Launcher L((cudaStream_t)a->stream, a->device);
  return dispatch_decay(a->dtype, a->head_dim, [&](auto tag, auto d) -> int {
    using T = decltype(tag);
    constexpr int D = decltype(d)::value, NW = D > 32 ? 32 : D;
    constexpr int NTN = D * NW / 4 < 256 ? D * NW / 4 : 256, NTW = D * D / 4 < 256 ? D * D / 4 : 256;
    L.begin();
    if (narrow) decay_step_kernel<T, D, NW><<<dim3((unsigned)BH, D / NW), NTN, 0, L.stream>>>(p);
    else decay_step_kernel<T, D, D><<<dim3((unsigned)BH, 1), NTW, 0, L.stream>>>(p);
    return L.end("decay_step");
  });
}

int fnb_check_norm_shape(const fnb_norm_shape* shape) { return check_norm_shape(shape); }
size_t fnb_norm_workspace_bytes(const fnb_norm_shape* shape) { return check_norm_shape(shape) ? 0 : norm_ws_bytes(*shape); }

int fnb_norm_forward(const fnb_norm_fwd_args* a) {
  if (!a) return fail(FNB_ERR_INVALID_ARGUMENT, "args is NULL");
  const fnb_norm_shape& s = a->shape;
  if (int rc = check_norm_shape(&s)) return rc;
  if (!a->x || !a->y) return fail(FNB_ERR_INVALID_ARGUMENT, "x and y must not be NULL");
  if (!typed(a->x, s.dtype) || !typed(a->y, s.dtype) || !typed(a->weight, s.param_dtype) || !typed(a->bias, s.param_dtype) ||
      !typed(a->mean, FNB_F32) || !typed(a->rstd, FNB_F32))
    return fail(FNB_ERR_INVALID_ARGUMENT, "a tensor is not aligned to its type");
  DeviceGuard g(a->device);
  if (!g.ok) return fail(FNB_ERR_CUDA, "cannot select CUDA device %d", a->device);
  int max_smem = 0, cc = 0, sms = 0;
  if (int rc = device_limits(a->device, &max_smem, &cc, &sms)) return rc;
  const NormAlign at[2] = {norm_align(a->x, a->x_stride, s.dtype), norm_align(a->y, a->y_stride, s.dtype)};
  const NormPlan n = norm_plan(s, norm_loads(s, at, 2, aligned16(a->weight) && aligned16(a->bias)), false, sms);
  NormParams p = norm_params(s, n);
  p.base_left = at[0].base; p.stride_left = at[0].stride;
  p.x = a->x; p.xs = a->x_stride; p.y = a->y; p.ys = a->y_stride; p.w = a->weight; p.b = a->bias; p.mean = a->mean; p.rstd = a->rstd;
  Launcher L((cudaStream_t)a->stream, a->device);
  return dispatch_norm(s, n, [&](auto tag, auto pf, auto vec, auto items, auto block, auto shift) -> int {
    L.begin();
    norm_fwd_kernel<decltype(tag), decltype(pf)::value, decltype(vec)::value, decltype(items)::value, decltype(block)::value, decltype(shift)::value>
        <<<n.ctas, n.threads, 0, L.stream>>>(p);
    return L.end("norm_fwd");
  });
}

int fnb_norm_backward(const fnb_norm_bwd_args* a) {
  if (!a) return fail(FNB_ERR_INVALID_ARGUMENT, "args is NULL");
  const fnb_norm_shape& s = a->shape;
  if (int rc = check_norm_shape(&s)) return rc;
  if (!a->x || !a->d_y || !a->mean || !a->rstd) return fail(FNB_ERR_INVALID_ARGUMENT, "x, d_y, mean and rstd must not be NULL");
  if (!typed(a->x, s.dtype) || !typed(a->d_y, s.dtype) || !typed(a->d_x, s.dtype) || !typed(a->weight, s.param_dtype) ||
      !typed(a->d_weight, s.param_dtype) || !typed(a->d_bias, s.param_dtype) || !typed(a->mean, FNB_F32) || !typed(a->rstd, FNB_F32))
    return fail(FNB_ERR_INVALID_ARGUMENT, "a tensor is not aligned to its type");
  DeviceGuard g(a->device);
  if (!g.ok) return fail(FNB_ERR_CUDA, "cannot select CUDA device %d", a->device);
  int max_smem = 0, cc = 0, sms = 0;
  if (int rc = device_limits(a->device, &max_smem, &cc, &sms)) return rc;
  const bool sums = a->d_weight || a->d_bias;
  if (!sums && !a->d_x) return 0;
  const size_t need = norm_ws_bytes(s);
  if (sums && (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace)))
    return fail(FNB_ERR_WORKSPACE, "workspace must be 16-byte aligned and >= %zu bytes (got %zu)", need, a->workspace_bytes);
  const NormAlign at[3] = {norm_align(a->x, a->x_stride, s.dtype), norm_align(a->d_y, a->d_y_stride, s.dtype), norm_align(a->d_x, a->d_x_stride, s.dtype)};
  const NormPlan n = norm_plan(s, norm_loads(s, at, a->d_x ? 3 : 2, aligned16(a->weight)), true, sms);
  NormParams p = norm_params(s, n);
  p.base_left = at[0].base; p.stride_left = at[0].stride;
  p.x = a->x; p.xs = a->x_stride; p.dy = a->d_y; p.dys = a->d_y_stride; p.y = a->d_x; p.ys = a->d_x_stride; p.w = a->weight;
  p.mean = const_cast<float*>(a->mean); p.rstd = const_cast<float*>(a->rstd);
  p.part = sums ? (float*)a->workspace : nullptr;
  const size_t smem = sums && !n.block ? (size_t)2 * n.span * norm_copies(n.lanes, n.per_row) * sizeof(float) : 0;
  Launcher L((cudaStream_t)a->stream, a->device);
  int rc = dispatch_norm(s, n, [&](auto tag, auto pf, auto vec, auto items, auto block, auto shift) -> int {
    auto kern = norm_bwd_kernel<decltype(tag), decltype(pf)::value, decltype(vec)::value, decltype(items)::value, decltype(block)::value, decltype(shift)::value>;
    if (smem > 32768)
      if (int e = set_smem(kern, smem, max_smem, "norm_bwd")) return e;
    L.begin();
    kern<<<n.ctas, n.threads, smem, L.stream>>>(p);
    return L.end("norm_bwd");
  });
  if (rc || !sums) return rc;
  auto reduce = [&](auto tag) -> int {
    using P = decltype(tag);
    L.begin();
    FNB_CUDA(launch_pdl(norm_reduce_kernel<P>, dim3((unsigned)((s.cols + 31) / 32), 2), dim3(1024), 0, L.stream, (const float*)p.part, (P*)a->d_weight,
                        (P*)a->d_bias, s.cols, p.n, n.per_row, n.gblocks, n.ctas, n.span));
    return L.end("norm_reduce");
  };
  switch (s.param_dtype) {
    case FNB_F32: return reduce(float{});
    case FNB_F16: return reduce(__half{});
    default: return reduce(__nv_bfloat16{});
  }
}

}  // extern "C"
