// The block norm's C entries, and the sums over rows of its gradient; the
// kernels of the rows, and what all of it computes, are in block_norm.cuh.
#include <string.h>

#include <initializer_list>

#include "block_norm.cuh"

namespace dgxm {

// The gradients of weights and modulations from the blocks' sums.
struct BlockNormSumParams {
  const float* partial;
  const char *gate, *scale, *norm_w, *norm_b, *branch_w;
  int64_t gate_sb, scale_sb;
  void *g_gate, *g_scale, *g_shift, *g_norm_w, *g_norm_b, *g_branch_w;
  int gate_form, mod_form;  // of the modulations
  int want, mod_dtype, weight_dtype;
  int batch, seq, width, rows_more;
  int64_t rows, rows_each;
};

__device__ __forceinline__ float bn_any(const char* base, int dtype, int col, float fill) {
  if (base == nullptr) return fill;
  if (dtype == DGXM_DTYPE_F32) return reinterpret_cast<const float*>(base)[col];
  if (dtype == DGXM_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[col]);
  return __half2float(reinterpret_cast<const __half*>(base)[col]);
}

__device__ __forceinline__ void bn_put(void* base, int dtype, int64_t at, float v) {
  if (base == nullptr) return;
  if (dtype == DGXM_DTYPE_F32) static_cast<float*>(base)[at] = v;
  else if (dtype == DGXM_DTYPE_BF16) static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(base)[at] = __float2half_rn(v);
}

constexpr int kBnSumWarps = 32;

// A block takes 32 columns.  Its warps form groups of equal size, up to one a
// sample; a group shares out the blocks with rows of a sample, and then takes
// another.  Sums of warps are added in order.
__global__ void __launch_bounds__(kBnSumWarps * 32) block_norm_sum_kernel(const __grid_constant__ BlockNormSumParams p) {
  __shared__ float part[kBnSumWarps][6][32];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * 32 + lane;
  const bool in = col < p.width;
  const float w = in ? bn_any(p.norm_w, p.weight_dtype, col, 1.f) : 0.f;
  const float bias = in ? bn_any(p.norm_b, p.weight_dtype, col, 0.f) : 0.f;
  const float w2 = in ? bn_any(p.branch_w, p.weight_dtype, col, 1.f) : 0.f;
  int groups = 1;
  while (groups < kBnSumWarps && groups < p.batch) groups *= 2;
  const int each = kBnSumWarps / groups, group = warp / each, turn = warp % each;
  float all[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // shift, scale, gate, norm_b, norm_w, branch_w over samples
  auto finish = [&](int b, const float (&s)[3], float up, float gate) {
    const float v[6] = {s[0], fmaf(w, s[1], bias * s[0]), w2 * s[2], up * s[0], up * s[1], gate * s[2]};
    if (in && p.mod_form == DGXM_MOD_SAMPLE) {
      bn_put(p.g_shift, p.mod_dtype, static_cast<int64_t>(b) * p.width + col, v[0]);
      bn_put(p.g_scale, p.mod_dtype, static_cast<int64_t>(b) * p.width + col, v[1]);
    }
    if (in && p.gate_form == DGXM_MOD_SAMPLE)
      bn_put(p.g_gate, p.mod_dtype, static_cast<int64_t>(b) * p.width + col, v[2]);
#pragma unroll
    for (int j = 0; j < 6; ++j) all[j] += v[j];
  };
  for (int64_t b0 = 0; b0 < p.batch; b0 += groups) {
    const bool there = b0 + group < p.batch;
    const int b = there ? static_cast<int>(b0) + group : 0;
    float s[3] = {0.f, 0.f, 0.f};
    const bool mine = in && there && turn == 0;
    const float up = !mine || p.scale == nullptr ? 1.f : 1.f + bn_any(p.scale + b * p.scale_sb, p.mod_dtype, col, 0.f);
    const float gate = !mine || p.gate == nullptr ? 1.f : bn_any(p.gate + b * p.gate_sb, p.mod_dtype, col, 0.f);
    // The blocks that hold rows of this sample.
    int64_t lo = 0, hi = 0;
    if (p.rows > 0 && there) {
      auto block = [&](int64_t row) -> int64_t {
        if (p.rows <= 0x7fffffff) {
          const uint32_t r = static_cast<uint32_t>(row), each = static_cast<uint32_t>(p.rows_each);
          const uint32_t more = p.rows_more, longer = more * (each + 1);
          return r < longer ? r / (each + 1) : more + (r - longer) / each;
        }
        const int64_t longer = p.rows_more * (p.rows_each + 1);
        return row < longer ? row / (p.rows_each + 1) : p.rows_more + (row - longer) / p.rows_each;
      };
      lo = block(static_cast<int64_t>(b) * p.seq);
      hi = block(static_cast<int64_t>(b) * p.seq + p.seq - 1) + 1;
    }
    const int64_t i0 = lo + (hi - lo) * turn / each, i1 = lo + (hi - lo) * (turn + 1) / each;
    if (in) {
      for (int64_t i = i0; i < i1; i += 4) {  // up to twelve loads under way
        float v[4][3];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float* from = p.partial + (min(i + u, i1 - 1) + b) * 3 * p.width + col;
#pragma unroll
          for (int j = 0; j < 3; ++j) v[u][j] = (p.want >> j & 1) && i + u < i1 ? from[j * p.width] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int j = 0; j < 3; ++j) s[j] += v[u][j];
      }
    }
    if (each > 1) {
#pragma unroll
      for (int j = 0; j < 3; ++j) part[warp][j][lane] = s[j];
      __syncthreads();
      if (turn == 0) {
#pragma unroll
        for (int j = 0; j < 3; ++j) s[j] = 0.f;
        for (int k = 0; k < each; ++k)
#pragma unroll
          for (int j = 0; j < 3; ++j) s[j] += part[warp + k][j][lane];
      }
      __syncthreads();
    }
    if (there && turn == 0) finish(b, s, up, gate);
  }
  if (groups > 1) {
#pragma unroll
    for (int j = 0; j < 6; ++j) part[warp][j][lane] = all[j];
    __syncthreads();
    if (warp == 0)
#pragma unroll
      for (int j = 0; j < 6; ++j) {
        all[j] = 0.f;
        for (int k = 0; k < groups; ++k) all[j] += part[k * each][j][lane];
      }
  }
  if (warp != 0 || !in) return;
  if (p.mod_form == DGXM_MOD_SHARED) {
    bn_put(p.g_shift, p.mod_dtype, col, all[0]);
    bn_put(p.g_scale, p.mod_dtype, col, all[1]);
  }
  if (p.gate_form == DGXM_MOD_SHARED) bn_put(p.g_gate, p.mod_dtype, col, all[2]);
  bn_put(p.g_norm_b, p.weight_dtype, col, all[3]);
  bn_put(p.g_norm_w, p.weight_dtype, col, all[4]);
  bn_put(p.g_branch_w, p.weight_dtype, col, all[5]);
}

static int bn_check(const dgxm_block_norm_desc* d) {
  if (d == nullptr) return fail(DGXM_ERR_INVALID, "NULL block norm descriptor");
  if (d->batch < 0 || d->seq < 0) return fail(DGXM_ERR_INVALID, "negative sizes (%d, %d)", d->batch, d->seq);
  if (d->width <= 0 || d->width > kBnMaxWidth)
    return fail(DGXM_ERR_UNSUPPORTED, "width %d (1 to %d)", d->width, kBnMaxWidth);
  if (d->dtype != DGXM_DTYPE_BF16 && d->dtype != DGXM_DTYPE_F16 && d->dtype != DGXM_DTYPE_F32)
    return fail(DGXM_ERR_UNSUPPORTED, "dtype %d (bf16, f16 or f32)", d->dtype);
  for (int t : {d->weight_dtype, d->mod_dtype})
    if (t != d->dtype && t != DGXM_DTYPE_F32)
      return fail(DGXM_ERR_UNSUPPORTED, "weight or modulation dtype %d (the tensors' or f32)", t);
  if (d->norm_mode != DGXM_BLOCK_NORM_NONE && d->norm_mode != DGXM_BLOCK_NORM_LAYER && d->norm_mode != DGXM_BLOCK_NORM_RMS)
    return fail(DGXM_ERR_UNSUPPORTED, "norm mode %d", d->norm_mode);
  for (int f : {d->gate_form, d->mod_form})
    if (f < DGXM_MOD_NONE || f > DGXM_MOD_TOKEN) return fail(DGXM_ERR_INVALID, "modulation form %d", f);
  if (!(d->eps >= 0.f)) return fail(DGXM_ERR_INVALID, "eps must not be negative or NaN");
  if (d->norm_mode == DGXM_BLOCK_NORM_NONE && d->mod_form != DGXM_MOD_NONE)
    return fail(DGXM_ERR_INVALID, "a scale or shift without a norm");
  return DGXM_OK;
}

// Samples of one row each are the rows of one sample: what serves a sample
// serves a token then, and comes with the rows instead of between them.
static const dgxm_block_norm_desc* bn_fold(const dgxm_block_norm_desc* d, dgxm_block_norm_desc* as) {
  if (d->seq != 1 || d->batch <= 1) return d;
  *as = *d;
  as->batch = 1;
  as->seq = d->batch;
  for (int64_t* stride : {as->x_stride, as->branch_stride, as->gate_stride, as->scale_stride, as->shift_stride, as->x_out_stride,
                          as->out_stride, as->dy_stride, as->dx_out_stride})
    stride[1] = stride[0];
  for (int* form : {&as->gate_form, &as->mod_form})
    if (*form == DGXM_MOD_SAMPLE) *form = DGXM_MOD_TOKEN;
  return as;
}

static int64_t bn_partial_bytes(const dgxm_block_norm_desc* d) {
  return (bn_cut<true>(d).blocks + static_cast<int64_t>(d->batch)) * 3 * d->width * 4;
}

// What both directions share of the parameters.
static void bn_common(const dgxm_block_norm_desc* d, BlockNormParams* p) {
  memset(p, 0, sizeof(*p));
  p->batch = d->batch;
  p->seq = d->seq;
  p->width = d->width;
  p->mode = d->norm_mode;
  p->branch_norm = d->branch_norm != 0;
  p->rows = bn_rows(d);
  p->eps = d->eps;
  p->inv_width = 1.f / d->width;
  p->mod_f32 = d->mod_dtype == DGXM_DTYPE_F32;
  p->w_f32 = d->weight_dtype == DGXM_DTYPE_F32;
}

static void bn_stream(BlockNormParams* p, int s, const void* base, const int64_t (&stride)[2], int dtype) {
  p->in[s] = static_cast<const char*>(base);
  p->in_sb[s] = stride[0] * bn_elt(dtype);
  p->in_sr[s] = stride[1] * bn_elt(dtype);
  p->in_elt[s] = bn_elt(dtype);
}

static int bn_aligned(std::initializer_list<const void*> ptrs, int elt, const char* what) {
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % elt) return fail(DGXM_ERR_INVALID, "%s not aligned to its elements", what);
  return DGXM_OK;
}

extern template int bn_launch<false, __nv_bfloat16>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);
extern template int bn_launch<false, __half>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);
extern template int bn_launch<false, float>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);
extern template int bn_launch<true, __nv_bfloat16>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);
extern template int bn_launch<true, __half>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);
extern template int bn_launch<true, float>(const dgxm_block_norm_desc*, BlockNormParams&, cudaStream_t);

template <bool BACK>
static int bn_run(const dgxm_block_norm_desc* d, BlockNormParams& p, cudaStream_t st) {
  if (d->dtype == DGXM_DTYPE_BF16) return bn_launch<BACK, __nv_bfloat16>(d, p, st);
  if (d->dtype == DGXM_DTYPE_F16) return bn_launch<BACK, __half>(d, p, st);
  return bn_launch<BACK, float>(d, p, st);
}

}  // namespace dgxm

extern "C" int dgxm_block_norm(const dgxm_block_norm_desc* d, const void* x, const void* branch, const void* gate,
                               const void* scale, const void* shift, const void* norm_w, const void* norm_b,
                               const void* branch_w, void* x_out, void* out, void* stream) {
  using namespace dgxm;
  if (int rc = bn_check(d)) return rc;
  dgxm_block_norm_desc folded;
  d = bn_fold(d, &folded);
  if (bn_rows(d) == 0) return DGXM_OK;  // empty tensors may be NULL
  const bool norm = d->norm_mode != DGXM_BLOCK_NORM_NONE;
  if ((branch == nullptr) != (x_out == nullptr)) return fail(DGXM_ERR_INVALID, "a branch and x_out come together");
  if (norm != (out != nullptr)) return fail(DGXM_ERR_INVALID, "out comes with a norm, and only then");
  if (!norm && branch == nullptr) return fail(DGXM_ERR_INVALID, "neither a norm nor a branch");
  if (branch == nullptr && (gate != nullptr || d->branch_norm || branch_w != nullptr))
    return fail(DGXM_ERR_INVALID, "a gate or a branch norm without a branch");
  if (branch_w != nullptr && !d->branch_norm) return fail(DGXM_ERR_INVALID, "branch_w without a branch norm");
  if (!norm && (norm_w != nullptr || norm_b != nullptr)) return fail(DGXM_ERR_INVALID, "norm weights without a norm");
  if (norm_b != nullptr && d->norm_mode == DGXM_BLOCK_NORM_RMS)
    return fail(DGXM_ERR_INVALID, "norm_b goes with the layer norm");
  if ((gate != nullptr) != (d->gate_form != DGXM_MOD_NONE)) return fail(DGXM_ERR_INVALID, "gate and gate_form do not match");
  if ((scale != nullptr || shift != nullptr) != (d->mod_form != DGXM_MOD_NONE))
    return fail(DGXM_ERR_INVALID, "scale, shift and mod_form do not match");
  if (x == nullptr) return fail(DGXM_ERR_INVALID, "NULL x");
  if (int rc = bn_aligned({x, branch, x_out, out}, bn_elt(d->dtype), "x, branch or an output is")) return rc;
  if (int rc = bn_aligned({gate, scale, shift}, bn_elt(d->mod_dtype), "a modulation is")) return rc;
  if (int rc = bn_aligned({norm_w, norm_b, branch_w}, bn_elt(d->weight_dtype), "a weight is")) return rc;
  BlockNormParams p;
  bn_common(d, &p);
  bn_stream(&p, kBnX, x, d->x_stride, d->dtype);
  bn_stream(&p, kBnBranch, branch, d->branch_stride, d->dtype);
  const int me = bn_elt(d->mod_dtype);
  if (d->gate_form == DGXM_MOD_TOKEN) {
    bn_stream(&p, kBnGate, gate, d->gate_stride, d->mod_dtype);
  } else if (gate != nullptr) {
    p.gate = static_cast<const char*>(gate);
    p.gate_sb = d->gate_form == DGXM_MOD_SAMPLE ? d->gate_stride[0] * me : 0;
  }
  if (d->mod_form == DGXM_MOD_TOKEN) {
    bn_stream(&p, kBnScale, scale, d->scale_stride, d->mod_dtype);
    bn_stream(&p, kBnShift, shift, d->shift_stride, d->mod_dtype);
  } else {
    p.scale = static_cast<const char*>(scale);
    p.shift = static_cast<const char*>(shift);
    p.scale_sb = d->mod_form == DGXM_MOD_SAMPLE ? d->scale_stride[0] * me : 0;
    p.shift_sb = d->mod_form == DGXM_MOD_SAMPLE ? d->shift_stride[0] * me : 0;
  }
  p.norm_w = static_cast<const char*>(norm_w);
  p.norm_b = static_cast<const char*>(norm_b);
  p.branch_w = static_cast<const char*>(branch_w);
  p.x_out = static_cast<char*>(x_out);
  p.out = static_cast<char*>(out);
  const int e = bn_elt(d->dtype);
  p.x_out_sb = d->x_out_stride[0] * e;
  p.x_out_sr = d->x_out_stride[1] * e;
  p.out_sb = d->out_stride[0] * e;
  p.out_sr = d->out_stride[1] * e;
  p.n_in = 5;
  return bn_run<false>(d, p, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t dgxm_block_norm_backward_workspace(const dgxm_block_norm_desc* d) {
  using namespace dgxm;
  if (bn_check(d)) return -1;
  dgxm_block_norm_desc folded;
  d = bn_fold(d, &folded);
  return bn_rows(d) == 0 ? 0 : bn_partial_bytes(d);
}

extern "C" int dgxm_block_norm_backward(const dgxm_block_norm_desc* d, const dgxm_block_norm_grads* g, const void* dy,
                                        const void* dx_out, const void* x_out, const void* branch, const void* gate,
                                        const void* scale, const void* norm_w, const void* norm_b, const void* branch_w,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace dgxm;
  if (int rc = bn_check(d)) return rc;
  if (g == nullptr) return fail(DGXM_ERR_INVALID, "NULL gradients");
  dgxm_block_norm_desc folded;
  d = bn_fold(d, &folded);
  const bool norm = d->norm_mode != DGXM_BLOCK_NORM_NONE;
  const int64_t rows = bn_rows(d);
  if (rows > 0) {  // empty tensors may be NULL
    if (norm && g->x == nullptr) return fail(DGXM_ERR_INVALID, "NULL gradient of x");
    if (branch == nullptr && (gate != nullptr || d->branch_norm || branch_w != nullptr || g->branch != nullptr ||
                              g->gate != nullptr || g->branch_w != nullptr))
      return fail(DGXM_ERR_INVALID, "a gate, a branch norm or their gradients without a branch");
    if ((branch_w != nullptr || g->branch_w != nullptr) && !d->branch_norm)
      return fail(DGXM_ERR_INVALID, "branch_w without a branch norm");
    if (!norm && (norm_w != nullptr || norm_b != nullptr || g->norm_w != nullptr || g->norm_b != nullptr))
      return fail(DGXM_ERR_INVALID, "norm weights without a norm");
    if ((norm_b != nullptr || g->norm_b != nullptr) && d->norm_mode == DGXM_BLOCK_NORM_RMS)
      return fail(DGXM_ERR_INVALID, "norm_b goes with the layer norm");
    if ((gate != nullptr) != (d->gate_form != DGXM_MOD_NONE) || (gate == nullptr && g->gate != nullptr))
      return fail(DGXM_ERR_INVALID, "gate, gate_form and the gate's gradient do not match");
    if (d->mod_form == DGXM_MOD_NONE && (scale != nullptr || g->scale != nullptr || g->shift != nullptr))
      return fail(DGXM_ERR_INVALID, "scale, shift and mod_form do not match");
    if (g->scale != nullptr && scale == nullptr) return fail(DGXM_ERR_INVALID, "the gradient of a scale without the scale");
  }
  const int me = bn_elt(d->mod_dtype), we = bn_elt(d->weight_dtype), e = bn_elt(d->dtype);
  if (int rc = bn_aligned({dy, dx_out, x_out, branch, g->x, g->branch}, e, "a tensor is")) return rc;
  if (int rc = bn_aligned({gate, scale, g->gate, g->scale, g->shift}, me, "a modulation is")) return rc;
  if (int rc = bn_aligned({norm_w, norm_b, branch_w, g->norm_w, g->norm_b, g->branch_w}, we, "a weight is")) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  BlockNormParams p;
  bn_common(d, &p);
  const bool tok_gate = d->gate_form == DGXM_MOD_TOKEN, tok_mod = d->mod_form == DGXM_MOD_TOKEN;
  const bool sum_shift = !tok_mod && g->shift != nullptr, sum_scale = !tok_mod && g->scale != nullptr;
  const bool sum_gate = !tok_gate && g->gate != nullptr;
  p.want = ((sum_shift || g->norm_b != nullptr || (sum_scale && norm_b != nullptr)) ? 1 : 0) |
           ((sum_scale || g->norm_w != nullptr) ? 2 : 0) | ((sum_gate || g->branch_w != nullptr) ? 4 : 0);
  int blocks = 0;
  if (rows > 0) {  // else the sums of nothing
    if (norm && (dy == nullptr || x_out == nullptr)) return fail(DGXM_ERR_INVALID, "NULL upstream gradient or x_out");
    if (!norm && dx_out == nullptr) return fail(DGXM_ERR_INVALID, "neither a norm nor an upstream gradient of x_out");
    if (p.want) {
      const int64_t need = bn_partial_bytes(d);
      if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 4 || workspace_bytes < need)
        return fail(DGXM_ERR_INVALID, "workspace of %lld bytes (%lld needed)", (long long)workspace_bytes, (long long)need);
      p.partial = static_cast<float*>(workspace);
    }
    bn_stream(&p, kBnDy, norm ? dy : nullptr, d->dy_stride, d->dtype);
    bn_stream(&p, kBnDr, dx_out, d->dx_out_stride, d->dtype);
    bn_stream(&p, kBnR, norm ? x_out : nullptr, d->x_stride, d->dtype);
    const bool apart = gate != nullptr || d->branch_norm;  // the branch's gradient is not the stream's
    if (apart) bn_stream(&p, kBnBranchB, branch, d->branch_stride, d->dtype);
    if (tok_gate) {
      bn_stream(&p, kBnGateB, gate, d->gate_stride, d->mod_dtype);
      p.g_gate = static_cast<char*>(g->gate);
    } else {
      p.gate = static_cast<const char*>(gate);
      p.gate_sb = d->gate_form == DGXM_MOD_SAMPLE ? d->gate_stride[0] * me : 0;
    }
    if (tok_mod) {
      if (scale != nullptr) bn_stream(&p, kBnScaleB, scale, d->scale_stride, d->mod_dtype);
      p.g_scale = static_cast<char*>(g->scale);
      p.g_shift = static_cast<char*>(g->shift);
    } else {
      p.scale = static_cast<const char*>(scale);
      p.scale_sb = d->mod_form == DGXM_MOD_SAMPLE ? d->scale_stride[0] * me : 0;
    }
    p.norm_w = static_cast<const char*>(norm_w);
    p.norm_b = static_cast<const char*>(norm_b);
    p.branch_w = static_cast<const char*>(branch_w);
    p.x_out = static_cast<char*>(g->x);
    p.out = apart ? static_cast<char*>(g->branch) : nullptr;
    p.x_out_sb = d->x_out_stride[0] * e;
    p.x_out_sr = d->x_out_stride[1] * e;
    p.out_sb = d->out_stride[0] * e;
    p.out_sr = d->out_stride[1] * e;
    if (!apart && g->branch != nullptr) return fail(DGXM_ERR_INVALID, "the branch's gradient is that of x: pass NULL");
    p.n_in = 6;
    blocks = bn_cut<true>(d).blocks;
    if (int rc = bn_run<true>(d, p, st)) return rc;
  }
  if (!p.want) return DGXM_OK;
  BlockNormSumParams sp;
  memset(&sp, 0, sizeof(sp));
  sp.partial = p.partial;
  sp.gate = tok_gate ? nullptr : static_cast<const char*>(gate);
  sp.scale = tok_mod ? nullptr : static_cast<const char*>(scale);
  sp.gate_sb = d->gate_form == DGXM_MOD_SAMPLE ? d->gate_stride[0] * me : 0;
  sp.scale_sb = d->mod_form == DGXM_MOD_SAMPLE ? d->scale_stride[0] * me : 0;
  sp.norm_w = static_cast<const char*>(norm_w);
  sp.norm_b = static_cast<const char*>(norm_b);
  sp.branch_w = static_cast<const char*>(branch_w);
  sp.g_gate = g->gate;
  sp.g_scale = g->scale;
  sp.g_shift = g->shift;
  sp.g_norm_w = g->norm_w;
  sp.g_norm_b = g->norm_b;
  sp.g_branch_w = g->branch_w;
  sp.gate_form = d->gate_form;
  sp.mod_form = d->mod_form;
  sp.want = p.want;
  sp.mod_dtype = d->mod_dtype;
  sp.weight_dtype = d->weight_dtype;
  sp.batch = d->batch;
  sp.seq = d->seq;
  sp.width = d->width;
  sp.rows = rows;
  if (blocks > 0) {
    sp.rows_each = rows / blocks;
    sp.rows_more = static_cast<int>(rows % blocks);
  }
  DGXM_CUDA_TRY(launch_overlapped(block_norm_sum_kernel, (d->width + 31) / 32, kBnSumWarps * 32, 0, st, sp));
  return DGXM_OK;
}
