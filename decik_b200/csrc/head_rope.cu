// The norm of each query and key head with the position rotation in the same pass, and the rotation
// by positions of several axes (time, height, width), forward and backward. For one head's row
// x = q (+ q_lora) of one token (D = head_dim, R = rotary_dim, j < R / 2):
//   r = rsqrt(mean(x^2) + eps),  y = x r w                      (without norms: y = x)
//   out[j] = y[j] cos[j] - y[j + R/2] sin[j],  out[j + R/2] = y[j + R/2] cos[j + R/2] + y[j] sin[j + R/2],
//   out[d] = y[d] for d >= R;
// backward, with g the transposed rotation of the gradient:
//   dw = sum over tokens and heads of g x r,  z = g w,  dx = r (z - x r^2 mean(z x)).
// The cosines come from fp32 tables [T, R] or, for several axes, from the token's positions:
// angle j = position[axis of j] * inv_freq[j].
//
// All arithmetic is fp32 with one rounding at the end. HBM-bound.
#include "common.cuh"

namespace decik {
namespace headrope {
namespace {

// where the angles come from: tables, or positions of up to four axes with the axis of each
// frequency in two bits
struct Angles {
  const float* cos;
  const float* sin;
  const void* pos;
  int pos32;
  int64_t ld_pos;
  const float* inv_freq;
  uint32_t axis[8];
};

struct Args {
  decik_tensor3 q, ql, k;          // forward inputs; in the backward the saved ones
  decik_tensor3 gq, gk;            // backward: gradients
  decik_tensor3_mut oq, ok;        // forward: outputs; backward: dq, dk
  const void* wq;
  const void* wk;
  float* part;                     // backward: [CTA][2][D] partial sums of the weight gradients
  Angles ang;
  int64_t n_tok;
  int hq, hk, D, R;
  float eps;
};

__device__ __forceinline__ float load_w(const void* w, int dtype, int i) {
  return dtype == DECIK_F32 ? __ldg(static_cast<const float*>(w) + i)
         : dtype == DECIK_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i])
                               : __half2float(static_cast<const __half*>(w)[i]);
}

// cos and sin of position * inv_freq, to fp32's last bits of the exact product's: the quarter turns
// are counted and taken off in 64 bits (a far position times a 24-bit frequency needs more than 32),
// so that what is rounded to fp32 is at most an eighth of a turn, exact relative to itself.
__device__ __forceinline__ void sincos_of(double pos, float inv_freq, float& s, float& c) {
  const double quarters = pos * static_cast<double>(inv_freq) * 0.63661977236758134;  // 2 / pi
  const double n = rint(quarters);
  const int quadrant = static_cast<int>(static_cast<long long>(n) & 3);
  float a, b;
  sincospif(0.5f * static_cast<float>(quarters - n), &a, &b);
  s = quadrant & 1 ? b : a;
  c = quadrant & 1 ? a : b;
  if (quadrant & 2) s = -s;
  if ((quadrant + 1) & 2) c = -c;
}

__device__ __forceinline__ double position(const Angles& a, int axis, int64_t t) {
  const int64_t i = axis * a.ld_pos + t;
  return a.pos32 ? static_cast<double>(__ldg(static_cast<const int*>(a.pos) + i))
                 : static_cast<double>(__ldg(static_cast<const long long*>(a.pos) + i));
}

// A row of D values is held by L lanes (the power of two at or above D / 16), 16 values each: lane c
// holds the 8 values from lo and the 8 from hi. Lanes below R / 16 hold rotation partners (hi = lo +
// R / 2), those below D / 16 the values behind R, the rest nothing.
struct Lane {
  int lo, hi;
  bool active, rot;
};
__device__ __forceinline__ Lane lane_of(int c, int D, int R) {
  Lane l;
  l.rot = 16 * c < R;
  l.active = 16 * c < D;
  l.lo = l.rot ? 8 * c : 16 * c;
  l.hi = l.rot ? R / 2 + 8 * c : 16 * c + 8;
  return l;
}

template <bool AXES>
__device__ __forceinline__ void load_angles(const Args& p, const Lane& l, int64_t t, float (&cl)[8], float (&ch)[8],
                                            float (&sl)[8], float (&sh)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cl[i] = ch[i] = 1.f;
    sl[i] = sh[i] = 0.f;
    if (!l.rot) continue;
    if constexpr (AXES) {
      const int j = l.lo + i;
      sincos_of(position(p.ang, (p.ang.axis[j >> 4] >> (2 * (j & 15))) & 3, t), __ldg(p.ang.inv_freq + j), sl[i], cl[i]);
      ch[i] = cl[i];
      sh[i] = sl[i];
    } else {
      cl[i] = __ldg(p.ang.cos + t * p.R + l.lo + i);
      ch[i] = __ldg(p.ang.cos + t * p.R + l.hi + i);
      sl[i] = __ldg(p.ang.sin + t * p.R + l.lo + i);
      sh[i] = __ldg(p.ang.sin + t * p.R + l.hi + i);
    }
  }
}

template <typename T>
__device__ __forceinline__ void load_row(const decik_tensor3& x, const Lane& l, int64_t t, int h, float (&lo)[8],
                                         float (&hi)[8]) {
  const T* p = static_cast<const T*>(x.ptr) + t * x.tok_stride + h * x.head_stride;
  unpack8<T>(ldg16(p + l.lo), lo);
  unpack8<T>(ldg16(p + l.hi), hi);
}
template <typename T>
__device__ __forceinline__ void store_row(const decik_tensor3_mut& x, const Lane& l, int64_t t, int h,
                                          const float (&lo)[8], const float (&hi)[8]) {
  T* p = static_cast<T*>(x.ptr) + t * x.tok_stride + h * x.head_stride;
  stg16(p + l.lo, pack8<T>(lo));
  stg16(p + l.hi, pack8<T>(hi));
}
// the row's x (with the LoRA delta of the queries added in fp32); zeros in lanes that hold nothing
template <typename T>
__device__ __forceinline__ void load_x(const Args& p, const Lane& l, int64_t t, int h, float (&lo)[8], float (&hi)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 0.f;
  if (!l.active) return;
  if (h >= p.hq) return load_row<T>(p.k, l, t, h - p.hq, lo, hi);
  load_row<T>(p.q, l, t, h, lo, hi);
  if (p.ql.ptr == nullptr) return;
  float a[8], b[8];
  load_row<T>(p.ql, l, t, h, a, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] += a[i];
    hi[i] += b[i];
  }
}

template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int L, bool NORM, bool AXES>
__global__ void __launch_bounds__(256) fwd_kernel(const Args p, int w_dtype) {
  const int heads = p.hq + p.hk;
  const int64_t rows = p.n_tok * heads, per_grid = static_cast<int64_t>(gridDim.x) * (256 / L);
  const Lane l = lane_of(threadIdx.x % L, p.D, p.R);
  // every lane of a warp takes every step: the row sums are warp shuffles
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  for (int64_t base = 0; base < rows; base += per_grid) {
    const int64_t row = base + first;
    const bool ok = row < rows && l.active;
    const int64_t t = ok ? row / heads : 0;
    const int h = ok ? static_cast<int>(row % heads) : 0;
    float lo[8], hi[8];
    load_x<T>(p, l, t, h, lo, hi);
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += lo[i] * lo[i] + hi[i] * hi[i];
      const float r = rsqrtf(row_sum<L>(ss) / p.D + p.eps);
      const void* w = h < p.hq ? p.wq : p.wk;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] *= r * (l.active ? load_w(w, w_dtype, l.lo + i) : 0.f);
        hi[i] *= r * (l.active ? load_w(w, w_dtype, l.hi + i) : 0.f);
      }
    }
    if (!ok) continue;
    float cl[8], ch[8], sl[8], sh[8], ol[8], oh[8];
    load_angles<AXES>(p, l, t, cl, ch, sl, sh);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ol[i] = lo[i] * cl[i] - hi[i] * sl[i];
      oh[i] = hi[i] * ch[i] + lo[i] * sh[i];
    }
    if (h < p.hq) store_row<T>(p.oq, l, t, h, ol, oh);
    else store_row<T>(p.ok, l, t, h - p.hq, ol, oh);
  }
}

// The weight gradients are summed in fp32: a thread's own rows (queries, then keys), then the CTA's
// threads that hold the same values, in shared memory, then the CTAs in a kernel of their own, all
// in a fixed order.
template <typename T, int L, bool NORM, bool AXES>
__global__ void __launch_bounds__(256) bwd_kernel(const Args p, int w_dtype) {
  __shared__ float red[NORM ? 256 * 17 : 1];
  const Lane l = lane_of(threadIdx.x % L, p.D, p.R);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  const int64_t per_grid = static_cast<int64_t>(gridDim.x) * (256 / L);
  for (int part = 0; part < 2; ++part) {  // queries, keys
    const int heads = part ? p.hk : p.hq;
    const int64_t rows = p.n_tok * heads;
    const void* w = part ? p.wk : p.wq;
    float dwl[8] = {}, dwh[8] = {};
    for (int64_t base = 0; base < rows; base += per_grid) {
      const int64_t row = base + first;
      const bool ok = row < rows && l.active;
      const int64_t t = ok ? row / heads : 0;
      const int h = ok ? static_cast<int>(row % heads) : 0;
      float gl[8], gh[8], cl[8], ch[8], sl[8], sh[8], zl[8], zh[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) gl[i] = gh[i] = 0.f;
      if (ok) load_row<T>(part ? p.gk : p.gq, l, t, h, gl, gh);
      load_angles<AXES>(p, l, t, cl, ch, sl, sh);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        zl[i] = gl[i] * cl[i] + gh[i] * sh[i];
        zh[i] = gh[i] * ch[i] - gl[i] * sl[i];
      }
      if constexpr (NORM) {
        float xl[8], xh[8];
        load_x<T>(p, l, t, part ? p.hq + h : h, xl, xh);
        float ss = 0.f, zx = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += xl[i] * xl[i] + xh[i] * xh[i];
        const float r = rsqrtf(row_sum<L>(ss) / p.D + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (ok) {
            dwl[i] += zl[i] * xl[i] * r;
            dwh[i] += zh[i] * xh[i] * r;
          }
          zl[i] *= l.active ? load_w(w, w_dtype, l.lo + i) : 0.f;
          zh[i] *= l.active ? load_w(w, w_dtype, l.hi + i) : 0.f;
          zx += zl[i] * xl[i] + zh[i] * xh[i];
        }
        const float m = r * r * row_sum<L>(zx) / p.D;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          zl[i] = r * (zl[i] - xl[i] * m);
          zh[i] = r * (zh[i] - xh[i] * m);
        }
      }
      if (ok) store_row<T>(part ? p.ok : p.oq, l, t, h, zl, zh);
    }
    if constexpr (NORM) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        red[threadIdx.x * 17 + i] = dwl[i];
        red[threadIdx.x * 17 + 8 + i] = dwh[i];
      }
      __syncthreads();
      if (threadIdx.x < 16 * L) {  // value i of lane c over the CTA's rows
        const int c = threadIdx.x / 16, i = threadIdx.x % 16;
        const Lane o = lane_of(c, p.D, p.R);
        float s = 0.f;
        for (int k = c; k < 256; k += L) s += red[k * 17 + i];
        if (o.active) p.part[(2 * static_cast<int64_t>(blockIdx.x) + part) * p.D + (i < 8 ? o.lo + i : o.hi + i - 8)] = s;
      }
    }
  }
}

// dw[d] = the sum of the CTAs' partials, in CTA order
__global__ void __launch_bounds__(256) dw_sum_kernel(const float* __restrict__ part, float* __restrict__ dwq,
                                                     float* __restrict__ dwk, int n_part, int D) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= 2 * D) return;
  float s = 0.f;
  for (int c = 0; c < n_part; ++c) s += part[static_cast<int64_t>(c) * 2 * D + i];
  (i < D ? dwq : dwk)[i < D ? i : i - D] = s;
}

int lanes_of(int D) {
  int l = 1;
  while (16 * l < D) l *= 2;
  return l;
}

constexpr int kMaxPart = 2048;  // CTAs of a backward pass with norms

int grid_of(int64_t rows, int D, int per_sm) {
  const int64_t want = (rows * lanes_of(D) + 255) / 256, cap = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<int>(want < 1 ? 1 : want < cap ? want : cap);
}

template <typename T, int L, bool BWD>
int launch_l(const Args& p, bool norm, bool axes, int w_dtype, int grid, cudaStream_t s) {
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(p, w_dtype); };
  if constexpr (BWD) {
    if (norm) axes ? go(bwd_kernel<T, L, true, true>) : go(bwd_kernel<T, L, true, false>);
    else go(bwd_kernel<T, L, false, true>);
  } else {
    if (norm) axes ? go(fwd_kernel<T, L, true, true>) : go(fwd_kernel<T, L, true, false>);
    else go(fwd_kernel<T, L, false, true>);
  }
  return check_launch(BWD ? "head_rope_bwd" : "head_rope_fwd");
}

template <typename T, bool BWD>
int launch(const Args& p, bool norm, bool axes, int w_dtype, int grid, cudaStream_t s) {
  switch (lanes_of(p.D)) {
    case 1: return launch_l<T, 1, BWD>(p, norm, axes, w_dtype, grid, s);
    case 2: return launch_l<T, 2, BWD>(p, norm, axes, w_dtype, grid, s);
    case 4: return launch_l<T, 4, BWD>(p, norm, axes, w_dtype, grid, s);
    case 8: return launch_l<T, 8, BWD>(p, norm, axes, w_dtype, grid, s);
    default: return launch_l<T, 16, BWD>(p, norm, axes, w_dtype, grid, s);
  }
}

bool view_ok(const void* ptr, int64_t ts, int64_t hs) { return ptr && aligned16(ptr) && ts % 8 == 0 && hs % 8 == 0; }

int check(const char* what, const Args& p, bool norm, bool bwd, int w_dtype, int dtype) {
  if (p.n_tok < 0 || p.n_tok > (int64_t(1) << 31) - 1 || p.hq <= 0 || p.hk <= 0 || p.D <= 0 || p.D % 16 != 0 ||
      p.D > 256 || p.R <= 0 || p.R % 16 != 0 || p.R > p.D)
    return set_error(DECIK_ERR_INVALID, "%s: T=%lld, heads %d/%d, head_dim %d, rotary_dim %d (multiples of 16, "
                     "rotary_dim <= head_dim <= 256)", what, (long long)p.n_tok, p.hq, p.hk, p.D, p.R);
  if (dtype != DECIK_F16 && dtype != DECIK_BF16)
    return set_error(DECIK_ERR_INVALID, "%s: dtype %d is not F16/BF16", what, dtype);
  if ((p.wq == nullptr) != (p.wk == nullptr))
    return set_error(DECIK_ERR_INVALID, "%s: norm weights for both queries and keys, or for neither", what);
  if (norm && ((w_dtype != DECIK_F32 && w_dtype != DECIK_F16 && w_dtype != DECIK_BF16) || !(p.eps >= 0.f)))
    return set_error(DECIK_ERR_INVALID, "%s: norm weights of dtype %d (F32, F16 or BF16), eps %g", what, w_dtype,
                     static_cast<double>(p.eps));
  if (p.n_tok == 0) return DECIK_OK;
  bool ok = view_ok(p.oq.ptr, p.oq.tok_stride, p.oq.head_stride) && view_ok(p.ok.ptr, p.ok.tok_stride, p.ok.head_stride);
  if (!bwd || norm)
    ok = ok && view_ok(p.q.ptr, p.q.tok_stride, p.q.head_stride) && view_ok(p.k.ptr, p.k.tok_stride, p.k.head_stride) &&
         (!p.ql.ptr || view_ok(p.ql.ptr, p.ql.tok_stride, p.ql.head_stride));
  if (bwd)
    ok = ok && view_ok(p.gq.ptr, p.gq.tok_stride, p.gq.head_stride) &&
         view_ok(p.gk.ptr, p.gk.tok_stride, p.gk.head_stride);
  if (!ok) return set_error(DECIK_ERR_INVALID, "%s: a view is NULL, or its pointer or strides are not 16-byte aligned", what);
  return DECIK_OK;
}

int set_tables(const char* what, Args& p, const float* cos, const float* sin) {
  if (p.n_tok != 0 && (!cos || !sin || !aligned16(cos) || !aligned16(sin)))
    return set_error(DECIK_ERR_INVALID, "%s: cos / sin NULL or not 16-byte aligned", what);
  p.ang.cos = cos;
  p.ang.sin = sin;
  return DECIK_OK;
}

int set_axes(const char* what, Args& p, const void* positions, int pos_dtype, int64_t ld_pos, int n_axes,
             const float* inv_freq, const uint8_t* axis_of) {
  if (n_axes < 1 || n_axes > 4 || (pos_dtype != 0 && pos_dtype != 1))
    return set_error(DECIK_ERR_INVALID, "%s: %d axes (1 to 4), position dtype %d (0 = int64, 1 = int32)", what, n_axes,
                     pos_dtype);
  if (!axis_of || (p.n_tok != 0 && (!positions || !inv_freq)) || (n_axes > 1 && ld_pos < p.n_tok))
    return set_error(DECIK_ERR_INVALID, "%s: null pointer, or rows of positions shorter than the tokens", what);
  p.ang.pos = positions;
  p.ang.pos32 = pos_dtype;
  p.ang.ld_pos = ld_pos;
  p.ang.inv_freq = inv_freq;
  for (int j = 0; j < 8; ++j) p.ang.axis[j] = 0;
  for (int j = 0; j < p.R / 2; ++j) {
    if (axis_of[j] >= n_axes)
      return set_error(DECIK_ERR_INVALID, "%s: frequency %d has axis %d of %d", what, j, axis_of[j], n_axes);
    p.ang.axis[j >> 4] |= static_cast<uint32_t>(axis_of[j]) << (2 * (j & 15));
  }
  return DECIK_OK;
}

int run_fwd(const char* what, const Args& p, bool axes, int w_dtype, int dtype, cudaStream_t s) {
  if (int rc = check(what, p, p.wq != nullptr, false, w_dtype, dtype)) return rc;
  if (p.n_tok == 0) return DECIK_OK;
  const int grid = grid_of(p.n_tok * (p.hq + p.hk), p.D, 16);
  return DECIK_DISPATCH_16(dtype, [&] { return launch<T, false>(p, p.wq != nullptr, axes, w_dtype, grid, s); });
}

int run_bwd(const char* what, Args p, bool axes, int w_dtype, float* dwq, float* dwk, void* workspace, int dtype,
            cudaStream_t s) {
  const bool norm = p.wq != nullptr;
  if (int rc = check(what, p, norm, true, w_dtype, dtype)) return rc;
  if (norm && (!dwq || !dwk)) return set_error(DECIK_ERR_INVALID, "%s: dq_weight or dk_weight NULL", what);
  if (p.n_tok == 0) {
    cudaError_t e = cudaSuccess;
    if (norm) e = cudaMemsetAsync(dwq, 0, sizeof(float) * p.D, s);
    if (norm && e == cudaSuccess) e = cudaMemsetAsync(dwk, 0, sizeof(float) * p.D, s);
    return e == cudaSuccess ? DECIK_OK : set_error(DECIK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  if (norm && (!workspace || !aligned16(workspace)))
    return set_error(DECIK_ERR_INVALID, "%s: workspace NULL or not 16-byte aligned", what);
  p.part = static_cast<float*>(workspace);
  int grid = grid_of(p.n_tok * p.hq, p.D, 4);
  if (grid > kMaxPart) grid = kMaxPart;
  if (int rc = DECIK_DISPATCH_16(dtype, [&] { return launch<T, true>(p, norm, axes, w_dtype, grid, s); })) return rc;
  if (!norm) return DECIK_OK;
  dw_sum_kernel<<<(2 * p.D + 255) / 256, 256, 0, s>>>(p.part, dwq, dwk, grid, p.D);
  return check_launch(what);
}

}  // namespace
}  // namespace headrope
}  // namespace decik

extern "C" int decik_qk_norm_rope_fwd(decik_tensor3 q, decik_tensor3 q_lora, decik_tensor3 k, const void* q_weight,
                                      const void* k_weight, int w_dtype, float eps, const float* cos, const float* sin,
                                      decik_tensor3_mut q_out, decik_tensor3_mut k_out, int64_t n_tok, int n_heads,
                                      int n_kv, int head_dim, int rotary_dim, int dtype, void* stream) {
  using namespace decik::headrope;
  Args p{q, q_lora, k, {}, {}, q_out, k_out, q_weight, k_weight, nullptr, {}, n_tok, n_heads, n_kv, head_dim,
         rotary_dim, eps};
  if (!q_weight || !k_weight) return decik::set_error(DECIK_ERR_INVALID, "qk_norm_rope_fwd: NULL norm weight");
  if (int rc = set_tables("qk_norm_rope_fwd", p, cos, sin)) return rc;
  return run_fwd("qk_norm_rope_fwd", p, false, w_dtype, dtype, decik::as_stream(stream));
}

extern "C" int decik_rope_axes_fwd(decik_tensor3 q, decik_tensor3 q_lora, decik_tensor3 k, const void* q_weight,
                                   const void* k_weight, int w_dtype, float eps, const void* positions, int pos_dtype,
                                   int64_t ld_pos, int n_axes, const float* inv_freq, const uint8_t* axis_of,
                                   decik_tensor3_mut q_out, decik_tensor3_mut k_out, int64_t n_tok, int n_heads,
                                   int n_kv, int head_dim, int rotary_dim, int dtype, void* stream) {
  using namespace decik::headrope;
  Args p{q, q_lora, k, {}, {}, q_out, k_out, q_weight, k_weight, nullptr, {}, n_tok, n_heads, n_kv, head_dim,
         rotary_dim, eps};
  if (int rc = check("rope_axes_fwd", p, q_weight != nullptr, false, w_dtype, dtype)) return rc;  // R before axis_of[R / 2]
  if (int rc = set_axes("rope_axes_fwd", p, positions, pos_dtype, ld_pos, n_axes, inv_freq, axis_of)) return rc;
  return run_fwd("rope_axes_fwd", p, true, w_dtype, dtype, decik::as_stream(stream));
}

extern "C" int64_t decik_qk_norm_rope_bwd_workspace(int head_dim) {
  return head_dim <= 0 ? 0 : static_cast<int64_t>(decik::headrope::kMaxPart) * 2 * head_dim * sizeof(float);
}

extern "C" int decik_qk_norm_rope_bwd(decik_tensor3 grad_q, decik_tensor3 grad_k, decik_tensor3 q, decik_tensor3 q_lora,
                                      decik_tensor3 k, const void* q_weight, const void* k_weight, int w_dtype,
                                      float eps, const float* cos, const float* sin, decik_tensor3_mut dq,
                                      decik_tensor3_mut dk, float* dq_weight, float* dk_weight, int64_t n_tok,
                                      int n_heads, int n_kv, int head_dim, int rotary_dim, int dtype, void* workspace,
                                      void* stream) {
  using namespace decik::headrope;
  Args p{q, q_lora, k, grad_q, grad_k, dq, dk, q_weight, k_weight, nullptr, {}, n_tok, n_heads, n_kv, head_dim,
         rotary_dim, eps};
  if (!q_weight || !k_weight) return decik::set_error(DECIK_ERR_INVALID, "qk_norm_rope_bwd: NULL norm weight");
  if (int rc = set_tables("qk_norm_rope_bwd", p, cos, sin)) return rc;
  return run_bwd("qk_norm_rope_bwd", p, false, w_dtype, dq_weight, dk_weight, workspace, dtype,
                 decik::as_stream(stream));
}

extern "C" int decik_rope_axes_bwd(decik_tensor3 grad_q, decik_tensor3 grad_k, decik_tensor3 q, decik_tensor3 q_lora,
                                   decik_tensor3 k, const void* q_weight, const void* k_weight, int w_dtype, float eps,
                                   const void* positions, int pos_dtype, int64_t ld_pos, int n_axes,
                                   const float* inv_freq, const uint8_t* axis_of, decik_tensor3_mut dq,
                                   decik_tensor3_mut dk, float* dq_weight, float* dk_weight, int64_t n_tok,
                                   int n_heads, int n_kv, int head_dim, int rotary_dim, int dtype, void* workspace,
                                   void* stream) {
  using namespace decik::headrope;
  Args p{q, q_lora, k, grad_q, grad_k, dq, dk, q_weight, k_weight, nullptr, {}, n_tok, n_heads, n_kv, head_dim,
         rotary_dim, eps};
  if (int rc = check("rope_axes_bwd", p, q_weight != nullptr, true, w_dtype, dtype)) return rc;
  if (int rc = set_axes("rope_axes_bwd", p, positions, pos_dtype, ld_pos, n_axes, inv_freq, axis_of)) return rc;
  return run_bwd("rope_axes_bwd", p, true, w_dtype, dq_weight, dk_weight, workspace, dtype,
                 decik::as_stream(stream));
}
