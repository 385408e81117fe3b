// The LoRA down projections of one input under counter-based dropout (philox.cuh), one mask for each
// branch, and their backward pass. No mask and no masked copy of the input is ever written: the
// forward and the backward compute the same mask bits from (seed, offset + stream + branch, index).
//   forward   x16 = dt(x),  u_b = dt(s_b (keep_b o x16) A_b^T)
//   backward  dx = addend + sum_b s_b keep_b o (du_b A_b),  dA_b = s_b du_b^T (keep_b o x16)
// The index of x[t, k] is t * width + k (width % 8 == 0: a group of 8 stays in one row).
#include "philox.cuh"

namespace decik {
namespace loradrop {
namespace {

constexpr int kMaxRank = 64;  // rows of A over all branches

struct Drop {  // per branch
  uint32_t cut[2];
  float scale[2];
};

template <typename X> __device__ __forceinline__ float load1(const X* p) { return Dt<X>::to_f(*p); }
template <> __device__ __forceinline__ float load1<float>(const float* p) { return *p; }

// One CTA per row: the masked 16-bit row of each branch in turn, then one warp per row of A.
template <typename X, typename T>
__global__ void __launch_bounds__(256)
down_kernel(const X* x, int64_t ldx, const T* __restrict__ a, int64_t lda, T* x16, int64_t ldx16, T* __restrict__ u,
            int64_t ldu, int width, int rank, int branches, Drop d, const int64_t* __restrict__ rng,
            int64_t stream_id) {
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int col = warp; col < rank * branches; col += 8) {
    const int b = col / rank;
    const philox::Key key = philox::make_key(rng, stream_id + b);
    float acc = 0.f;
    for (int g = lane; g < width / 8; g += 32) {
      const uint4 w = philox::words(key, static_cast<unsigned long long>(t) * (width / 8) + g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = 8 * g + j;
        if (philox::keep_lane(w, j, d.cut[b]))
          acc += Dt<T>::to_f(Dt<T>::from_f(load1(x + t * ldx + k))) * Dt<T>::to_f(a[col * lda + k]);
      }
    }
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) u[t * ldu + col] = Dt<T>::from_f(acc * d.scale[b]);
  }
  if (x16 != nullptr)
    for (int k = threadIdx.x; k < width; k += blockDim.x) x16[t * ldx16 + k] = Dt<T>::from_f(load1(x + t * ldx + k));
}

// One thread per group of 8 columns of one token.
template <typename T>
__global__ void __launch_bounds__(256)
dx_kernel(const T* __restrict__ du, int64_t ld_du, const T* __restrict__ a, int64_t lda, const float* addend,
          int64_t ld_add, float* dx, int64_t ld_dx, int64_t n_tok, int width, int rank, int branches, Drop d,
          const int64_t* __restrict__ rng, int64_t stream_id) {
  const int64_t gw = width / 8, total = n_tok * gw, stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += stride) {
    const int64_t t = i / gw;
    const int k = 8 * static_cast<int>(i % gw);
    float out[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = addend != nullptr ? addend[t * ld_add + k + j] : 0.f;
    for (int b = 0; b < branches; ++b) {
      const uint4 w = philox::words(philox::make_key(rng, stream_id + b), static_cast<unsigned long long>(i));
      float acc[8] = {};
      for (int r = b * rank; r < (b + 1) * rank; ++r) {
        const float g = Dt<T>::to_f(du[t * ld_du + r]);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += g * Dt<T>::to_f(a[r * lda + k + j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] += philox::keep_lane(w, j, d.cut[b]) ? d.scale[b] * acc[j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) dx[t * ld_dx + k + j] = out[j];
  }
}

constexpr int kChunk = 512;  // tokens of one partial sum of dA

// Partial dA of one token chunk (blockIdx.y): one thread per (row of A, group of 8 columns).
template <typename T>
__global__ void __launch_bounds__(256)
da_kernel(const T* __restrict__ du, int64_t ld_du, const T* __restrict__ x16, int64_t ldx, float* __restrict__ part,
          int64_t n_tok, int width, int rank, int branches, Drop d, const int64_t* __restrict__ rng,
          int64_t stream_id) {
  const int gw = width / 8, i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= gw * rank * branches) return;
  const int r = i / gw, g = i % gw, b = r / rank;
  const philox::Key key = philox::make_key(rng, stream_id + b);
  const int64_t t0 = static_cast<int64_t>(blockIdx.y) * kChunk, t1 = t0 + kChunk < n_tok ? t0 + kChunk : n_tok;
  float acc[8] = {};
  for (int64_t t = t0; t < t1; ++t) {
    const uint4 w = philox::words(key, static_cast<unsigned long long>(t) * gw + g);
    const float du_r = Dt<T>::to_f(du[t * ld_du + r]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (philox::keep_lane(w, j, d.cut[b])) acc[j] += du_r * Dt<T>::to_f(x16[t * ldx + 8 * g + j]);
  }
  float* p = part + (static_cast<int64_t>(blockIdx.y) * rank * branches + r) * width + 8 * g;
#pragma unroll
  for (int j = 0; j < 8; ++j) p[j] = acc[j];
}

// dA = scale * the sum of the chunks' partials, in chunk order (no atomics: the same bits every time)
__global__ void __launch_bounds__(256)
da_sum_kernel(const float* __restrict__ part, float* __restrict__ da, int n_chunks, int width, int rank, int branches,
              Drop d) {
  const int n = width * rank * branches, i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float acc = 0.f;
  for (int c = 0; c < n_chunks; ++c) acc += part[static_cast<int64_t>(c) * n + i];
  da[i] = d.scale[i / width / rank] * acc;
}

int check_sizes(const char* what, int64_t n_tok, int width, int rank, int branches, double p0, double p1, int dtype) {
  if (n_tok < 0 || n_tok > (int64_t(1) << 24) || width <= 0 || width % 8 != 0)
    return set_error(DECIK_ERR_INVALID, "%s: T=%lld, width %d (a positive multiple of 8)", what, (long long)n_tok,
                     width);
  if (branches < 1 || branches > 2 || rank <= 0 || rank % 8 != 0 || branches * ((rank + 15) / 16) * 16 > kMaxRank)
    return set_error(DECIK_ERR_UNSUPPORTED, "%s: %d branches of rank %d (1 or 2; multiples of 8; %d rows in all, each "
                     "branch rounded up to 16)", what, branches, rank, kMaxRank);
  if (!philox::valid_p(p0) || (branches > 1 && !philox::valid_p(p1)))
    return set_error(DECIK_ERR_INVALID, "%s: p=%g, %g are not in [0, 1]", what, p0, p1);
  if (dtype != DECIK_F16 && dtype != DECIK_BF16) return set_error(DECIK_ERR_INVALID, "%s: dtype %d is not F16/BF16",
                                                                  what, dtype);
  return DECIK_OK;
}

Drop make_drop(double p0, double p1) {
  Drop d;
  d.cut[0] = philox::cut_of(p0);
  d.cut[1] = philox::cut_of(p1);
  for (int b = 0; b < 2; ++b) d.scale[b] = philox::scale_of(d.cut[b]);
  return d;
}

}  // namespace
}  // namespace loradrop
}  // namespace decik

extern "C" int decik_lora_down_dropout(const void* x, int x_dtype, int64_t ldx, const void* a, int64_t lda, void* x16,
                                       int64_t ldx16, void* u, int64_t ldu, int64_t n_tok, int width, int rank,
                                       int n_branch, double p0, double p1, const int64_t* rng, int64_t stream_id,
                                       int dtype, void* stream) {
  using namespace decik;
  using namespace decik::loradrop;
  if (int rc = check_sizes("lora_down_dropout", n_tok, width, rank, n_branch, p0, p1, dtype)) return rc;
  if (x_dtype != DECIK_F32 && x_dtype != dtype)
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout: x of dtype %d (F32 or the compute dtype %d)", x_dtype, dtype);
  if (n_tok == 0) return DECIK_OK;
  if (!x || !a || !u || !rng) return set_error(DECIK_ERR_INVALID, "lora_down_dropout: null pointer");
  if (ldx < width || lda < width || (x16 && ldx16 < width) || ldu < rank * n_branch)
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout: row strides shorter than the rows");
  const int xe = x_dtype == DECIK_F32 ? 4 : 8;
  if (ldx % xe || lda % 8 || (x16 && ldx16 % 8) || ldu % 8 || !aligned16(x) || !aligned16(a) ||
      (x16 && !aligned16(x16)) || !aligned16(u))
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout: rows and pointers need 16-byte alignment");
  const Drop d = make_drop(p0, p1);
  cudaStream_t s = as_stream(stream);
  return DECIK_DISPATCH_16(dtype, [&] {
    if (x_dtype == DECIK_F32)
      down_kernel<float, T><<<static_cast<unsigned>(n_tok), 256, 0, s>>>(
          static_cast<const float*>(x), ldx, static_cast<const T*>(a), lda, static_cast<T*>(x16), ldx16,
          static_cast<T*>(u), ldu, width, rank, n_branch, d, rng, stream_id);
    else
      down_kernel<T, T><<<static_cast<unsigned>(n_tok), 256, 0, s>>>(
          static_cast<const T*>(x), ldx, static_cast<const T*>(a), lda, static_cast<T*>(x16), ldx16,
          static_cast<T*>(u), ldu, width, rank, n_branch, d, rng, stream_id);
    return check_launch("lora_down_dropout");
  });
}

extern "C" int64_t decik_lora_down_dropout_bwd_workspace(int64_t n_tok, int width, int rank, int n_branch) {
  using namespace decik::loradrop;
  if (n_tok <= 0 || width <= 0 || rank <= 0 || n_branch <= 0) return 0;
  return (n_tok + kChunk - 1) / kChunk * rank * n_branch * width * static_cast<int64_t>(sizeof(float));
}

extern "C" int decik_lora_down_dropout_bwd(const void* du, int64_t ld_du, const void* x16, int64_t ldx, const void* a,
                                           int64_t lda, const float* addend, int64_t ld_add, float* dx, int64_t ld_dx,
                                           float* da, int64_t n_tok, int width, int rank, int n_branch, double p0,
                                           double p1, const int64_t* rng, int64_t stream_id, int dtype,
                                           void* workspace, void* stream) {
  using namespace decik;
  using namespace decik::loradrop;
  if (int rc = check_sizes("lora_down_dropout_bwd", n_tok, width, rank, n_branch, p0, p1, dtype)) return rc;
  if (!da || !aligned16(da)) return set_error(DECIK_ERR_INVALID, "lora_down_dropout_bwd: da NULL or not 16-byte aligned");
  cudaStream_t s = as_stream(stream);
  if (n_tok == 0) {
    const cudaError_t e = cudaMemsetAsync(da, 0, sizeof(float) * rank * n_branch * width, s);
    return e == cudaSuccess ? DECIK_OK : set_error(DECIK_ERR_CUDA, "lora_down_dropout_bwd: %s", cudaGetErrorString(e));
  }
  if (!du || !x16 || !a || !dx || !rng || !workspace)
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout_bwd: null pointer");
  if (ld_du < rank * n_branch || ldx < width || lda < width || ld_dx < width || (addend && ld_add < width))
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout_bwd: row strides shorter than the rows");
  if (ld_du % 8 || ldx % 8 || lda % 8 || ld_dx % 4 || (addend && ld_add % 4) || !aligned16(du) || !aligned16(x16) ||
      !aligned16(a) || !aligned16(dx) || (addend && !aligned16(addend)) || !aligned16(workspace))
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout_bwd: rows and pointers need 16-byte alignment");
  const Drop d = make_drop(p0, p1);
  const int n_chunks = static_cast<int>((n_tok + kChunk - 1) / kChunk);
  const int64_t groups = n_tok * (width / 8);
  const int64_t want = (groups + 255) / 256, cap = static_cast<int64_t>(sm_count()) * 16;
  return DECIK_DISPATCH_16(dtype, [&] {
    dx_kernel<T><<<static_cast<int>(want < cap ? want : cap), 256, 0, s>>>(
        static_cast<const T*>(du), ld_du, static_cast<const T*>(a), lda, addend, ld_add, dx, ld_dx, n_tok, width, rank,
        n_branch, d, rng, stream_id);
    float* part = static_cast<float*>(workspace);
    const int n = rank * n_branch * width;
    da_kernel<T><<<dim3((n / 8 + 255) / 256, n_chunks), 256, 0, s>>>(static_cast<const T*>(du), ld_du,
                                                                     static_cast<const T*>(x16), ldx, part, n_tok,
                                                                     width, rank, n_branch, d, rng, stream_id);
    da_sum_kernel<<<(n + 255) / 256, 256, 0, s>>>(part, da, n_chunks, width, rank, n_branch, d);
    return check_launch("lora_down_dropout_bwd");
  });
}
