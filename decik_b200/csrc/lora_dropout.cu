// The LoRA down projections of one input under counter-based dropout (philox.cuh), one mask for each
// branch, and their backward pass. No mask and no masked copy of the input is ever written: the
// forward and the backward compute the same mask bits from (seed, offset + stream + branch, index).
//   forward   x16 = dt(x),  u_b = dt(s_b (keep_b o x16) A_b^T)
//   backward  dx = addend + sum_b s_b keep_b o (du_b A_b),  dA_b = s_b du_b^T (keep_b o x16)
// The index of x[t, k] is t * width + k (width % 8 == 0: a group of 8 stays in one row).
#include "philox.cuh"
#include "ptx.cuh"

namespace decik {
namespace loradrop {
namespace {

constexpr int kMaxRank = 64;  // rows of A over all branches

struct Drop {  // per branch
  uint32_t cut[2];
  float scale[2];
};

// the kept values of a 16-bit pair v under the two lanes of one word of the generator
__device__ __forceinline__ uint32_t mask_pair(uint32_t w, uint32_t v, uint32_t cut) {
  const uint32_t m = ((w & 0xFFFFu) >= cut ? 0x0000FFFFu : 0u) | ((w >> 16) >= cut ? 0xFFFF0000u : 0u);
  return v & m;
}
__device__ __forceinline__ void mask8(const uint4& w, const uint4& v, uint32_t cut, uint32_t (&m)[4]) {
  m[0] = mask_pair(w.x, v.x, cut);
  m[1] = mask_pair(w.y, v.y, cut);
  m[2] = mask_pair(w.z, v.z, cut);
  m[3] = mask_pair(w.w, v.w, cut);
}

// 8 consecutive values of x as 16-bit pairs
template <typename T, typename X>
__device__ __forceinline__ uint4 load8(const X* p) {
  if constexpr (sizeof(X) == 2) {
    return ldg16(p);
  } else {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    return pack8<T>(f);
  }
}

// transpose of an 8 x 8 matrix of 16-bit values held by a warp (lane 4 i + c: row i, columns 2 c, 2 c + 1)
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// A CTA takes 16 MT rows; its 8 warps share out the width in blocks of 32 columns and their partial
// sums meet in shared memory. In a block, lane 4 g + c holds the 8 columns from 8 c of rows g and g + 8
// (of each 16): 32 bytes of x in one go, one call of the generator per row and branch, and, because
// the order of a sum's terms is free, an operand fragment of mma.sync m16n8k16 without any exchange:
// the instruction's columns 2 c, 2 c + 1 and 2 c + 8, 2 c + 9 of step s are the lane's pairs 2 s and
// 2 s + 1. lora_A's rows, read the same way (16 bytes of row g), are the other operand.
constexpr int kWarps = 8;

template <typename X, typename T, int NB, int NTB, int MT>
__global__ void __launch_bounds__(32 * kWarps, NB * NTB <= 4 ? 2 : 1)
down_kernel(const X* __restrict__ x, int64_t ldx, const T* __restrict__ a, int64_t lda, T* __restrict__ x16,
            int64_t ldx16, T* __restrict__ u, int64_t ldu, int64_t n_tok, int width, int rank, Drop d,
            const int64_t* __restrict__ rng, int64_t stream_id) {
  constexpr int NT = NB * NTB;            // n8 tiles of u's columns
  constexpr int LD = 8 * NT + 4;
  __shared__ float red[kWarps][16][LD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (16 * MT);
  philox::Key key[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) key[b] = philox::make_key(rng, stream_id + b);
  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int k = 32 * warp + 8 * c; k - 8 * c < width; k += 32 * kWarps) {
    const bool in = k < width;
    uint4 xv[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t t = t0 + 16 * m + 8 * h + g;
        xv[m][h] = in && t < n_tok ? load8<T>(x + t * ldx + k) : zero;
      }
    uint4 av[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * (n % NTB);
      av[n] = in && r < rank ? ldg16(a + static_cast<int64_t>(n / NTB * rank + r + g) * lda + k) : zero;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t t = t0 + 16 * m + 8 * h + g;
        if (x16 != nullptr && in && t < n_tok) stg16(x16 + t * ldx16 + k, xv[m][h]);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        uint32_t lo[4], hi[4];
        const unsigned long long group = static_cast<unsigned long long>(t0 + 16 * m + g) * (width / 8) + k / 8;
        mask8(philox::words(key[b], group), xv[m][0], d.cut[b], lo);
        mask8(philox::words(key[b], group + static_cast<unsigned long long>(width)), xv[m][1], d.cut[b], hi);
        const uint32_t f0[4] = {lo[0], hi[0], lo[1], hi[1]}, f1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
        for (int n = b * NTB; n < (b + 1) * NTB; ++n) {
          ptx::mma16816<T>(acc[m][n], f0, av[n].x, av[n].y);
          ptx::mma16816<T>(acc[m][n], f1, av[n].z, av[n].w);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m > 0) __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      *reinterpret_cast<float2*>(&red[warp][g][8 * n + 2 * c]) = make_float2(acc[m][n][0], acc[m][n][1]);
      *reinterpret_cast<float2*>(&red[warp][g + 8][8 * n + 2 * c]) = make_float2(acc[m][n][2], acc[m][n][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 4 * NT; i += 32 * kWarps) {  // a pair of u's columns
      const int row = i / (4 * NT), col = 2 * (i % (4 * NT)), b = col / (8 * NTB), r = col % (8 * NTB);
      const int64_t t = t0 + 16 * m + row;
      if (t >= n_tok || r >= rank) continue;
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 v = *reinterpret_cast<const float2*>(&red[w][row][col]);
        s.x += v.x;
        s.y += v.y;
      }
      const float scale = NB == 2 && b == 1 ? d.scale[1] : d.scale[0];
      *reinterpret_cast<uint32_t*>(u + t * ldu + b * rank + r) = Dt<T>::pack2(s.x * scale, s.y * scale);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
// One pass gives dx and the partial dA: both need the same masks, and x16, the addend and dx are read
// or written once. A warp owns 32 columns and walks over its chunk of tokens in tiles of 16, with dA's
// 32 columns in its accumulators. Lane 4 g + c holds the 8 columns from 8 c of tokens g and g + 8, as in
// the forward. With the columns of an n8 tile j numbered n <-> 8 (n / 2) + 2 j + n % 2, both products fit
// these registers:
//   P = du A (m = token, k = rank): the accumulators of tiles 0..3 are the lane's own 8 columns, so mask,
//       scale and addend are applied in place and dx leaves in 16-byte pieces;
//   dA += du^T (keep x) (m = rank, k = token): the masked pair j of the lanes, as an 8 x 8 matrix
//       (token, column), transposed by movmatrix is the operand fragment of tile j.
template <typename T, int NB, int KR>
__global__ void __launch_bounds__(128, NB * KR <= 2 ? 4 : 2)
bwd_kernel(const T* __restrict__ du, int64_t ld_du, const T* __restrict__ x16, int64_t ldx, const T* __restrict__ a,
           int64_t lda, const float* addend, int64_t ld_add, float* dx, int64_t ld_dx, float* __restrict__ part,
           int64_t n_tok, int width, int rank, int chunk, int col_blocks, int n_units, Drop d,
           const int64_t* __restrict__ rng, int64_t stream_id) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 5);  // (token chunk, block of 32 columns)
  if (unit >= n_units) return;
  const int cb = unit % col_blocks;
  const int64_t first = static_cast<int64_t>(unit / col_blocks) * chunk;
  const int64_t last = first + chunk < n_tok ? first + chunk : n_tok;
  const int k = 32 * cb + 8 * c;
  const bool in = k < width;
  philox::Key key[NB];
  uint32_t af[NB][KR][4][2];   // A as P's operand: rows (rank) 2 c, 2 c + 1 (+ 8) of column n = g of tile j
  float acc[NB][KR][4][4];     // dA
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    key[b] = philox::make_key(rng, stream_id + b);
#pragma unroll
    for (int r = 0; r < KR; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = 32 * cb + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = 16 * r + 8 * h + 2 * c;
          uint32_t v = 0u;
          if (col < width && row < rank) {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(a + static_cast<int64_t>(b * rank + row) * lda + col);
            v = static_cast<uint32_t>(p[0]) | static_cast<uint32_t>(p[lda]) << 16;
          }
          af[b][r][j][h] = v;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[b][r][j][e] = 0.f;
      }
  }
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t t0 = first; t0 < last; t0 += 16) {
    const int64_t t[2] = {t0 + g, t0 + g + 8};
    const bool ok[2] = {t[0] < last, t[1] < last};
    uint4 xv[2];
    float out[2][8];
    uint32_t df[NB][KR][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      xv[h] = ok[h] && in ? ldg16(x16 + t[h] * ldx + k) : zero;
      float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
      if (addend != nullptr && ok[h] && in) {
        lo = *reinterpret_cast<const float4*>(addend + t[h] * ld_add + k);
        hi = *reinterpret_cast<const float4*>(addend + t[h] * ld_add + k + 4);
      }
      out[h][0] = lo.x, out[h][1] = lo.y, out[h][2] = lo.z, out[h][3] = lo.w;
      out[h][4] = hi.x, out[h][5] = hi.y, out[h][6] = hi.z, out[h][7] = hi.w;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < KR; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // (tokens g | g + 8, ranks 2 c .. | 2 c + 8 ..)
          const int h = q & 1, row = 16 * r + 8 * (q >> 1) + 2 * c;
          df[b][r][q] = ok[h] && row < rank
                            ? __ldg(reinterpret_cast<const unsigned int*>(du + t[h] * ld_du + b * rank + row)) : 0u;
        }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t m[2][4];
      float p[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[j][e] = 0.f;
#pragma unroll
        for (int r = 0; r < KR; ++r) ptx::mma16816<T>(p[j], df[b][r], af[b][r][j][0], af[b][r][j][1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 w = philox::words(key[b], static_cast<unsigned long long>(t[h]) * (width / 8) + k / 8);
        mask8(w, xv[h], d.cut[b], m[h]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (philox::keep_lane(w, i, d.cut[b])) out[h][i] += d.scale[b] * p[i >> 1][2 * h + (i & 1)];
      }
      uint32_t bf[4][2];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) bf[j][h] = transpose8x8(m[h][j]);
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        const uint32_t dt[4] = {transpose8x8(df[b][r][0]), transpose8x8(df[b][r][2]), transpose8x8(df[b][r][1]),
                                transpose8x8(df[b][r][3])};
#pragma unroll
        for (int j = 0; j < 4; ++j) ptx::mma16816<T>(acc[b][r][j], dt, bf[j][0], bf[j][1]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (ok[h] && in) {
        float4* o = reinterpret_cast<float4*>(dx + t[h] * ld_dx + k);
        o[0] = make_float4(out[h][0], out[h][1], out[h][2], out[h][3]);
        o[1] = make_float4(out[h][4], out[h][5], out[h][6], out[h][7]);
      }
  }
  if (!in) return;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < KR; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 16 * r + 8 * h + g;
        if (row >= rank) continue;
        float4* o = reinterpret_cast<float4*>(
            part + (static_cast<int64_t>(unit / col_blocks) * NB * rank + b * rank + row) * width + k);
        o[0] = make_float4(acc[b][r][0][2 * h], acc[b][r][0][2 * h + 1], acc[b][r][1][2 * h], acc[b][r][1][2 * h + 1]);
        o[1] = make_float4(acc[b][r][2][2 * h], acc[b][r][2][2 * h + 1], acc[b][r][3][2 * h], acc[b][r][3][2 * h + 1]);
      }
}

// dA = scale * the sum of the chunks' partials, in chunk order (no atomics: the same bits every time)
__global__ void __launch_bounds__(128)
da_sum_kernel(const float* __restrict__ part, float* __restrict__ da, int n_chunks, int width, int rank, int branches,
              Drop d) {
  const int n4 = width / 4 * rank * branches, i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n4) return;
  const float4* p = reinterpret_cast<const float4*>(part) + i;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int c = 0; c < n_chunks; ++c) {
    const float4 v = __ldg(p + static_cast<int64_t>(c) * n4);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  const float scale = i / (width / 4) / rank == 1 ? d.scale[1] : d.scale[0];
  reinterpret_cast<float4*>(da)[i] = make_float4(scale * s.x, scale * s.y, scale * s.z, scale * s.w);
}

// The token chunks of a backward pass: enough (chunk, 32 columns) units to give every SM 16 warps, at
// most 1024 tokens each (dA's accumulators on the tensor cores truncate: a chain of at most 64 of
// their sums, then fp32 additions), at least one tile of 16.
struct Split {
  int chunk, n_chunks, col_blocks;
};
Split split_of(int64_t n_tok, int width) {
  Split s;
  s.col_blocks = (width + 31) / 32;
  const int64_t tiles = (n_tok + 15) / 16;
  int64_t want = (static_cast<int64_t>(sm_count()) * 16 + s.col_blocks - 1) / s.col_blocks;
  const int64_t least = (n_tok + 1023) / 1024;
  if (want < least) want = least;
  if (want > tiles) want = tiles;
  s.chunk = static_cast<int>((tiles + want - 1) / want * 16);
  s.n_chunks = static_cast<int>((n_tok + s.chunk - 1) / s.chunk);
  return s;
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

struct DownArgs {
  const void* x;
  int64_t ldx;
  const void* a;
  int64_t lda;
  void* x16;
  int64_t ldx16;
  void* u;
  int64_t ldu, n_tok;
  int width, rank;
  Drop d;
  const int64_t* rng;
  int64_t stream_id;
  cudaStream_t s;
};

template <typename X, typename T, int NB, int NTB>
int launch_down_t(const DownArgs& p) {
  auto go = [&](auto kernel, int rows) {
    kernel<<<static_cast<unsigned>((p.n_tok + rows - 1) / rows), 32 * kWarps, 0, p.s>>>(
        static_cast<const X*>(p.x), p.ldx, static_cast<const T*>(p.a), p.lda, static_cast<T*>(p.x16), p.ldx16,
        static_cast<T*>(p.u), p.ldu, p.n_tok, p.width, p.rank, p.d, p.rng, p.stream_id);
  };
  if (p.n_tok <= 32 * static_cast<int64_t>(sm_count())) go(down_kernel<X, T, NB, NTB, 1>, 16);
  else go(down_kernel<X, T, NB, NTB, 2>, 32);
  return check_launch("lora_down_dropout");
}

template <typename X, typename T>
int launch_down(const DownArgs& p, int branches) {
  if (branches == 2) return p.rank <= 16 ? launch_down_t<X, T, 2, 2>(p) : launch_down_t<X, T, 2, 4>(p);
  if (p.rank <= 16) return launch_down_t<X, T, 1, 2>(p);
  return p.rank <= 32 ? launch_down_t<X, T, 1, 4>(p) : launch_down_t<X, T, 1, 8>(p);
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
  const DownArgs p{x, ldx, a, lda, x16, ldx16, u, ldu, n_tok, width, rank, make_drop(p0, p1), rng, stream_id,
                   as_stream(stream)};
  return DECIK_DISPATCH_16(dtype, [&] {
    return x_dtype == DECIK_F32 ? launch_down<float, T>(p, n_branch) : launch_down<T, T>(p, n_branch);
  });
}

extern "C" int64_t decik_lora_down_dropout_bwd_workspace(int64_t n_tok, int width, int rank, int n_branch) {
  using namespace decik::loradrop;
  if (n_tok <= 0 || width <= 0 || rank <= 0 || n_branch <= 0) return 0;
  return split_of(n_tok, width).n_chunks * static_cast<int64_t>(sizeof(float)) * rank * n_branch * width;
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
  const Split sp = split_of(n_tok, width);
  const int n_units = sp.n_chunks * sp.col_blocks, n4 = width / 4 * rank * n_branch;
  float* part = static_cast<float*>(workspace);
  return DECIK_DISPATCH_16(dtype, [&] {
    auto go = [&](auto kernel) {
      kernel<<<(n_units + 3) / 4, 128, 0, s>>>(static_cast<const T*>(du), ld_du, static_cast<const T*>(x16), ldx,
                                               static_cast<const T*>(a), lda, addend, ld_add, dx, ld_dx, part, n_tok,
                                               width, rank, sp.chunk, sp.col_blocks, n_units, d, rng, stream_id);
    };
    const int kr = (rank + 15) / 16;
    if (n_branch == 2) kr == 1 ? go(bwd_kernel<T, 2, 1>) : go(bwd_kernel<T, 2, 2>);
    else if (kr == 1) go(bwd_kernel<T, 1, 1>);
    else kr == 2 ? go(bwd_kernel<T, 1, 2>) : go(bwd_kernel<T, 1, 4>);
    da_sum_kernel<<<(n4 + 127) / 128, 128, 0, s>>>(part, da, sp.n_chunks, width, rank, n_branch, d);
    return check_launch("lora_down_dropout_bwd");
  });
}
