// The LoRA down projections of one input under counter-based dropout (philox.cuh), one mask for each
// branch, and their backward pass. No mask and no masked copy of the input is ever written: the
// forward and the backward compute the same mask bits from (seed, offset + stream + branch, index).
//   forward   x16 = dt(x),  u_b = dt(s_b (keep_b o x16) A_b^T)
//   backward  dx = addend + sum_b s_b keep_b o (du_b A_b),  dA_b = s_b du_b^T (keep_b o x16)
// The index of x[t, k] is t * width + k (width % 8 == 0: a group of 8 stays in one row).
//
// At 16,384 x 1536, fp32 x, bf16, rank 16 x 2: forward 33.0 us (152 MB, 4.6 TB/s), backward 49.7 us (253 MB,
// 5.1 TB/s). The bytes alone would take 23.2 and 38.6 us. No unit is full: the generator's 14 products a call
// (50 M mask bits each way) keep the multipliers 64 % busy in the forward, the masks' logic the ALU 53 % in both,
// issue slots 59 and 58 %, DRAM 70 and 78 %; what is left is latency, with 16 and 14 warps an SM (the ring
// and the registers allow no more). mma.sync is far from its limit (rank 32: 10 and 13 %), so the tensor cores
// of the larger kind would change nothing. Ranks above 16 are further from the bytes: rank 32 x 2 takes 50.9 us
// forward and 65.1 backward (23.4 and 38.8), rank 64 44.1 and 58.7; 830 rows are 52 CTAs for 148 SMs.
#include <type_traits>

#include "philox.cuh"
#include "ptx.cuh"

namespace decik {
namespace loradrop {
namespace {

constexpr int kMaxRank = 64;  // rows of A over all branches

// per branch: a 16-bit lane of the generator is kept iff it is >= cut; a scale of 0 means that nothing is
// kept (p = 1, whose cut does not fit the lane)
struct Drop {
  uint32_t cut[2];    // in both halves of the word
  float scale[2];
  // 0xffff, 65536 and -1, as arguments: products with values that the compiler does not know stay products,
  // on the FMA pipe, where constants would become shifts and additions on the ALU pipe, the busiest here
  uint32_t ones, shift, minus;
};

// The kept values of a pair v of 16-bit values under one word of the generator, in 3 instructions of the ALU
// pipe and 2 products: max(w, cut) - w is 0 in the halves that are kept (no borrow crosses them), min with
// 1 makes that a bit, times 0xffff a mask.
__device__ __forceinline__ uint32_t mask_pair(uint32_t w, uint32_t v, uint32_t cut, const Drop& k) {
  uint32_t m, d;
  asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(w), "r"(cut));
  asm("min.u16x2 %0, %1, %2;" : "=r"(d) : "r"(w * k.minus + m), "r"(0x00010001u));
  return v & ~(d * k.ones);
}
__device__ __forceinline__ void mask8(const uint4& w, const uint4& v, uint32_t cut, const Drop& k, uint32_t (&m)[4]) {
  m[0] = mask_pair(w.x, v.x, cut, k);
  m[1] = mask_pair(w.y, v.y, cut, k);
  m[2] = mask_pair(w.z, v.z, cut, k);
  m[3] = mask_pair(w.w, v.w, cut, k);
}
// The same for a pair whose products are wanted too: v masked, and o0, o1 += scale * p0, p1 where kept. One
// compare serves a value's two uses, as the predicate of an fma and of an and.
__device__ __forceinline__ uint32_t mask_add_pair(uint32_t w, uint32_t v, uint32_t limit, uint32_t shift, float scale,
                                                  float p0, float p1, float& o0, float& o1) {
  asm("{\n\t.reg .pred l, h;\n\t.reg .b32 t;\n\t"
      "mul.lo.u32 t, %3, %5;\n\t"
      "setp.ge.u32 l, t, %4;\n\t"
      "setp.ge.u32 h, %3, %4;\n\t"
      "@l fma.rn.f32 %1, %6, %7, %1;\n\t"
      "@h fma.rn.f32 %2, %6, %8, %2;\n\t"
      "@!l and.b32 %0, %0, 0xffff0000;\n\t"
      "@!h and.b32 %0, %0, 0x0000ffff;\n\t}"
      : "+r"(v), "+f"(o0), "+f"(o1)
      : "r"(w), "r"(limit), "r"(shift), "f"(scale), "f"(p0), "f"(p1));
  return v;
}

// fp32 blocks of 32 columns in shared memory: row r's 16-byte piece q (of 8) at r * 128 + 16 (q ^ r % 8). They
// are copied a whole row by 8 lanes (whole 32-byte sectors; a lane fetching its own 32 bytes in two
// pieces asked L2 for every sector twice) and read back as two pieces 2 c, 2 c + 1 of row g without bank
// conflicts.
__device__ __forceinline__ uint32_t block_at(int r, int q) { return r * 128 + ((q ^ (r & 7)) * 16); }
__device__ __forceinline__ void block_read(const unsigned char* p, int r, int c, float (&f)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p + block_at(r, 2 * c));
  const float4 b = *reinterpret_cast<const float4*>(p + block_at(r, 2 * c + 1));
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// 8 fp32 values to global memory: one 32-byte store where the rows allow it
__device__ __forceinline__ void store32(float* p, const float (&f)[8], bool whole) {
  if (whole) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]),
                 "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                 : "memory");
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
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
// A CTA takes 16 rows; its 8 warps share out the width in blocks of 32 columns and their partial sums meet
// in shared memory. In a block, lane 4 g + c holds the 8 columns from 8 c of rows g and g + 8: one call of
// the generator per row and branch, and, because the order of a sum's terms is free, an operand fragment
// of mma.sync m16n8k16 without any exchange: the instruction's columns 2 c, 2 c + 1 and 2 c + 8, 2 c + 9
// of step s are the lane's pairs 2 s and 2 s + 1. lora_A's rows, read the same way (16 bytes of row g),
// are the other operand. The next kStages - 1 blocks' bytes are on their way through cp.async, into the
// warp's own ring, while one is computed.
// Measured at 16,384 x 1536: 8 warps and 3 stages 33.0 us, 2 stages 38.8, 4 stages (one CTA an SM) 41.0;
// 4 warps and 2 stages 34.3, 32 rows a CTA 37.8. At 830 rows 5.8 us with 8 warps, 7.2 with 4, 5.9 with 16.
constexpr int kWarps = 8, kStages = 3;

template <typename X, int NT>  // NT: n8 tiles of u's columns
struct DownTile {
  static constexpr int kXPieces = sizeof(X) / 2;                // 16-byte pieces of 8 columns
  static constexpr int kStage = (2 * kXPieces + NT) * 512;      // bytes of a warp's stage
  static constexpr int kLd = 8 * NT + 4;                        // row of the partial sums
  static constexpr int kRing = kStages * kWarps * kStage, kRed = kWarps * 16 * kLd * 4;
  static constexpr int kSmem = kRing > kRed ? kRing : kRed;
};

template <typename X, typename T, int NB, int NTB>
__global__ void __launch_bounds__(32 * kWarps, 2)
down_kernel(const X* __restrict__ x, int64_t ldx, const T* __restrict__ a, int64_t lda, T* __restrict__ x16,
            int64_t ldx16, T* __restrict__ u, int64_t ldu, int u_cols, int64_t n_tok, int width, int rank, Drop d,
            const int64_t* __restrict__ rng, int64_t stream_id) {
  constexpr int NT = NB * NTB;
  using Tile = DownTile<X, NT>;
  constexpr int XP = Tile::kXPieces, LD = Tile::kLd, kXBytes = 2 * XP * 512;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int rows = n_tok - t0 < 16 ? static_cast<int>(n_tok - t0) : 16;
  // The pieces of the block with its columns at k0, zeros behind the width. Rows that are not there (of x
  // behind the last token, of A behind the rank) are others read again: what comes of them is not stored.
  constexpr int XN = 2 * XP, XR = XP == 2 ? 4 : 8, XE = 16 / sizeof(X);  // a copy's pieces, rows, elements
  const int xr = XP == 2 ? lane >> 3 : g, xc = XP == 2 ? 4 * (lane & 7) : 8 * c;  // the lane's row and column
  const X* xp[XN];
  const T* ap[NT];
#pragma unroll
  for (int i = 0; i < XN; ++i) xp[i] = x + (t0 + (XR * i + xr < rows ? XR * i + xr : 0)) * ldx;
#pragma unroll
  for (int n = 0; n < NT; ++n)
    ap[n] = a + static_cast<int64_t>(8 * (n % NTB) < rank ? n / NTB * rank + 8 * (n % NTB) + g : 0) * lda;
  unsigned char* const ring = smem + warp * (kStages * Tile::kStage);  // x, then A: a lane's own piece n at 512 n + 16 lane
  const uint32_t ring_at = ptx::smem_u32(ring);
  auto issue = [&](int stage, int k0) {
    if (k0 < width) {
      const uint32_t dst = ring_at + stage * Tile::kStage;
      const bool xin = k0 + xc < width, ain = k0 + 8 * c < width;
      const int xk = xin ? k0 + xc : width - XE, ak = ain ? k0 + 8 * c : width - 8;
#pragma unroll
      for (int i = 0; i < XN; ++i)
        ptx::cp_async16(dst + (XP == 2 ? block_at(XR * i + xr, lane & 7) : i * 512 + lane * 16), xp[i] + xk, xin);
#pragma unroll
      for (int n = 0; n < NT; ++n) ptx::cp_async16(dst + kXBytes + n * 512 + lane * 16, ap[n] + ak, ain);
    }
    ptx::cp_async_commit();
  };
  constexpr int kStep = 32 * kWarps;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s, 32 * warp + s * kStep);
  const philox::Key key = philox::make_key(rng);
  philox::Stream ctr[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) ctr[b] = philox::make_stream(rng, stream_id + b);
  float acc[NT][4] = {};
  T* const x16p = x16 + (t0 + g) * ldx16;
  const unsigned long long group0 = static_cast<unsigned long long>(t0 + g) * (width / 8);
  int stage = 0;
  for (int k0 = 32 * warp; k0 < width; k0 += kStep) {
    const int k = k0 + 8 * c;
    ptx::cp_async_wait<kStages - 2>();
    __syncwarp();  // this stage has landed for every lane, and the one issued next has been read by all
    issue(stage == 0 ? kStages - 1 : stage - 1, k0 + (kStages - 1) * kStep);
    const unsigned char* const got = ring + stage * Tile::kStage;
    uint4 av[NT], xv[2];
#pragma unroll
    for (int n = 0; n < NT; ++n) av[n] = *reinterpret_cast<const uint4*>(got + kXBytes + n * 512 + lane * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (XP == 1) {
        xv[h] = *reinterpret_cast<const uint4*>(got + h * 512 + lane * 16);
      } else {
        float f[8];
        block_read(got, 8 * h + g, c, f);
        xv[h] = pack8<T>(f);
      }
      if (x16 != nullptr && k < width && 8 * h + g < rows) stg16(x16p + 8 * h * ldx16 + k, xv[h]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t lo[4], hi[4];
      const unsigned long long group = group0 + static_cast<unsigned long long>(k / 8);
      mask8(philox::words(key, ctr[b], group), xv[0], d.cut[b], d, lo);
      mask8(philox::words(key, ctr[b], group + static_cast<unsigned long long>(width)), xv[1], d.cut[b], d, hi);
      const uint32_t f0[4] = {lo[0], hi[0], lo[1], hi[1]}, f1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
      for (int n = b * NTB; n < (b + 1) * NTB; ++n) {
        ptx::mma16816<T>(acc[n], f0, av[n].x, av[n].y);
        ptx::mma16816<T>(acc[n], f1, av[n].z, av[n].w);
      }
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  // the warps' sums in shared memory, over the rings
  ptx::cp_async_wait<0>();
  __syncthreads();
  float* const red = reinterpret_cast<float*>(smem);  // [kWarps][16][LD]
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float* const p = red + (warp * 16 + g) * LD + 8 * n + 2 * c;
    *reinterpret_cast<float2*>(p) = make_float2(acc[n][0], acc[n][1]);
    *reinterpret_cast<float2*>(p + 8 * LD) = make_float2(acc[n][2], acc[n][3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 4 * NT; i += 32 * kWarps) {  // a pair of u's columns
    const int row = i / (4 * NT), col = 2 * (i % (4 * NT)), b = col / (8 * NTB), r = col % (8 * NTB);
    if (row >= rows || r >= rank) continue;
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 v = *reinterpret_cast<const float2*>(red + (w * 16 + row) * LD + col);
      s.x += v.x;
      s.y += v.y;
    }
    const float scale = NB == 2 && b == 1 ? d.scale[1] : d.scale[0];
    *reinterpret_cast<uint32_t*>(u + (t0 + row) * ldu + b * rank + r) =
        scale == 0.f ? 0u : Dt<T>::pack2(s.x * scale, s.y * scale);
  }
  // the columns behind the branches': a 1 (it multiplies the bias in the projection's extra K block), zeros
  const int n_u = NB * rank, more = (u_cols - n_u) / 2;
  for (int i = threadIdx.x; i < rows * more; i += 32 * kWarps)
    *reinterpret_cast<uint32_t*>(u + (t0 + i / more) * ldu + n_u + 2 * (i % more)) =
        i % more == 0 ? Dt<T>::pack2(1.f, 0.f) : 0u;
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
// A tile's bytes are on their way two tiles ahead through cp.async into the warp's own ring (49.7 us at
// 16,384 x 1536; one tile ahead 49.7, three, with fewer CTAs an SM, 60.0; without the ring 85.5).
// Four operand blocks of 16 ranks (two branches of 32, one of 64) take 240 registers, 8 warps an SM: 38.8 us
// for 11,170 x 1056, rank 32 x 2; held to 168 registers for 12 warps they spill, 59.5 us.
constexpr int kBwdStages = 3, kBwdWarps = 4;
template <int NB, int KR>
constexpr int bwd_stage() {  // x16: 2 pieces of 16 bytes a lane, the addend: 4, du: 16 tokens x 16 NB KR columns
  return (2 + 4 + NB * KR) * 512;
}

template <typename T, int NB, int KR>
__global__ void __launch_bounds__(32 * kBwdWarps, NB * KR <= 2 ? 4 : 2)
bwd_kernel(const T* __restrict__ du, int64_t ld_du, const T* __restrict__ x16, int64_t ldx, const T* __restrict__ a,
           int64_t lda, const float* addend, int64_t ld_add, float* dx, int64_t ld_dx, float* __restrict__ part,
           int64_t n_tok, int width, int rank, int chunk, int col_blocks, int n_units, Drop d,
           const int64_t* __restrict__ rng, int64_t stream_id) {
  constexpr int kStage = bwd_stage<NB, KR>(), C = 2 * NB * KR;  // C: 16-byte pieces of a row of du
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int unit = blockIdx.x * kBwdWarps + (threadIdx.x >> 5);  // (token chunk, block of 32 columns)
  if (unit >= n_units) return;
  const int cb = unit % col_blocks;
  const int64_t first = static_cast<int64_t>(unit / col_blocks) * chunk;
  const int n = n_tok - first < chunk ? static_cast<int>(n_tok - first) : chunk;  // tokens of the chunk
  const int k = 32 * cb + 8 * c;
  const bool in = k < width;
  const philox::Key key = philox::make_key(rng);
  philox::Stream ctr[NB];
  uint32_t af[NB][KR][4][2];   // A as P's operand: rows (rank) 2 c, 2 c + 1 (+ 8) of column n = g of tile j
  float acc[NB][KR][4][4];     // dA
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    ctr[b] = philox::make_stream(rng, stream_id + b);
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
  unsigned char* const ring = smem + (threadIdx.x >> 5) * (kBwdStages * kStage);
  const uint32_t ring_at = ptx::smem_u32(ring);
  // running addresses: of the tile issued next, and of dx and the generator's group of the one computed
  const T* xp = x16 + (first + g) * ldx + k;
  const int ar = lane >> 3, ac = 32 * cb + 4 * (lane & 7);  // the lane's row and column in a copy of the addend
  const float* addp = addend != nullptr ? addend + (first + ar) * ld_add + ac : nullptr;
  const bool whole = ld_dx % 8 == 0 && (reinterpret_cast<uintptr_t>(dx) & 31) == 0;
  float* dxp = dx + (first + g) * ld_dx + k;
  const T* dup[NB * KR];
  uint32_t du_dst[NB * KR];
  int du_row[NB * KR];  // past the chunk for a piece that is not there
#pragma unroll
  for (int q = 0; q < NB * KR; ++q) {  // du's rows, their pieces swizzled for ldmatrix
    const int row = (lane + 32 * q) / C, piece = (lane + 32 * q) % C, b = piece / (2 * KR), r = 8 * (piece % (2 * KR));
    dup[q] = du + (first + row) * ld_du + b * rank + r;
    du_dst[q] = 6 * 512 + (row * C + (piece ^ (row * C / 8 & (C - 1)))) * 16;
    du_row[q] = r < rank ? row : 1 << 30;
  }
  auto issue = [&](int stage, int i0) {
    const uint32_t dst = ring_at + stage * kStage;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool ok = in && i0 + 8 * h + g < n;
      ptx::cp_async16(dst + h * 512 + lane * 16, ok ? xp + 8 * h * ldx : x16, ok);
    }
    if (addend != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * i + ar;
        const bool ok = ac < width && r < n - i0;
        ptx::cp_async16(dst + 2 * 512 + block_at(r, lane & 7), ok ? addp + 4 * i * ld_add : addend, ok);
      }
    }
#pragma unroll
    for (int q = 0; q < NB * KR; ++q) {
      const bool ok = du_row[q] < n - i0;
      ptx::cp_async16(dst + du_dst[q], ok ? dup[q] : du, ok);
      dup[q] += 16 * ld_du;
    }
    xp += 16 * ldx;
    addp += 16 * ld_add;
  };
#pragma unroll
  for (int s = 0; s < kBwdStages - 1; ++s) {
    if (16 * s < n) issue(s, 16 * s);
    ptx::cp_async_commit();
  }
  int stage = 0;
  unsigned long long group = static_cast<unsigned long long>(first + g) * (width / 8) + k / 8;
  for (int i0 = 0; i0 < n; i0 += 16, group += 2 * width, dxp += 16 * ld_dx) {
    ptx::cp_async_wait<kBwdStages - 2>();
    __syncwarp();  // this stage has landed for every lane, and the one issued next has been read by all
    const int ahead = i0 + 16 * (kBwdStages - 1);
    if (ahead < n) issue(stage == 0 ? kBwdStages - 1 : stage - 1, ahead);
    ptx::cp_async_commit();
    const unsigned char* const got = ring + stage * kStage;
    uint4 xv[2];
    float out[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      xv[h] = *reinterpret_cast<const uint4*>(got + h * 512 + lane * 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) out[h][i] = 0.f;
      if (addend != nullptr) block_read(got + 2 * 512, 8 * h + g, c, out[h]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (d.scale[b] == 0.f) continue;  // nothing is kept
      const uint32_t limit = d.cut[b] & 0xFFFF0000u;
      uint32_t m[2][4];
      float p[4][4] = {};
      // rows (tokens) lane & 15, rank columns 8 (lane >> 4) ..
      auto at = [&](int r) {
        const int row = lane & 15, piece = 2 * (b * KR + r) + (lane >> 4);
        return ring_at + stage * kStage + 6 * 512 + (row * C + (piece ^ (row * C / 8 & (C - 1)))) * 16;
      };
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        uint32_t df[4];
        ptx::ldsm_x4(at(r), df[0], df[1], df[2], df[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) ptx::mma16816<T>(p[j], df, af[b][r][j][0], af[b][r][j][1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 w = philox::words(key, ctr[b], group + static_cast<unsigned long long>(h * width));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w}, xs[4] = {xv[h].x, xv[h].y, xv[h].z, xv[h].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m[h][j] = mask_add_pair(ws[j], xs[j], limit, d.shift, d.scale[b], p[j][2 * h], p[j][2 * h + 1], out[h][2 * j],
                                  out[h][2 * j + 1]);
        }
      }
      uint32_t bf[4][2];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) bf[j][h] = transpose8x8(m[h][j]);
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        uint32_t dt[4];  // du^T: rows rank g | g + 8, columns tokens 2 c .. | 2 c + 8 ..
        ptx::ldsm_x4_t(at(r), dt[0], dt[2], dt[1], dt[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) ptx::mma16816<T>(acc[b][r][j], dt, bf[j][0], bf[j][1]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (in && i0 + 8 * h + g < n) store32(dxp + 8 * h * ld_dx, out[h], whole);
    stage = stage + 1 == kBwdStages ? 0 : stage + 1;
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

// dA = scale * the sum of the chunks' partials in a fixed order (no atomics: the same bits every time):
// warp w of a CTA sums chunks w, w + 8, ... of 128 values, then the warps' sums are added in order.
__global__ void __launch_bounds__(256)
da_sum_kernel(const float* __restrict__ part, float* __restrict__ da, int n_chunks, int width, int rank, Drop d, int n4) {
  __shared__ float4 red[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < n4) {
    const float4* p = reinterpret_cast<const float4*>(part) + i;
#pragma unroll 8
    for (int c = warp; c < n_chunks; c += 8) {
      const float4 v = __ldg(p + static_cast<int64_t>(c) * n4);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || i >= n4) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) {
    const float4 v = red[w][lane];
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
  const double p[2] = {p0, p1};
  for (int b = 0; b < 2; ++b) {
    const uint32_t cut = philox::cut_of(p[b]), lane = cut < 65536u ? cut : 0u;
    d.cut[b] = lane << 16 | lane;
    d.scale[b] = philox::scale_of(cut);
  }
  d.ones = 0xFFFFu;
  d.shift = 65536u;
  d.minus = 0xFFFFFFFFu;
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
  int64_t ldu;
  int u_cols;
  int64_t n_tok;
  int width, rank;
  Drop d;
  const int64_t* rng;
  int64_t stream_id;
  cudaStream_t s;
};

template <typename X, typename T, int NB, int NTB>
int launch_down_t(const DownArgs& p) {
  static std::atomic<unsigned long long> done{0};
  constexpr int smem = DownTile<X, NB * NTB>::kSmem;
  auto kernel = down_kernel<X, T, NB, NTB>;
  if (int rc = ensure_dyn_smem(kernel, smem, done, "lora_down_dropout")) return rc;
  kernel<<<static_cast<unsigned>((p.n_tok + 15) / 16), 32 * kWarps, smem, p.s>>>(
      static_cast<const X*>(p.x), p.ldx, static_cast<const T*>(p.a), p.lda, static_cast<T*>(p.x16), p.ldx16,
      static_cast<T*>(p.u), p.ldu, p.u_cols, p.n_tok, p.width, p.rank, p.d, p.rng, p.stream_id);
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
                                       int64_t ldx16, void* u, int64_t ldu, int u_cols, int64_t n_tok, int width,
                                       int rank, int n_branch, double p0, double p1, const int64_t* rng, int64_t stream_id,
                                       int dtype, void* stream) {
  using namespace decik;
  using namespace decik::loradrop;
  if (int rc = check_sizes("lora_down_dropout", n_tok, width, rank, n_branch, p0, p1, dtype)) return rc;
  if (x_dtype != DECIK_F32 && x_dtype != dtype)
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout: x of dtype %d (F32 or the compute dtype %d)", x_dtype, dtype);
  if (u_cols < rank * n_branch || u_cols % 8 != 0)
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout: u_cols %d (a multiple of 8 from %d on)", u_cols, rank * n_branch);
  if (n_tok == 0) return DECIK_OK;
  if (!x || !a || !u || !rng) return set_error(DECIK_ERR_INVALID, "lora_down_dropout: null pointer");
  if (ldx < width || lda < width || (x16 && ldx16 < width) || ldu < u_cols)
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout: row strides shorter than the rows");
  const int xe = x_dtype == DECIK_F32 ? 4 : 8;
  if (ldx % xe || lda % 8 || (x16 && ldx16 % 8) || ldu % 8 || !aligned16(x) || !aligned16(a) ||
      (x16 && !aligned16(x16)) || !aligned16(u))
    return set_error(DECIK_ERR_INVALID, "lora_down_dropout: rows and pointers need 16-byte alignment");
  if (!aligned_to(rng, 8)) return set_error(DECIK_ERR_INVALID, "lora_down_dropout: rng is not aligned to its values");
  const DownArgs p{x, ldx, a, lda, x16, ldx16, u, ldu, u_cols, n_tok, width, rank, make_drop(p0, p1), rng, stream_id,
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
  if (!aligned_to(rng, 8)) return set_error(DECIK_ERR_INVALID, "lora_down_dropout_bwd: rng is not aligned to its values");
  const Drop d = make_drop(p0, p1);
  const Split sp = split_of(n_tok, width);
  const int n_units = sp.n_chunks * sp.col_blocks, n4 = width / 4 * rank * n_branch;
  float* part = static_cast<float*>(workspace);
  return DECIK_DISPATCH_16(dtype, [&] {
    auto go = [&](auto nb, auto kr) -> int {
      static std::atomic<unsigned long long> done{0};
      constexpr int smem = kBwdWarps * kBwdStages * bwd_stage<nb(), kr()>();
      auto kernel = bwd_kernel<T, nb(), kr()>;
      if (int rc = ensure_dyn_smem(kernel, smem, done, "lora_down_dropout_bwd")) return rc;
      kernel<<<(n_units + kBwdWarps - 1) / kBwdWarps, 32 * kBwdWarps, smem, s>>>(
          static_cast<const T*>(du), ld_du, static_cast<const T*>(x16), ldx, static_cast<const T*>(a), lda, addend,
          ld_add, dx, ld_dx, part, n_tok, width, rank, sp.chunk, sp.col_blocks, n_units, d, rng, stream_id);
      return check_launch("lora_down_dropout_bwd");
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    const int kr = (rank + 15) / 16;
    const int rc = n_branch == 2 ? (kr == 1 ? go(two, one) : go(two, two))
                                 : kr == 1 ? go(one, one) : kr == 2 ? go(one, two) : go(one, four);
    if (rc) return rc;
    da_sum_kernel<<<(n4 + 31) / 32, 256, 0, s>>>(part, da, sp.n_chunks, width, rank, d, n4);
    return check_launch("lora_down_dropout_bwd");
  });
}
