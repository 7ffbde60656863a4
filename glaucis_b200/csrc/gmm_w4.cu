// Grouped products with 4-bit weights and one fp32 scale per 128 weights of a
// column, for few rows (a decoding batch), and the quantiser of the weights.
//   out[m, n] = sum_b s[g, b, n] * sum_{k in block b} x[m, k] q[g, k, n]
// Format: q in -8..7, stored as the nibble u = q + 8; nibble j of the 32-bit
// word w4[g, i, n] is k = 8 i + j.
//
// With few rows the product reads each weight of the groups in use once and
// computes little with it: it is bound by HBM, and what must not get in the
// way is the work of widening 4-bit weights.  So:
//   * Weights go through mma.sync (m16n8k16, fp16 in, fp32 sums) as the 16-row
//     operand, 8 rows of x as the 8 columns: enough rate for a memory-bound
//     product, no shared memory, fragments straight from global loads.  (A
//     tcgen05 tile has 128 rows of shared-memory operands that would have to
//     be widened and written first.)
//   * A nibble is used as it lies in the word: masked, it is the fp16
//     subnormal u * 2^-24 (or 16 u * 2^-24 four bits up), exact in the matrix
//     unit.  Eight weights cost four ANDs and one shift.  The x that meets the
//     second nibble of a byte is stored divided by 16, and the offset 8 * sum(x)
//     starts the sum with its negative.
//   * x is bf16, whose range fp16 lacks: every 128-block of a row is scaled by
//     a power of two that takes its largest value to [2^13, 2^14), which is
//     exact (values 2^38 below the largest lose bits far under the sum's
//     rounding), and scaled back where the block's fp32 sum meets the weights'
//     scale.  A first small launch does this once for all groups' rows, in the
//     order the fragments want; the product's CTAs start beside it, find their
//     group and load their first weights before they wait for it.
#include "common.cuh"

#include <cuda_fp16.h>

namespace gl {
namespace w4 {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int COLS = 32;  // columns of a CTA
constexpr int ROWS = 8;   // rows of a tile

struct PrepArgs {
  const uint4* x;
  const int* sizes;
  int64_t M;
  int G, kb;         // kb: K / 128
  uint4* xf;         // fp16 [M, K], each 8 in the order 0 4 1 5 2 6 3 7, odd ones / 16
  float2* xs;        // [M, K / 128]: -8 * 2^-24 * sum of the scaled x, 2^(e + 12)
  void* out;         // rows of no group are zeroed when zero_tail
  int64_t row_words; // 16-byte words of an output row
  int zero_tail;
  int* err;
};

// 16 threads take a 128-block of a row.
__global__ void __launch_bounds__(256) w4_prep_kernel(const PrepArgs a) {
  cudaTriggerProgrammaticLaunchCompletion();
  const int64_t blocks = a.M * a.kb;
  const int sub = threadIdx.x & 15;
  for (int64_t b0 = static_cast<int64_t>(blockIdx.x) * 16; b0 < blocks;
       b0 += static_cast<int64_t>(gridDim.x) * 16) {
    const int64_t b = b0 + (threadIdx.x >> 4);
    const bool in = b < blocks;
    const uint4 v = in ? __ldg(a.x + b * 16 + sub) : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float f[8];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = bf16x2_to_f32x2(w[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
      m = fmaxf(m, fmaxf(fabsf(p.x), fabsf(p.y)));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
    // exponent of the largest value, to 2^13; blocks below 2^-113 take 2^126
    int e = static_cast<int>(__float_as_uint(m) >> 23) - 127 - 13;
    e = e < -126 ? -126 : e;
    const float scale = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] *= scale;
      sum += f[i];
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
    if (in) {
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float d = i & 1 ? 0.0625f : 1.0f;
        const __half2 p = __floats2half2_rn(f[i] * d, f[i + 4] * d);
        h[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
      a.xf[b * 16 + sub] = make_uint4(h[0], h[1], h[2], h[3]);
      if (sub == 0)
        a.xs[b] = make_float2(sum * -0x1p-21f, __uint_as_float(static_cast<uint32_t>(127 + e + 12) << 23));
    }
  }
  // one CTA checks the sizes, all zero the rows of no group
  __shared__ long long total;
  __shared__ int bad;
  if (threadIdx.x == 0) total = bad = 0;
  __syncthreads();
  long long own = 0;
  for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
    const int n = __ldg(a.sizes + g);
    if (n < 0) bad = 1;
    own += n;
  }
  if (own) atomicAdd(reinterpret_cast<unsigned long long*>(&total), static_cast<unsigned long long>(own));
  __syncthreads();
  if (bad || total > a.M) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicExch(a.err, GL_DEV_BAD_GROUPS);
    return;
  }
  if (a.zero_tail)
    for (int64_t i = total * a.row_words + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
         i < a.M * a.row_words; i += static_cast<int64_t>(gridDim.x) * blockDim.x)
      static_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0);
}

struct Args {
  const uint4* w;      // [G, K / 8, N / 4] words of four columns
  const float4* s;     // [G, K / 128, N / 4]
  const int* sizes;
  const uint4* xf;
  const float2* xs;
  int64_t M;
  int G, kb, n4;       // n4: N / 4
  void* out;
  int out_f32;
};

// Streaming 16-byte load: weights are read once, L1 is left to x.
__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Group, first row and number of rows of tile `tile` (tiles of 8 rows, groups
// in order); false when there are fewer.  A warp looks at 128 groups a step.
__device__ __forceinline__ bool find_tile(const Args& a, int64_t tile, int& group, int64_t& row0, int& nrows) {
  const int lane = threadIdx.x & 31;
  int64_t rows_before = 0, tiles_before = 0;
  for (int g0 = 0; g0 < a.G; g0 += 128) {
    int n[4], rows = 0, tiles = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int g = g0 + 4 * lane + j;
      n[j] = g < a.G ? __ldg(a.sizes + g) : 0;
      n[j] = n[j] < 0 ? 0 : n[j] > a.M ? static_cast<int>(a.M) : n[j];  // reported by the first launch
      rows += n[j];
      tiles += (n[j] + ROWS - 1) / ROWS;
    }
    int64_t r = rows, t = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t ro = __shfl_up_sync(FULL, r, o), to = __shfl_up_sync(FULL, t, o);
      if (lane >= o) {
        r += ro;
        t += to;
      }
    }
    const uint32_t past = __ballot_sync(FULL, tiles_before + t > tile);
    if (past) {
      const int src = __ffs(past) - 1;
      int64_t r0 = rows_before + r - rows, t0 = tiles_before + t - tiles;
      int g = 0, cnt = 0;
      int64_t first = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int nt = (n[j] + ROWS - 1) / ROWS;
        if (tile >= t0 && tile < t0 + nt) {
          g = g0 + 4 * lane + j;
          first = r0 + (tile - t0) * ROWS;
          const int64_t left = r0 + n[j] - first;
          cnt = static_cast<int>(left < ROWS ? left : ROWS);
        }
        t0 += nt;
        r0 += n[j];
      }
      group = __shfl_sync(FULL, g, src);
      row0 = __shfl_sync(FULL, first, src);
      nrows = __shfl_sync(FULL, cnt, src);
      return row0 + nrows <= a.M;
    }
    rows_before += __shfl_sync(FULL, r, 31);
    tiles_before += __shfl_sync(FULL, t, 31);
  }
  return false;
}

// A CTA takes 32 columns of a tile; its W warps take the K blocks in turn and
// add up through shared memory.  Lane (g, t) of a warp holds columns 4 g .. 4 g
// + 3 and, of every 32 k, words (k / 8) t: four columns' words are one 16-byte
// load, and one load of the warp covers four whole 128-byte lines.
template <int W>
__global__ void __launch_bounds__(32 * W) gmm_w4_kernel(const Args a) {
  __shared__ float part[W][ROWS][COLS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, t = lane & 3;
  int group = 0, nrows = 0;
  int64_t row0 = 0;
  if (!find_tile(a, blockIdx.y, group, row0, nrows)) {
    cudaGridDependencySynchronize();  // the launch ends no earlier than the first one
    return;
  }
  const int col4 = blockIdx.x * (COLS / 4) + gq;
  const uint4* wp = a.w + (static_cast<int64_t>(group) * a.kb * 16 + t) * a.n4 + col4;
  const float4* sp = a.s + static_cast<int64_t>(group) * a.kb * a.n4 + col4;
  const uint4* xp = a.xf + (row0 + gq) * a.kb * 16 + t;
  const float2* xsp = a.xs + (row0 + 2 * t) * a.kb;
  const bool has_x = gq < nrows, r0 = 2 * t < nrows, r1 = 2 * t + 1 < nrows;
  const int64_t line = 4 * static_cast<int64_t>(a.n4);  // 32 k further

  uint4 nw[4];
  float4 ns;
  if (warp < a.kb) {
#pragma unroll
    for (int i = 0; i < 4; ++i) nw[i] = ld_stream(wp + (4 * warp + i) * line);
    ns = __ldg(sp + static_cast<int64_t>(warp) * a.n4);
  }
  cudaGridDependencySynchronize();  // x in fragment order

  float tot[2][4] = {};
  for (int kb = warp; kb < a.kb; kb += W) {
    uint4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = nw[i];
    const float4 s = ns;
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = has_x ? __ldg(xp + kb * 16 + 4 * i) : make_uint4(0, 0, 0, 0);
    const float2 xs0 = r0 ? __ldg(xsp + kb) : make_float2(0.0f, 0.0f);
    const float2 xs1 = r1 ? __ldg(xsp + a.kb + kb) : make_float2(0.0f, 0.0f);
    if (kb + W < a.kb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) nw[i] = ld_stream(wp + (4 * (kb + W) + i) * line);
      ns = __ldg(sp + static_cast<int64_t>(kb + W) * a.n4);
    }
    float acc[2][4];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      acc[p][0] = acc[p][2] = xs0.x;
      acc[p][1] = acc[p][3] = xs1.x;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t u = c[2 * p], v = c[2 * p + 1];
        mma(acc[p], u & 0x000F000Fu, v & 0x000F000Fu, u & 0x00F000F0u, v & 0x00F000F0u, x[i].x, x[i].y);
        mma(acc[p], (u >> 8) & 0x000F000Fu, (v >> 8) & 0x000F000Fu, (u >> 8) & 0x00F000F0u,
            (v >> 8) & 0x00F000F0u, x[i].z, x[i].w);
      }
    }
    // 2^24 of the nibbles and 2^e of x, 12 of them on the scale: neither
    // product leaves fp32's range before the other factor brings it back
    const float sc[4] = {s.x * 4096.0f, s.y * 4096.0f, s.z * 4096.0f, s.w * 4096.0f};
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      tot[p][0] = fmaf(acc[p][0] * sc[2 * p], xs0.y, tot[p][0]);
      tot[p][1] = fmaf(acc[p][1] * sc[2 * p], xs1.y, tot[p][1]);
      tot[p][2] = fmaf(acc[p][2] * sc[2 * p + 1], xs0.y, tot[p][2]);
      tot[p][3] = fmaf(acc[p][3] * sc[2 * p + 1], xs1.y, tot[p][3]);
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    *reinterpret_cast<float2*>(&part[warp][2 * t][4 * gq + 2 * p]) = make_float2(tot[p][0], tot[p][2]);
    *reinterpret_cast<float2*>(&part[warp][2 * t + 1][4 * gq + 2 * p]) = make_float2(tot[p][1], tot[p][3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * COLS; i += 32 * W) {
    const int r = i / COLS, c = i % COLS;
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) v += part[k][r][c];
    const int64_t at = (row0 + r) * a.n4 * 4 + static_cast<int64_t>(blockIdx.x) * COLS + c;
    if (a.out_f32)
      static_cast<float*>(a.out)[at] = v;
    else
      static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  }
}

// Quantiser: a thread takes 128 k of two neighbouring columns, twice (the
// second read hits the caches).  s = max|w| / 7, 1 for a zero block; q =
// round-half-even(w / s).
__global__ void __launch_bounds__(128) quant_w4_kernel(const uint32_t* w, int64_t N2, int kb, uint2* q,
                                                       float2* s) {
  const int64_t n2 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (n2 >= N2) return;
  const int64_t b = static_cast<int64_t>(blockIdx.z) * kb + blockIdx.y;
  const uint32_t* p = w + b * 128 * N2 + n2;
  float m0 = 0.0f, m1 = 0.0f;
#pragma unroll 16
  for (int k = 0; k < 128; ++k) {
    const float2 v = bf16x2_to_f32x2(__ldg(p + k * N2));
    m0 = fmaxf(m0, fabsf(v.x));
    m1 = fmaxf(m1, fabsf(v.y));
  }
  const float s0 = m0 == 0.0f ? 1.0f : m0 / 7.0f, s1 = m1 == 0.0f ? 1.0f : m1 / 7.0f;
  s[b * N2 + n2] = make_float2(s0, s1);
  for (int i = 0; i < 16; ++i) {
    uint32_t a = 0, c = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 v = bf16x2_to_f32x2(__ldg(p + (8 * i + j) * N2));
      // the bounds also give non-finite weights a defined nibble
      const int q0 = static_cast<int>(fminf(fmaxf(rintf(v.x / s0), -7.0f), 7.0f));
      const int q1 = static_cast<int>(fminf(fmaxf(rintf(v.y / s1), -7.0f), 7.0f));
      a |= static_cast<uint32_t>(q0 + 8) << (4 * j);
      c |= static_cast<uint32_t>(q1 + 8) << (4 * j);
    }
    q[(b * 16 + i) * N2 + n2] = make_uint2(a, c);
  }
}

int launched(const char** why) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  *why = cudaGetErrorString(e);
  return -2;
}

template <int W>
cudaError_t launch(const Args& a, unsigned tiles, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.n4 * 4 / COLS), tiles);
  cfg.blockDim = dim3(32 * W);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, gmm_w4_kernel<W>, a);
}

}  // namespace w4
}  // namespace gl

// x in fragment order, then two floats a 128-block.
size_t gl_gmm_w4_ws_bytes(int64_t M, int64_t K) {
  return static_cast<size_t>(M) * K * 2 + static_cast<size_t>(M) * (K / 128) * 8;
}

// Launchers: 0 on a launch, -1 on a bad argument, -2 on a launch error (why set).
int gl_launch_gmm_w4(const void* x, const void* w4, const float* s, const int32_t* group_sizes, int64_t G,
                     int64_t M, int64_t K, int64_t N, void* out, int out_f32, int zero_tail, void* ws,
                     int* err, cudaStream_t st, int num_sms, const char** why) {
  using namespace gl::w4;
  const int kb = static_cast<int>(K / 128);
  uint4* xf = static_cast<uint4*>(ws);
  float2* xs = reinterpret_cast<float2*>(xf + M * (K / 8));
  const PrepArgs p{static_cast<const uint4*>(x), group_sizes, M, static_cast<int>(G), kb, xf, xs, out,
                   N * (out_f32 ? 4 : 2) / 16, zero_tail, err};
  const int64_t need = (M * kb + 15) / 16, most = 4 * static_cast<int64_t>(num_sms);
  w4_prep_kernel<<<static_cast<unsigned>(need < most ? need : most), 256, 0, st>>>(p);
  if (const int rc = launched(why)) return rc;
  const Args a{static_cast<const uint4*>(w4), reinterpret_cast<const float4*>(s), group_sizes, xf, xs, M,
               static_cast<int>(G), kb, static_cast<int>(N / 4), out, out_f32};
  // at most one short tile for every group that can have rows
  const int64_t tiles = M / ROWS + (M < G ? M : G);
  if (tiles > 65535) {
    *why = "too many rows";
    return -1;
  }
  const cudaError_t e = launch<8>(a, static_cast<unsigned>(tiles), st);
  if (e == cudaSuccess) return 0;
  *why = cudaGetErrorString(e);
  return -2;
}

int gl_launch_quant_w4(const void* w, int64_t G, int64_t K, int64_t N, void* q, float* s, cudaStream_t st,
                       const char** why) {
  using namespace gl::w4;
  quant_w4_kernel<<<dim3(static_cast<unsigned>((N / 2 + 127) / 128), static_cast<unsigned>(K / 128),
                         static_cast<unsigned>(G)),
                    128, 0, st>>>(static_cast<const uint32_t*>(w), N / 2, static_cast<int>(K / 128),
                                  static_cast<uint2*>(q), reinterpret_cast<float2*>(s));
  return launched(why);
}
