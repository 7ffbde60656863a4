// Tokens into expert order and back.
//   dispatch  out[pos[t, j]] = x[t] for every choice with pos >= 0; rows at or
//             past sum(group_sizes) are zero (their scales 1), as the rows of
//             a quantised zero block
//   combine   out[t] = residual[t] + sum_j w[t, j] * y[pos[t, j]], summed in
//             32 bits in slot order and rounded once
//   combine's backward  dy[pos[t, j]] = w[t, j] * dout[t],
//             dw[t, j] = <dout[t], y[pos[t, j]]>
// (dispatch's backward is a combine with weights 1.)
//
// All are bound by HBM: every row is moved once, in 16-byte vectors.  Dispatch
// goes by tokens, not by output rows, so a token is read once and stored k
// times; a warp takes a 2 KB piece of a row, which gives even small calls
// enough warps to reach all SMs (pieces of 1 KB: 5 % slower).  It writes up to
// nine tenths of what it moves: 4096 tokens, topk 8, rows of 7168 bytes take 58
// us, 4.2 TB/s of stores, where a fill runs at 3.9 TB/s.
#include "common.cuh"

namespace gl {
namespace moe {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int MAX_K = 32;  // choices of a token: a lane each

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}

// Row of the lane's choice, -1 for none; one past the rows is reported and
// treated as none.
__device__ __forceinline__ int load_pos(const int* pos, int64_t t, int k, int64_t rows, int* err) {
  const int lane = threadIdx.x & 31;
  int p = lane < k ? fetch(pos + t * k + lane) : -1;
  if (p >= rows) {
    atomicExch(err, GL_DEV_BAD_INDEX);
    p = -1;
  }
  return p;
}

// First row that belongs to no group, to every thread of the CTA; rows (none
// left) when the sizes are not a partition of at most `rows`.
__device__ __forceinline__ int64_t first_tail_row(const int* sizes, int G, int64_t rows, int* err) {
  __shared__ long long total;
  __shared__ int bad;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = 0;
    bad = 0;
  }
  __syncthreads();
  long long own = 0;
  bool neg = false;
  for (int g = threadIdx.x; g < G; g += blockDim.x) {
    const int n = fetch(sizes + g);
    neg = neg || n < 0;
    own += n;
  }
  if (own) atomicAdd(reinterpret_cast<unsigned long long*>(&total), static_cast<unsigned long long>(own));
  if (neg) bad = 1;
  __syncthreads();
  if (bad || total > rows) {
    if (threadIdx.x == 0) atomicExch(err, GL_DEV_BAD_GROUPS);
    return rows;
  }
  return total;
}

// Zeroes vectors of rows [first, rows), the grid's threads side by side.
__device__ __forceinline__ void zero_rows(uint4* out, int nvec, int64_t first, int64_t rows) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = first * nvec + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
       i < rows * nvec; i += step)
    out[i] = make_uint4(0, 0, 0, 0);
}

struct DispatchArgs {
  const uint4* x;
  const float* s;      // null without scales (ns 0) or tokens
  const int* pos;
  const int* sizes;
  int64_t T, rows;
  int k, G, nvec, ns;  // 16-byte vectors and scales of a row
  uint4* out;
  float* out_s;
  int* err;
};

__global__ void __launch_bounds__(256) dispatch_kernel(const DispatchArgs a) {
  constexpr int U = 4;
  follow();
  const int lane = threadIdx.x & 31;
  const int segs = (a.nvec + 32 * U - 1) / (32 * U);
  const int64_t units = a.T * segs, step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units;
       u += step) {
    const int64_t t = u / segs;
    const int seg = static_cast<int>(u - t * segs), v0 = seg * 32 * U + lane;
    uint4 v[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v0 + 32 * i < a.nvec) v[i] = fetch(a.x + t * a.nvec + v0 + 32 * i);
    const int own = load_pos(a.pos, t, a.k, a.rows, a.err);
    for (int j = 0; j < a.k; ++j) {
      const int64_t p = __shfl_sync(FULL, own, j);
      if (p < 0) continue;
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (v0 + 32 * i < a.nvec) a.out[p * a.nvec + v0 + 32 * i] = v[i];
      if (seg == 0)
        for (int i = lane; i < a.ns; i += 32) a.out_s[p * a.ns + i] = fetch(a.s + t * a.ns + i);
    }
  }
  const int64_t tail = first_tail_row(a.sizes, a.G, a.rows, a.err);
  zero_rows(a.out, a.nvec, tail, a.rows);
  if (a.ns)  // also without tokens, where s has no address
    for (int64_t i = tail * a.ns + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
         i < a.rows * a.ns; i += static_cast<int64_t>(gridDim.x) * blockDim.x)
      a.out_s[i] = 1.0f;
}

// Eight consecutive features of y as floats.
template <bool kF32>
struct Vec8 {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* y, int64_t vec) {
    if (kF32) {
      a = fetch(static_cast<const uint4*>(y) + 2 * vec);
      b = fetch(static_cast<const uint4*>(y) + 2 * vec + 1);
    } else {
      a = fetch(static_cast<const uint4*>(y) + vec);
    }
  }
  __device__ __forceinline__ void zero() { a = b = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void floats(float (&f)[8]) const {
    if (kF32) {
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    } else {
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = bf16x2_to_f32x2(w[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
};

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}

struct CombineArgs {
  const void* y;
  const int* pos;
  const float* w;     // or null: 1
  const uint4* res;   // or null
  int64_t T, rows;
  int k, nvec;        // vectors of 8 features
  uint4* out;
  int* err;
};

// B choices of a token are loaded at a time, U vectors of a lane from each.  Four
// loads in flight a lane with four CTAs an SM reach HBM's rate: 4096 tokens,
// topk 8, K 7168 take 91 us with B = U = 2 (floor 90), 133 us with eight loads
// and the two CTAs that their registers leave, 95 us with B = 4, U = 1; topk 2
// 81, 92 and 81 us (16387 tokens, K 4096).
template <bool kF32, int B, int U>
__global__ void __launch_bounds__(256, 4) combine_kernel(const CombineArgs a) {
  follow();
  const int lane = threadIdx.x & 31;
  const int segs = (a.nvec + 32 * U - 1) / (32 * U);
  const int64_t units = a.T * segs, step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units;
       u += step) {
    const int64_t t = u / segs;
    const int v0 = static_cast<int>(u - t * segs) * 32 * U + lane;
    const int own = load_pos(a.pos, t, a.k, a.rows, a.err);
    float w_own = own < 0 ? 0.0f : 1.0f;
    if (a.w && own >= 0) w_own = fetch(a.w + t * a.k + lane);
    float acc[U][8] = {};
    if (a.res) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        // a plain load: out may be the residual's own buffer
        Vec8<false> r;
        r.zero();
        if (v0 + 32 * i < a.nvec) r.a = a.res[t * a.nvec + v0 + 32 * i];
        r.floats(acc[i]);
      }
    }
    for (int j0 = 0; j0 < a.k; j0 += B) {
      Vec8<kF32> v[B][U];
#pragma unroll
      for (int j = 0; j < B; ++j) {
        // lanes from topk on hold -1
        const int64_t p = __shfl_sync(FULL, own, (j0 + j) & 31);
        const bool in = j0 + j < a.k && p >= 0;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          v[j][i].zero();
          if (in && v0 + 32 * i < a.nvec) v[j][i].load(a.y, p * a.nvec + v0 + 32 * i);
        }
      }
#pragma unroll
      for (int j = 0; j < B; ++j) {
        float w = __shfl_sync(FULL, w_own, (j0 + j) & 31);
        if (j0 + j >= a.k) w = 0.0f;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          float f[8];
          v[j][i].floats(f);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[i][e] = fmaf(w, f[e], acc[i][e]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v0 + 32 * i < a.nvec) a.out[t * a.nvec + v0 + 32 * i] = pack8(acc[i]);
  }
}

struct CombineBwdArgs {
  const uint4* dout;
  const void* y;
  const int* pos;
  const float* w;
  const int* sizes;
  int64_t T, rows;
  int k, G, nvec;
  void* dy;
  float* dw;
  int* err;
};

// A CTA takes a token: its gradient stays in registers (V vectors a thread)
// while the rows of its choices pass.  Four CTAs an SM where the registers do
// (4096 tokens, topk 8, K 7168: 167 us against 181 with two; 1.0 GB moved, half
// of it written).
template <int V, bool kF32>
__global__ void __launch_bounds__(256, V <= 4 ? 4 : 2) combine_bwd_kernel(const CombineBwdArgs a) {
  __shared__ float part[MAX_K][8];
  follow();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    float d[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int vec = threadIdx.x + i * blockDim.x;
      Vec8<false> g;
      g.zero();
      if (vec < a.nvec) g.load(a.dout, t * a.nvec + vec);
      g.floats(d[i]);
    }
    const int own = load_pos(a.pos, t, a.k, a.rows, a.err);
    const float w_own = own >= 0 ? fetch(a.w + t * a.k + lane) : 0.0f;
    for (int j = 0; j < a.k; ++j) {
      const int64_t p = __shfl_sync(FULL, own, j);
      const float w = __shfl_sync(FULL, w_own, j);
      float dot = 0.0f;
      if (p >= 0) {
        Vec8<kF32> v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int vec = threadIdx.x + i * blockDim.x;
          v[i].zero();
          if (vec < a.nvec) v[i].load(a.y, p * a.nvec + vec);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int vec = threadIdx.x + i * blockDim.x;
          if (vec < a.nvec) {
            float f[8], g[8], sum = 0.0f;
            v[i].floats(f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              sum = fmaf(d[i][e], f[e], sum);
              g[e] = w * d[i][e];
            }
            dot += sum;
            if (kF32) {
              float4* o = static_cast<float4*>(a.dy) + 2 * (p * a.nvec + vec);
              o[0] = make_float4(g[0], g[1], g[2], g[3]);
              o[1] = make_float4(g[4], g[5], g[6], g[7]);
            } else {
              static_cast<uint4*>(a.dy)[p * a.nvec + vec] = pack8(g);
            }
          }
        }
      }
      dot = warp_sum(dot);
      if (lane == 0) part[j][warp] = dot;
    }
    __syncthreads();
    if (threadIdx.x < a.k) {
      float s = 0.0f;
      for (int i = 0; i < nw; ++i) s += part[threadIdx.x][i];
      a.dw[t * a.k + threadIdx.x] = s;
    }
    __syncthreads();
  }
  const int64_t tail = first_tail_row(a.sizes, a.G, a.rows, a.err);
  zero_rows(static_cast<uint4*>(a.dy), kF32 ? 2 * a.nvec : a.nvec, tail, a.rows);
}

int launched(const char** why) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  *why = cudaGetErrorString(e);
  return -2;
}

// Tokens' worth of rows that a launch has to fill its grid for: of its tokens, or
// of the rows that no choice can name where there are more (a fixed capacity of
// 32768 rows of 14 KB for one token: 0.08 ms, 7.5 with its own CTAs).
int64_t grid_tokens(int64_t T, int64_t k, int64_t rows) { return rows - T * k > T ? rows - T * k : T; }

// CTAs of 8 warps for `units` warps' work: at most 8 a SM.
unsigned warp_ctas(int64_t units, int num_sms) {
  const int64_t need = (units + 7) / 8, most = 8 * static_cast<int64_t>(num_sms);
  const int64_t n = need < most ? need : most;
  return static_cast<unsigned>(n > 0 ? n : 1);
}

template <bool kF32, int B, int U>
void combine(const CombineArgs& a, int num_sms, cudaStream_t st) {
  const int64_t units = a.T * ((a.nvec + 32 * U - 1) / (32 * U));
  launch_following(combine_kernel<kF32, B, U>, warp_ctas(units, num_sms), 256, 0, st, a);
}

template <int V>
void combine_bwd(const CombineBwdArgs& a, int f32, unsigned ctas, int threads, cudaStream_t st) {
  if (f32)
    launch_following(combine_bwd_kernel<V, true>, ctas, threads, 0, st, a);
  else
    launch_following(combine_bwd_kernel<V, false>, ctas, threads, 0, st, a);
}

}  // namespace moe
}  // namespace gl

// Launchers: 0 on a launch, -2 on a launch error (why set).
int gl_launch_moe_dispatch(const void* x, int64_t row_bytes, const float* s, int64_t scales,
                           const int32_t* pos, const int32_t* group_sizes, int64_t G, int64_t T, int64_t k,
                           int64_t rows, void* out, float* out_s, int* err, cudaStream_t st, int num_sms,
                           const char** why) {
  using namespace gl::moe;
  const DispatchArgs a{static_cast<const uint4*>(x), s, pos, group_sizes, T, rows, static_cast<int>(k),
                       static_cast<int>(G), static_cast<int>(row_bytes / 16), static_cast<int>(scales),
                       static_cast<uint4*>(out), out_s, err};
  const int64_t units = grid_tokens(T, k, rows) * ((a.nvec + 127) / 128);
  gl::launch_following(dispatch_kernel, warp_ctas(units, num_sms), 256, 0, st, a);
  return launched(why);
}

int gl_launch_moe_combine(const void* y, int y_f32, const int32_t* pos, const float* weights,
                          const void* residual, int64_t T, int64_t k, int64_t K, int64_t rows, void* out,
                          int* err, cudaStream_t st, int num_sms, const char** why) {
  using namespace gl::moe;
  const CombineArgs a{y, pos, weights, static_cast<const uint4*>(residual), T, rows, static_cast<int>(k),
                      static_cast<int>(K / 8), static_cast<uint4*>(out), err};
  if (k == 1)
    y_f32 ? combine<true, 1, 4>(a, num_sms, st) : combine<false, 1, 4>(a, num_sms, st);
  else
    y_f32 ? combine<true, 2, 2>(a, num_sms, st) : combine<false, 2, 2>(a, num_sms, st);
  return launched(why);
}

int gl_launch_moe_combine_bwd(const void* dout, const void* y, int y_f32, const int32_t* pos,
                              const float* weights, const int32_t* group_sizes, int64_t G, int64_t T,
                              int64_t k, int64_t K, int64_t rows, void* dy, float* dweights, int* err,
                              cudaStream_t st, int num_sms, const char** why) {
  using namespace gl::moe;
  const CombineBwdArgs a{static_cast<const uint4*>(dout), y, pos, weights, group_sizes, T, rows,
                         static_cast<int>(k), static_cast<int>(G), static_cast<int>(K / 8), dy, dweights,
                         err};
  // A thread takes 4 vectors of 8 (2 of fp32) where there are tokens enough to
  // fill the SMs: small CTAs and more loads in flight.  us against 256 threads
  // with as many vectors as the row then needs: 16387 tokens, topk 2, K 4096: 103
  // (120); 4096, 8, 2048: 54 (72); 8192, 4, 512: 18 (33).  With fewer tokens
  // a wide CTA is the shorter path (33 tokens, topk 8, K 4096: 6.5 against 8.2);
  // above 160 threads whole CTAs of 256 were faster (4096, 8, 7168: 168 against
  // 186 with 224).
  const int per = T <= 4 * static_cast<int64_t>(num_sms) ? 1 : y_f32 ? 2 : 4;
  const int need = ((a.nvec + per - 1) / per + 31) / 32 * 32;
  const int threads = need < 192 ? need : 256;
  const int v = (a.nvec + threads - 1) / threads;
  const int64_t most = 2048 / threads * static_cast<int64_t>(num_sms);
  const int64_t n = grid_tokens(T, k, rows);
  const unsigned ctas = static_cast<unsigned>(n < 1 ? 1 : n < most ? n : most);
  if (v <= 1)
    combine_bwd<1>(a, y_f32, ctas, threads, st);
  else if (v <= 2)
    combine_bwd<2>(a, y_f32, ctas, threads, st);
  else if (v <= 4)
    combine_bwd<4>(a, y_f32, ctas, threads, st);
  else
    combine_bwd<8>(a, y_f32, ctas, threads, st);
  return launched(why);
}
