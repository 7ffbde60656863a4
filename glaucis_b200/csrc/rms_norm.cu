// RMS norm with the residual's addition, forward and backward.
//
//   h = bf16(x + residual)            (h = x without a residual)
//   r = 1 / sqrt(mean_k h^2 + eps),   y = h * r * w
// out: y in bf16 and / or, per 128 features, the e4m3 pair of the activation
// quantiser (s = max|y| / 448, 1 for an all-zero block; q = e4m3(y / s)),
// quantised from y in 32 bits: the 8-bit output is rounded once, not first to
// bf16.  The norm is that of the stored (rounded) h, so the backward pass,
// which starts from h, differentiates exactly what ran forward.
//   backward, u = w * dy, xh = h * r:
//   dx = r * (u - xh * mean_k(u * xh)) + dh,   dw = sum_rows dy * xh
//
// Both passes are bound by HBM: a row is read once, held in registers as
// 16-byte vectors (8 features a thread and vector) and written once.  The row
// sums are held in 32 bits and reduced in a fixed order.  Of 64 Mi elements the
// 8-bit output with residual takes 0.86 to 1.02 of the copy rate from 128 to
// 16384 features, the backward 0.82 to 1.09, the bf16 output alone 0.81 to 1.0.
#include "common.cuh"

namespace gl {
namespace rms {

constexpr int SMALL_T = 256;  // threads of a CTA whose warps take rows of their own

struct FwdArgs {
  const uint4* x;
  const uint4* res;   // or null
  const void* w;
  uint4* h;           // with res
  uint4* y;           // or null
  uint2* q;           // or null
  float* s;           // with q
  float* rstd;        // or null
  int64_t M;
  int nvec;           // K / 8
  float inv_k, eps;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Eight features as four pairs: the arithmetic runs on packed f32x2
// instructions, without which a row of 7168 with its 8-bit output costs twice
// the issue slots and runs below HBM's rate at the clocks of a power-capped
// part (143 us against 126 for 16384 rows).
struct F8 {
  float2 p[4];
};

__device__ __forceinline__ F8 unpack8(const uint4& u) {
  return {{bf16x2_to_f32x2(u.x), bf16x2_to_f32x2(u.y), bf16x2_to_f32x2(u.z), bf16x2_to_f32x2(u.w)}};
}

__device__ __forceinline__ uint4 pack8(const F8& f) {
  return make_uint4(pack_bf16x2(f.p[0].x, f.p[0].y), pack_bf16x2(f.p[1].x, f.p[1].y),
                    pack_bf16x2(f.p[2].x, f.p[2].y), pack_bf16x2(f.p[3].x, f.p[3].y));
}

__device__ __forceinline__ F8 neg8(const F8& a) {
  F8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.p[j] = make_float2(-a.p[j].x, -a.p[j].y);
  return r;
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ F8 mul8(const F8& a, const F8& b) {
  F8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.p[j] = __fmul2_rn(a.p[j], b.p[j]);
  return r;
}

__device__ __forceinline__ F8 scale8(const F8& a, float v) {
  F8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.p[j] = __fmul2_rn(a.p[j], both(v));
  return r;
}

// acc += a * b, pair by pair
__device__ __forceinline__ void dot8(const F8& a, const F8& b, float2& acc) {
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = __ffma2_rn(a.p[j], b.p[j], acc);
}

template <bool kW32>
__device__ __forceinline__ F8 load_w8(const void* w, int vec) {
  if (kW32) {
    const float4 a = fetch(static_cast<const float4*>(w) + 2 * vec);
    const float4 b = fetch(static_cast<const float4*>(w) + 2 * vec + 1);
    return {{make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)}};
  }
  return unpack8(fetch(static_cast<const uint4*>(w) + vec));
}

// Sum over the threads of a row: L lanes of a warp, or (L = 0) the CTA's warps
// through `part` (one slot per warp).
template <int L>
__device__ __forceinline__ float row_sum(float v, float* part) {
  if (L == 16) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
  }
  v = warp_sum(v);
  if (L == 32) return v;
  const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (lane == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < nw ? part[lane] : 0.0f);
}

// V vectors a thread.  L lanes a row (16 up to 128 features, a warp up to 1024),
// SMALL_T threads a CTA; L = 0: a CTA per row, in 32 registers with two vectors
// (h is kept packed and unpacked again), so that 2048 threads fit an SM: 7168
// features 73 us for 9362 rows, 78 with 38 registers.
template <int V, int L, bool kQuant, bool kW32>
__global__ void __launch_bounds__(L ? SMALL_T : 1024, L == 0 && V == 2 ? 2 : 1) rms_norm_fwd_kernel(const FwdArgs a) {
  constexpr int LL = L ? L : 1;
  __shared__ float part[32];
  follow();
  const int64_t row = L ? static_cast<int64_t>(blockIdx.x) * (SMALL_T / LL) + threadIdx.x / LL
                        : static_cast<int64_t>(blockIdx.x);
  // rows end inside a warp (two a warp): past them a thread goes on with none
  const bool live = !L || row < a.M;
  const int tid = L ? threadIdx.x % LL : threadIdx.x;
  const int step = L ? L : blockDim.x;
  const int nvec = live ? a.nvec : 0;
  const int64_t base = row * a.nvec;

  // plain loads: h may be x's or the residual's own buffer (every element is
  // read before the same thread writes it)
  uint4 xv[V], rv[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int vec = tid + i * step;
    xv[i] = vec < nvec ? a.x[base + vec] : make_uint4(0, 0, 0, 0);
    if (a.res) rv[i] = vec < nvec ? a.res[base + vec] : make_uint4(0, 0, 0, 0);
  }
  float2 sum2 = both(0.0f);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int vec = tid + i * step;
    F8 h = unpack8(xv[i]);
    if (a.res) {
      const F8 g = unpack8(rv[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) h.p[j] = __fadd2_rn(h.p[j], g.p[j]);
      xv[i] = pack8(h);  // the sum as it is stored: the one rounding of h
      if (vec < nvec) a.h[base + vec] = xv[i];
      h = unpack8(xv[i]);
    }
    dot8(h, h, sum2);
  }
  const float sum = row_sum<L>(sum2.x + sum2.y, part);
  // 2 ulp; a correctly rounded root costs the 8-bit output 1 to 3 %
  const float r = rsqrtf(fmaf(sum, a.inv_k, a.eps));
  if (a.rstd && tid == 0 && live) a.rstd[row] = r;

#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int vec = tid + i * step;
    const bool in = vec < nvec;
    // y, or with the 8-bit output -y, as its division takes it (markstein2)
    F8 f = scale8(unpack8(xv[i]), kQuant ? -r : r);
    if (in) {  // past the row all are 0
      f = mul8(f, load_w8<kW32>(a.w, vec));
      if (a.y) a.y[base + vec] = pack8(kQuant ? neg8(f) : f);
    }
    if (kQuant) {
      // a block of 128 features is a half-warp's vectors (nvec % 16 == 0, so
      // a half-warp is inside the row or past it as a whole)
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) m = fmaxf(m, fmaxf(fabsf(f.p[j].x), fabsf(f.p[j].y)));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      float s;
      if (m == 0.0f || (m >= 0x1p-55f && m <= 3.40282347e38f)) {
        // m / 448 correctly rounded (Markstein: the rounded product with the
        // rounded reciprocal, then one correction), then the elements' quotients
        // likewise: the scale stays above BlockDiv's bound
        constexpr float R = 1.0f / 448.0f;
        s = m * R;
        s = m == 0.0f ? 1.0f : fmaf(fmaf(-s, 448.0f, m), R, s);
        const float2 ny = both(-__frcp_rn(s)), s2 = both(s);
#pragma unroll
        for (int j = 0; j < 4; ++j) f.p[j] = markstein2(f.p[j], ny, s2);
      } else {  // tiny or infinite: each element divided
        s = m / 448.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f.p[j] = make_float2(-f.p[j].x / s, -f.p[j].y / s);
      }
      if (in) {
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = cvt_e4m3x2(f.p[j].x, f.p[j].y);
        a.q[base + vec] = make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
        if ((tid & 15) == 0) a.s[row * (a.nvec >> 4) + (vec >> 4)] = s;
      }
    }
  }
}

struct BwdArgs {
  const uint4* dy;
  const uint4* dh;    // or null
  const uint4* h;
  const void* w;
  const float* rstd;
  uint4* dx;
  float* part;        // fp32 [gridDim.x, K]: each CTA's share of dw
  int64_t M;
  int nvec;
  float inv_k;
};

// A persistent CTA takes rows blockIdx.x, + gridDim.x, ... (L lanes each, or L =
// 0: the CTA one row at a time) and keeps its columns' share of dw in registers.
// dy and h of the next row are loaded while this row's sum is under way, dh,
// which only dx needs, with the row itself (4099 x 4096: 28 us without).  Above
// 6144 features a second CTA on the SM is worth more than those registers (7168:
// 88 us for 9362 rows, 98 with one CTA and loads ahead).
template <int V, int L, int MAX_T, int CTAS, bool kW32>
__global__ void __launch_bounds__(MAX_T, CTAS) rms_norm_bwd_kernel(const BwdArgs a) {
  constexpr bool kAhead = MAX_T <= 384;
  constexpr int LL = L ? L : 1, ROWS = L ? SMALL_T / LL : 1;
  __shared__ float part[2][32];
  __shared__ __align__(16) float cross[ROWS][L ? L * V * 8 : 2];
  const int tid = L ? threadIdx.x % LL : threadIdx.x;
  const int step = L ? L : blockDim.x;
  const int64_t rows_step = static_cast<int64_t>(gridDim.x) * ROWS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + (L ? threadIdx.x / LL : 0);
  uint4 gn[V], hn[V];
  auto load = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int vec = tid + i * step;
      const bool in = r < a.M && vec < a.nvec;
      gn[i] = in ? __ldg(a.dy + r * a.nvec + vec) : make_uint4(0, 0, 0, 0);
      hn[i] = in ? __ldg(a.h + r * a.nvec + vec) : make_uint4(0, 0, 0, 0);
    }
  };
  F8 dw[V];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[i].p[j] = both(0.0f);
  if (kAhead) load(row);
  // as many rounds for every lane of a warp (rows may end inside one)
  const int64_t rounds = (a.M - static_cast<int64_t>(blockIdx.x) * ROWS + rows_step - 1) / rows_step;
  for (int64_t n = 0; n < rounds; ++n, row += rows_step) {
    const int it = static_cast<int>(n & 1);
    const int64_t base = row * a.nvec;
    const int nvec = row < a.M ? a.nvec : 0;
    const float r = row < a.M ? __ldg(a.rstd + row) : 0.0f;
    uint4 gv[V], hv[V], dv[V];
    if (!kAhead) load(row);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      gv[i] = gn[i];
      hv[i] = hn[i];
      const int vec = tid + i * step;
      dv[i] = a.dh && vec < nvec ? __ldg(a.dh + base + vec) : make_uint4(0, 0, 0, 0);
    }
    if (kAhead) load(row + rows_step);
    float2 c2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int vec = tid + i * step;
      if (vec < nvec) {
        const F8 g = unpack8(gv[i]), xh = scale8(unpack8(hv[i]), r);
        dot8(mul8(g, load_w8<kW32>(a.w, vec)), xh, c2);
#pragma unroll
        for (int j = 0; j < 4; ++j) dw[i].p[j] = __ffma2_rn(g.p[j], xh.p[j], dw[i].p[j]);
      }
    }
    // two sets of slots: a warp may reach the next row's sum while another
    // still reads this one's
    const float c = row_sum<L>(c2.x + c2.y, part[it]) * a.inv_k;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int vec = tid + i * step;
      if (vec < nvec) {
        const F8 u = mul8(unpack8(gv[i]), load_w8<kW32>(a.w, vec)), xh = scale8(unpack8(hv[i]), r);
        F8 d = unpack8(dv[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          d.p[j] = __ffma2_rn(both(r), __ffma2_rn(xh.p[j], both(-c), u.p[j]), d.p[j]);
        a.dx[base + vec] = pack8(d);
      }
    }
  }
  float* out = a.part + static_cast<int64_t>(blockIdx.x) * a.nvec * 8;
  if (L) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float2*>(&cross[threadIdx.x / LL][(tid + i * L) * 8 + 2 * j]) = dw[i].p[j];
    __syncthreads();
    for (int k = threadIdx.x; k < a.nvec * 8; k += blockDim.x) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) s += cross[i][k];
      out[k] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int vec = tid + i * step;
      if (vec < a.nvec) {
        reinterpret_cast<float4*>(out)[2 * vec] =
            make_float4(dw[i].p[0].x, dw[i].p[0].y, dw[i].p[1].x, dw[i].p[1].y);
        reinterpret_cast<float4*>(out)[2 * vec + 1] =
            make_float4(dw[i].p[2].x, dw[i].p[2].y, dw[i].p[3].x, dw[i].p[3].y);
      }
    }
  }
}

// dw[k] = sum over the CTAs' shares, in a fixed order.  32 columns x 32 row
// lanes a CTA.
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float* part, int n, int K, int w32,
                                                           void* dw) {
  __shared__ float sh[32][33];
  follow();
  const int k = blockIdx.x * 32 + (threadIdx.x & 31), rl = threadIdx.x >> 5;
  float s = 0.0f;
  if (k < K)
    for (int i = rl; i < n; i += 32) s += fetch(part + static_cast<int64_t>(i) * K + k);
  sh[rl][threadIdx.x & 31] = s;
  __syncthreads();
  s = warp_sum(sh[threadIdx.x & 31][rl]);
  const int kk = blockIdx.x * 32 + rl;
  if ((threadIdx.x & 31) == 0 && kk < K) {
    if (w32)
      static_cast<float*>(dw)[kk] = s;
    else
      static_cast<__nv_bfloat16*>(dw)[kk] = __float2bfloat16_rn(s);
  }
}

// Threads of a CTA that takes a row with two vectors a thread.
int row_threads(int nvec, int v) { return ((nvec + v - 1) / v + 31) / 32 * 32; }

// The backward's variant for a row length: as many CTAs of it as run at once on
// an SM (also given to the compiler), and the rows that a CTA takes at a time.
struct BwdShape {
  int threads, rows, per_sm;
};

BwdShape bwd_shape(int nvec) {
  if (nvec <= 16) return {SMALL_T, SMALL_T / 16, 4};
  if (nvec <= 32) return {SMALL_T, SMALL_T / 32, 4};
  if (nvec <= 64) return {SMALL_T, SMALL_T / 32, 3};
  const int t = row_threads(nvec, 2);
  return {t, 1, t <= 256 ? 768 / t : t <= 512 ? 2 : 1};
}

// CTAs of the backward (also the rows of its workspace).
int bwd_ctas(int64_t M, int nvec, int num_sms) {
  const BwdShape b = bwd_shape(nvec);
  const int64_t need = (M + b.rows - 1) / b.rows, most = static_cast<int64_t>(b.per_sm) * num_sms;
  return static_cast<int>(need < most ? need : most);
}

template <bool kQuant, bool kW32>
void launch_fwd(const FwdArgs& a, cudaStream_t st) {
  const int n = a.nvec;
  const auto ctas = [&](int lanes) {
    return static_cast<unsigned>((a.M + SMALL_T / lanes - 1) / (SMALL_T / lanes));
  };
  const unsigned rows = static_cast<unsigned>(a.M);
  if (n <= 16)
    launch_following(rms_norm_fwd_kernel<1, 16, kQuant, kW32>, ctas(16), SMALL_T, 0, st, a);
  else if (n <= 32)
    launch_following(rms_norm_fwd_kernel<1, 32, kQuant, kW32>, ctas(32), SMALL_T, 0, st, a);
  else if (n <= 64)
    launch_following(rms_norm_fwd_kernel<2, 32, kQuant, kW32>, ctas(32), SMALL_T, 0, st, a);
  else if (n <= 128)
    launch_following(rms_norm_fwd_kernel<4, 32, kQuant, kW32>, ctas(32), SMALL_T, 0, st, a);
  else if (n <= 1024)
    launch_following(rms_norm_fwd_kernel<2, 0, kQuant, kW32>, rows, row_threads(n, 2), 0, st, a);
  else  // CTAs of half the threads, more of them an SM: K = 12288 in bf16 59 -> 47 us (5461 rows)
    launch_following(rms_norm_fwd_kernel<4, 0, kQuant, kW32>, rows, row_threads(n, 4), 0, st, a);
}

// t: threads of a row that a CTA takes.  The shapes are bwd_shape's.
template <bool kW32>
void launch_bwd(const BwdArgs& a, int ctas, int t, cudaStream_t st) {
  const int n = a.nvec;
  if (n <= 16)
    rms_norm_bwd_kernel<1, 16, SMALL_T, 4, kW32><<<ctas, SMALL_T, 0, st>>>(a);
  else if (n <= 32)
    rms_norm_bwd_kernel<1, 32, SMALL_T, 4, kW32><<<ctas, SMALL_T, 0, st>>>(a);
  else if (n <= 64)
    rms_norm_bwd_kernel<2, 32, SMALL_T, 3, kW32><<<ctas, SMALL_T, 0, st>>>(a);
  else if (t <= 256)
    rms_norm_bwd_kernel<2, 0, 256, 3, kW32><<<ctas, t, 0, st>>>(a);
  else if (t <= 384)
    rms_norm_bwd_kernel<2, 0, 384, 2, kW32><<<ctas, t, 0, st>>>(a);
  else if (t <= 512)
    rms_norm_bwd_kernel<2, 0, 512, 2, kW32><<<ctas, t, 0, st>>>(a);
  else
    rms_norm_bwd_kernel<2, 0, 1024, 1, kW32><<<ctas, t, 0, st>>>(a);
}

}  // namespace rms
}  // namespace gl

static int launched(const char** why) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  *why = cudaGetErrorString(e);
  return -2;
}

// Launchers: 0 on a launch, -1 on a bad argument (why set), -2 on a launch error.
int gl_launch_rms_norm_fwd(const void* x, const void* residual, const void* weight, int w32, float eps,
                           int64_t M, int64_t K, void* h, void* y, void* q, float* s, float* rstd,
                           cudaStream_t st, const char** why) {
  using namespace gl::rms;
  FwdArgs a{static_cast<const uint4*>(x), static_cast<const uint4*>(residual), weight,
            static_cast<uint4*>(h), static_cast<uint4*>(y), static_cast<uint2*>(q), s, rstd, M,
            static_cast<int>(K / 8), 1.0f / static_cast<float>(K), eps};
  if (q)
    w32 ? launch_fwd<true, true>(a, st) : launch_fwd<true, false>(a, st);
  else
    w32 ? launch_fwd<false, true>(a, st) : launch_fwd<false, false>(a, st);
  return launched(why);
}

size_t gl_rms_norm_bwd_ws_bytes(int64_t M, int64_t K, int num_sms) {
  return static_cast<size_t>(gl::rms::bwd_ctas(M, static_cast<int>(K / 8), num_sms)) * K * sizeof(float);
}

int gl_launch_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* weight, int w32,
                           const float* rstd, int64_t M, int64_t K, void* dx, void* dw, void* ws,
                           cudaStream_t st, int num_sms, const char** why) {
  using namespace gl::rms;
  const int n = static_cast<int>(K / 8), t = row_threads(n, 2);
  const int ctas = bwd_ctas(M, n, num_sms);
  const BwdArgs a{static_cast<const uint4*>(dy), static_cast<const uint4*>(dh), static_cast<const uint4*>(h),
                  weight, rstd, static_cast<uint4*>(dx), static_cast<float*>(ws), M, n,
                  1.0f / static_cast<float>(K)};
  if (ctas > 0) {  // no rows: dw is a sum over nothing
    w32 ? launch_bwd<true>(a, ctas, t, st) : launch_bwd<false>(a, ctas, t, st);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
      *why = cudaGetErrorString(e);
      return -2;
    }
  }
  const cudaError_t e =
      gl::launch_following(rms_norm_dw_kernel, static_cast<unsigned>((K + 31) / 32), 1024, 0, st,
                           static_cast<const float*>(ws), ctas, static_cast<int>(K), w32, dw);
  if (e == cudaSuccess) return 0;
  *why = cudaGetErrorString(e);
  return -2;
}
