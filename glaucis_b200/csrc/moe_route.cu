// Router of a mixture of experts: softmax over E experts, the k largest logits
// of every token (ties to the lowest expert), the tokens each expert gets
// (group_sizes of the grouped matmul), the row of every choice when the
// choices are sorted by (expert, token, slot), and the balance loss
//   loss = E * sum_e f_e P_e,  f_e = counts_e / sum(counts),
//   P_e = mean of the softmax over the routed tokens;
// and the gradient of the logits for gradients of the weights and the loss.
//
// A warp takes a token, lane l holding the V experts from l V on: the softmax's
// sums and the k rounds of the selection are warp reductions on registers.
// Each lane keeps the largest of its own keys at hand, so a round is one
// redux.max for the key, a redux.min for the lowest expert that has it, and the
// winner's next key taking its place.  With E floats a token to read it is bound
// by issuing these instructions, mostly integer ones (460 a token of 128 experts
// and 8 choices), not by HBM.
//
// Rows need the counts of all earlier tokens: each CTA takes consecutive tokens
// and leaves its counts per expert, a second launch (not needed when one CTA
// takes all tokens) adds up those of the CTAs before it and ranks its choices
// in order.  Counts are integers and the loss's sums run in a fixed order over
// warps and CTAs: results do not depend on timing.
//
// Measured in a CUDA graph, 128 experts, top 8: 3 tokens 4.0 us, 4096 10 us, 32771
// with the gradient 39 us; 32768 tokens of 256 experts 37 us, 16384 of 384 42 us,
// 8192 of 1024 69 us.
#include "common.cuh"

#include <atomic>

namespace gl {
namespace route {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int MAX_CTAS = 148;

// Warps of a CTA: the per-warp rows of E values must fit 32 KB.
template <int V>
constexpr int warps() {
  return V <= 8 ? 32 : V == 16 ? 16 : 8;
}

struct Args {
  const void* logits;
  const uint8_t* mask;  // or null
  int64_t T;
  int E, k, f32, renorm;
  int vec;              // rows may be read in vectors
  int64_t chunk;        // tokens of a CTA
  int* ids;
  float* weights;
  int* counts;
  int* pos;
  float* loss;
  float* routed;        // routed tokens, as a float
  int* hist;            // [CTAs, E]     } of the first launch, for the second
  float* psum;          // [CTAs, E]     }
  int* live;            // [CTAs]        }
};

// Warps of a CTA of the second launch: more, where the first one's registers
// and rows of sums are not in the way.
template <int V>
constexpr int rank_warps() {
  return V <= 16 ? 32 : 16;
}

// W warps, P rows of sums.
template <int V, int W, int P>
struct Shared {
  union {
    float psum[P][32 * V];     // parts of the softmax's sum
    uint16_t cnt[W][32 * V];   // choices of an expert in a batch of entries
  };
  int hist[32 * V];   // this CTA's counts, then the row of an expert's next choice
  int total[32 * V];
  float red[2][32];
  int live;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}

// A load of what the caller passed in: off the read-only path where the kernel
// starts before the one in front of it is done (kFollows).
template <bool kFollows, class T>
__device__ __forceinline__ T get(const T* p) {
  return kFollows ? fetch(p) : __ldg(p);
}

template <bool kFollows>
__device__ __forceinline__ float load_logit(const void* p, int f32, int64_t i) {
  return f32 ? get<kFollows>(static_cast<const float*>(p) + i)
             : __bfloat162float(get<kFollows>(static_cast<const __nv_bfloat16*>(p) + i));
}

// Orders floats as unsigned integers (+0 and -0 alike); -inf and NaN, which
// are never chosen, give 0.
__device__ __forceinline__ uint32_t key_of(float z) {
  if (!(z > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(z + 0.0f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

template <int V>
using RouteShared = Shared<V, warps<V>(), warps<V>()>;  // a row of sums for every warp
template <int V>
using RankShared = Shared<V, rank_warps<V>(), (rank_warps<V>() > V ? rank_warps<V>() / V : 1)>;

// The lane's V logits of token t (experts lane V .. lane V + V - 1), -inf past
// the last expert and for a token that the mask takes out.
template <int V, bool kFollows>
__device__ __forceinline__ void load_token(const Args& a, int64_t t, float (&z)[V]) {
  const int e0 = (threadIdx.x & 31) * V;
  const bool kept = a.mask == nullptr || get<kFollows>(a.mask + t) != 0;
  const int64_t at = t * a.E + e0;
  if (a.vec) {
    const bool in = kept && e0 < a.E;  // V divides E: all of the lane's or none
    if (a.f32) {
      const float* p = static_cast<const float*>(a.logits) + at;
      if constexpr (V == 1) {
        z[0] = in ? get<kFollows>(p) : -INFINITY;
      } else if constexpr (V == 2) {
        const float2 v = in ? get<kFollows>(reinterpret_cast<const float2*>(p)) : make_float2(-INFINITY, -INFINITY);
        z[0] = v.x;
        z[1] = v.y;
      } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const float4 v = in ? get<kFollows>(reinterpret_cast<const float4*>(p + i))
                              : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          z[i] = v.x;
          z[i + 1] = v.y;
          z[i + 2] = v.z;
          z[i + 3] = v.w;
        }
      }
    } else {
      constexpr uint32_t kNegInf2 = 0xFF80FF80u;  // two bf16 -inf
      const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.logits) + at;
      if constexpr (V == 1) {
        z[0] = in ? __bfloat162float(get<kFollows>(p)) : -INFINITY;
      } else if constexpr (V < 8) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const uint32_t w = in ? get<kFollows>(reinterpret_cast<const uint32_t*>(p + i)) : kNegInf2;
          const float2 v = bf16x2_to_f32x2(w);
          z[i] = v.x;
          z[i + 1] = v.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; i += 8) {
          const uint4 u = in ? get<kFollows>(reinterpret_cast<const uint4*>(p + i))
                             : make_uint4(kNegInf2, kNegInf2, kNegInf2, kNegInf2);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 v = bf16x2_to_f32x2(w[j]);
            z[i + 2 * j] = v.x;
            z[i + 2 * j + 1] = v.y;
          }
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = kept && e0 + i < a.E ? load_logit<kFollows>(a.logits, a.f32, at + i) : -INFINITY;
  }
}

// A token takes part when a logit of it is not -inf (NaN takes part, to show).
template <int V>
__device__ __forceinline__ bool takes_part(const float (&z)[V]) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < V; ++i) any = any || z[i] != -INFINITY;
  return __any_sync(FULL, any);
}

// e^x for x <= 0 as 2^t (1 + d ln 2), t = x log2 e rounded and d what that rounding
// and the constant's own left out: within 2 ulp at every x, where 2^t alone is off
// by |x| 2^-24 relative.  Results below 2^-126 are 0; -inf, whose d has no value,
// is held at -200, and NaN goes through.  (32768 tokens of 128 experts, forward
// and gradient: 39.1 us, 38.1 with 2^t alone, 40.4 with expf.)
constexpr float LOG2E = 1.44269504f, LOG2E_LOW = 1.92596299e-8f;  // 24 bits and the next ones
constexpr float LN2 = 0.693147181f;

__device__ __forceinline__ float bounded(float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-200.0f));
  return x;
}

__device__ __forceinline__ float exp2_of(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

__device__ __forceinline__ float exp_of(float x) {
  x = bounded(x);
  const float t = x * LOG2E, r = exp2_of(t);
  return fmaf(r, fmaf(x, LOG2E_LOW, fmaf(x, LOG2E, -t)) * LN2, r);
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Two at once on packed f32x2 arithmetic.
__device__ __forceinline__ float2 exp_of(float2 x) {
  x = make_float2(bounded(x.x), bounded(x.y));
  const float2 nt = __fmul2_rn(x, both(-LOG2E));
  const float2 r = make_float2(exp2_of(-nt.x), exp2_of(-nt.y));
  const float2 d = __ffma2_rn(x, both(LOG2E_LOW), __ffma2_rn(x, both(LOG2E), nt));
  return __ffma2_rn(r, __fmul2_rn(d, both(LN2)), r);
}

// Softmax numerators e of the logits z (0 where z is -inf and zmax is not);
// returns 1 / their sum.
template <int V>
__device__ __forceinline__ float softmax(const float (&z)[V], float zmax, float (&e)[V]) {
  float2 s = both(0.0f);
  if constexpr (V == 1) {
    s.x = e[0] = exp_of(z[0] - zmax);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 v = exp_of(__fadd2_rn(make_float2(z[i], z[i + 1]), both(-zmax)));
      s = __fadd2_rn(s, v);
      e[i] = v.x;
      e[i + 1] = v.y;
    }
  }
  return __fdividef(1.0f, warp_sum(s.x + s.y));  // the sum is 1 to 1024: within 2 ulp
}

// A lane's keys and where they are, so that the largest is at hand and the next
// takes its place when it is chosen.  Fours of consecutive experts are kept
// sorted (equal keys in the experts' order, which stands in a word, a byte
// each), and the largest is that of the fours' heads; of 32, where the order of
// eight fours costs more than it saves (8192 tokens of 1024 experts: 84 us
// against 81; 16384 of 384, where it saves: 42 against 52), it is looked for again.
template <int V>
struct Keys {
  static constexpr bool kSorted = V <= 16;
  static constexpr int F = V < 4 ? V : 4, N = V / F;  // keys of a four, fours
  uint32_t key[V];
  uint32_t at[kSorted ? N : 1];  // kSorted: a four's experts, a byte each; else index of the largest
  uint32_t own;
  int four;   // whose head it is

  __device__ __forceinline__ void look() {
    own = key[0];
    if constexpr (kSorted) {
      four = 0;
#pragma unroll
      for (int n = 1; n < N; ++n)
        if (key[n * F] > own) {
          own = key[n * F];
          four = n;
        }
    } else {
      at[0] = 0;
#pragma unroll
      for (int i = 1; i < V; ++i)
        if (key[i] > own) {
          own = key[i];
          at[0] = i;
        }
    }
  }
  __device__ __forceinline__ void begin(const float (&z)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = key_of(z[i]);
    if constexpr (kSorted) {
      // exchange of neighbours only, which keeps equal keys in order
#pragma unroll
      for (int b = 0; b < N; ++b) {
        uint32_t x[F];
#pragma unroll
        for (int i = 0; i < F; ++i) x[i] = b * F + i;
#pragma unroll
        for (int n = F - 1; n > 0; --n)
#pragma unroll
          for (int i = 0; i < n; ++i) {
            uint32_t &p = key[b * F + i], &q = key[b * F + i + 1];
            const bool swap = q > p;
            const uint32_t k = swap ? p : q, t = swap ? x[i] : x[i + 1];
            p = swap ? q : p;
            x[i] = swap ? x[i + 1] : x[i];
            q = k;
            x[i + 1] = t;
          }
        at[b] = x[0];
#pragma unroll
        for (int i = 1; i < F; ++i) at[b] |= x[i] << (8 * i);
      }
    }
    look();
  }
  __device__ __forceinline__ int expert() const {
    uint32_t i = at[0];
    if constexpr (kSorted) {
#pragma unroll
      for (int n = 1; n < N; ++n) i = four == n ? at[n] : i;
    }
    return i;
  }
  // Takes the largest away (in the lane with `won`).
  __device__ __forceinline__ void next(bool won) {
    if constexpr (kSorted) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (won && (N == 1 || four == n)) {
#pragma unroll
          for (int i = n * F; i + 1 < (n + 1) * F; ++i) key[i] = key[i + 1];
          key[(n + 1) * F - 1] = 0;
          at[n] >>= 8;
        }
      }
      look();
    } else if (won) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i == at[0]) key[i] = 0;
      look();
    }
  }
};

// Routes tokens [t0, t1): ids, weights; counts into sh.hist, each warp's
// softmax sums into sh.psum and the number of routed tokens into sh.live.
template <int V, bool kFollows>
__device__ void route_tokens(const Args& a, int64_t t0, int64_t t1, RouteShared<V>& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < 32 * V; e += blockDim.x) sh.hist[e] = 0;
  if (threadIdx.x == 0) sh.live = 0;
  __syncthreads();
  float psum[V] = {}, next[V];
  int live = 0;
  if (t0 + warp < t1) load_token<V, kFollows>(a, t0 + warp, next);
  for (int64_t t = t0 + warp; t < t1; t += warps<V>()) {
    float z[V], e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = next[i];
    if (t + warps<V>() < t1) load_token<V, kFollows>(a, t + warps<V>(), next);
    int id = -1;
    float p = 0.0f;
    Keys<V> keys;
    keys.begin(z);
    uint32_t m = __reduce_max_sync(FULL, keys.own), mine = 0;
    if (m != 0 || takes_part<V>(z)) {  // a key, or NaN alone
      ++live;
      const float zmax = m ? of_key(m) : -INFINITY;
      const float inv = softmax<V>(z, zmax, e);
#pragma unroll
      for (int i = 0; i < V; ++i) psum[i] = fmaf(e[i], inv, psum[i]);
      for (int j = 0; m != 0; ) {  // 0: nothing left to choose
        const uint32_t x = keys.own == m ? lane * V + (keys.expert() & 255) : 0xffffu;
        const uint32_t at = __reduce_min_sync(FULL, x);
        if (lane == j) {
          id = at;
          mine = m;
        }
        if (++j == a.k) break;
        keys.next(x == at);
        m = __reduce_max_sync(FULL, keys.own);
      }
      if (id >= 0) p = exp_of(of_key(mine) - zmax) * inv;
      if (a.renorm) {
        // the quotient with its remainder put right (s is 2^-10 to 1): a single
        // choice has weight 1 exactly and no gradient
        const float s = warp_sum(p);
        const float r = __fdividef(1.0f, s), q = p * r;
        if (id >= 0) p = fmaf(fmaf(-q, s, p), r, q);
      }
    }
    if (lane < a.k) {
      const int n = static_cast<int>(t) * a.k + lane;  // T * topk fits 31 bits
      a.ids[n] = id;
      a.weights[n] = p;
      if (id >= 0) atomicAdd(&sh.hist[id], 1);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) sh.psum[warp][lane * V + i] = psum[i];
  if (lane == 0 && live) atomicAdd(&sh.live, live);
  __syncthreads();
}

// Exclusive scan of sh.total over the experts, added to sh.hist: warp 0, V
// consecutive experts a lane.
template <int V, class Sh>
__device__ __forceinline__ void add_scan(Sh& sh) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int n[V], own = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      n[i] = sh.total[lane * V + i];
      own += n[i];
    }
    int inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(FULL, inc, o);
      if (lane >= o) inc += v;
    }
    int run = inc - own;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sh.hist[lane * V + i] += run;
      run += n[i];
    }
  }
  __syncthreads();
}

// sh.total: choices of every expert; sh.hist: the first row of this CTA's
// choices of it.  `ctas` CTAs' counts, `cta` of them before this one.
template <int V, class Sh>
__device__ void first_rows(const Args& a, Sh& sh, int ctas, int cta) {
  for (int e = threadIdx.x; e < 32 * V; e += blockDim.x) sh.total[e] = sh.hist[e] = 0;
  __syncthreads();
  const int slices = blockDim.x >= 32 * V ? blockDim.x / (32 * V) : 1;
  for (int i = threadIdx.x; i < slices * 32 * V; i += blockDim.x) {
    const int e = i % (32 * V);
    if (e >= a.E) continue;
    int before = 0, total = 0;
#pragma unroll 16
    for (int b = i / (32 * V); b < ctas; b += slices) {
      const int h = __ldcg(a.hist + static_cast<int64_t>(b) * a.E + e);
      total += h;
      before += b < cta ? h : 0;
    }
    if (total) atomicAdd(&sh.total[e], total);
    if (before) atomicAdd(&sh.hist[e], before);
  }
  __syncthreads();
  add_scan<V>(sh);
}

// The warp's row of counts: only its own lanes write it before the next barrier.
template <int V, class Sh>
__device__ __forceinline__ void zero_counts(Sh& sh) {
  uint32_t* row = reinterpret_cast<uint32_t*>(sh.cnt[threadIdx.x >> 5]);
  for (int i = threadIdx.x & 31; i < 16 * V; i += 32) row[i] = 0;
  __syncwarp();
}

// Rows of the choices of tokens [t0, t1), a batch of one choice a thread at a
// time: rank among the batch's earlier choices of the same expert (within the
// warp by match, over the warps by a column of counts).  The warps' rows of
// counts are zero at the call.
template <int V, class Sh>
__device__ void assign_rows(const Args& a, Sh& sh, int64_t t0, int64_t t1) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n1 = t1 * a.k;
  int id = t0 * a.k + threadIdx.x < n1 ? a.ids[t0 * a.k + threadIdx.x] : -1;
  for (int64_t b = t0 * a.k; b < n1; b += blockDim.x) {
    const int64_t left = n1 - b, n = b + threadIdx.x;
    const int used = left < blockDim.x ? static_cast<int>((left + 31) / 32) : static_cast<int>(blockDim.x >> 5);
    const int next = n + blockDim.x < n1 ? a.ids[n + blockDim.x] : -1;
    const uint32_t same = __match_any_sync(FULL, id);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (id >= 0 && rank == 0) sh.cnt[warp][id] = static_cast<uint16_t>(__popc(same));
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
      int run = 0;
#pragma unroll 8
      for (int w = 0; w < used; ++w) {
        const int c = sh.cnt[w][e];
        sh.cnt[w][e] = static_cast<uint16_t>(run);
        run += c;
      }
      const int first = sh.hist[e];  // of the batch; this thread alone goes on with it
      sh.total[e] = first;
      sh.hist[e] = first + run;
    }
    __syncthreads();
    if (n < n1) a.pos[n] = id >= 0 ? sh.total[id] + sh.cnt[warp][id] + rank : -1;
    if (b + blockDim.x >= n1) break;
    __syncwarp();
    zero_counts<V>(sh);
    id = next;
  }
}

// counts and the loss: sh.total are all choices of an expert, sh.psum[0..rows)
// parts of the softmax's sum over `n` routed tokens.
template <int V, class Sh>
__device__ void finish(const Args& a, Sh& sh, int rows, int n) {
  float part = 0.0f, chosen = 0.0f;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    float p = 0.0f;
#pragma unroll 8
    for (int w = 0; w < rows; ++w) p += sh.psum[w][e];
    const int c = sh.total[e];
    a.counts[e] = c;
    part = fmaf(static_cast<float>(c), p, part);
    chosen += static_cast<float>(c);
  }
  part = warp_sum(part);
  chosen = warp_sum(chosen);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) {
    sh.red[0][warp] = part;
    sh.red[1][warp] = chosen;
  }
  __syncthreads();
  if (warp == 0) {
    part = warp_sum(lane < static_cast<int>(blockDim.x >> 5) ? sh.red[0][lane] : 0.0f);
    chosen = warp_sum(lane < static_cast<int>(blockDim.x >> 5) ? sh.red[1][lane] : 0.0f);
    if (lane == 0) {
      const float tokens = static_cast<float>(max(n, 1));
      *a.loss = static_cast<float>(a.E) * (part / fmaxf(chosen, 1.0f) / tokens);
      *a.routed = tokens;
    }
  }
}

// One CTA takes every token.
template <int V>
__global__ void __launch_bounds__(32 * warps<V>(), 1) route_one_kernel(const Args a) {
  __shared__ RouteShared<V> sh;
  follow();
  route_tokens<V, true>(a, 0, a.T, sh);
  for (int e = threadIdx.x; e < 32 * V; e += blockDim.x) {
    sh.total[e] = sh.hist[e];
    sh.hist[e] = 0;
  }
  __syncthreads();
  finish<V>(a, sh, a.T < warps<V>() ? static_cast<int>(a.T) : warps<V>(), sh.live);
  add_scan<V>(sh);
  zero_counts<V>(sh);
  assign_rows<V>(a, sh, 0, a.T);
}

// First of two launches: the choices, and what the CTA adds to counts and loss.
// Up to 128 experts it keeps to half of an SM's registers, so that the second
// launch's CTAs start beside it (65536 tokens of 128: 45 us against 51).
template <int V>
__global__ void __launch_bounds__(32 * warps<V>(), V <= 4 ? 2 : 1) route_kernel(const Args a) {
  __shared__ RouteShared<V> sh;
  may_follow();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.chunk;
  const int64_t t1 = t0 + a.chunk < a.T ? t0 + a.chunk : a.T;
  route_tokens<V, false>(a, t0, t1, sh);
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    float s = 0.0f;
#pragma unroll 8
    for (int w = 0; w < warps<V>(); ++w) s += sh.psum[w][e];
    a.psum[static_cast<int64_t>(blockIdx.x) * a.E + e] = s;
    a.hist[static_cast<int64_t>(blockIdx.x) * a.E + e] = sh.hist[e];
  }
  if (threadIdx.x == 0) a.live[blockIdx.x] = sh.live;
}

// Second launch: the CTAs of the first rank their choices, one more finishes.
template <int V>
__global__ void __launch_bounds__(32 * rank_warps<V>()) rank_kernel(const Args a) {
  __shared__ RankShared<V> sh;
  const int ctas = gridDim.x - 1, cta = blockIdx.x;
  const int64_t t0 = static_cast<int64_t>(cta) * a.chunk;
  const int64_t t1 = t0 + a.chunk < a.T ? t0 + a.chunk : a.T;
  zero_counts<V>(sh);
  follow();
  first_rows<V>(a, sh, ctas, cta);
  if (cta == ctas) {
    // the CTAs' softmax sums, in as many slices as there are threads for
    const int slices = blockDim.x >= 32 * V ? blockDim.x / (32 * V) : 1;
    for (int i = threadIdx.x; i < slices * 32 * V; i += blockDim.x) {
      const int e = i % (32 * V);
      float s = 0.0f;
      if (e < a.E) {
#pragma unroll 16
        for (int b = i / (32 * V); b < ctas; b += slices) s += __ldcg(a.psum + static_cast<int64_t>(b) * a.E + e);
      }
      sh.psum[i / (32 * V)][e] = s;
    }
    int n = 0;
    for (int b = threadIdx.x & 31; b < ctas; b += 32) n += __ldcg(a.live + b);
    n = __reduce_add_sync(FULL, n);
    __syncthreads();
    finish<V>(a, sh, slices, n);
    return;
  }
  assign_rows<V>(a, sh, t0, t1);
}

struct BwdArgs {
  const int* ids;
  const float* weights;
  const int* counts;
  const float* routed;
  const float* dweights;  // or null
  const float* dloss;     // or null
  void* dlogits;
};

__device__ __forceinline__ void store_logit(void* p, int f32, int64_t i, float v) {
  if (f32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// The lane's V values of token t's row.
template <int V>
__device__ __forceinline__ void store_token(const Args& a, void* out, int64_t t, const float (&v)[V]) {
  const int e0 = (threadIdx.x & 31) * V;
  const int64_t at = t * a.E + e0;
  if (a.vec && V > 1) {
    if (e0 >= a.E) return;
    if (a.f32) {
      float* p = static_cast<float*>(out) + at;
      if constexpr (V == 2) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
      } else if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4)
          *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    } else {
      __nv_bfloat16* p = static_cast<__nv_bfloat16*>(out) + at;
      if constexpr (V >= 8) {
#pragma unroll
        for (int i = 0; i < V; i += 8)
          *reinterpret_cast<uint4*>(p + i) =
              make_uint4(pack_bf16x2(v[i], v[i + 1]), pack_bf16x2(v[i + 2], v[i + 3]),
                         pack_bf16x2(v[i + 4], v[i + 5]), pack_bf16x2(v[i + 6], v[i + 7]));
      } else if constexpr (V >= 2) {
#pragma unroll
        for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(p + i) = pack_bf16x2(v[i], v[i + 1]);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e0 + i < a.E) store_logit(out, a.f32, at + i, v[i]);
}

// dlogit_e = p_e (c_e - sum_e' p_e' c_e'), c_e = dloss E f_e / n for the loss; for
// the gradient d of the chosen experts' weights w plus w_e (d_e - sum_e' w_e' d_e')
// on those, or, where w is p as it is, p_e d_e there less p_e sum_e' p_e' d_e'
// everywhere.
// Five CTAs an SM with up to two experts a lane: 22.1 us for 65536 tokens of 64, 24.4
// with the four that its registers would leave.
template <int V>
__global__ void __launch_bounds__(256, V <= 2 ? 5 : 0) route_bwd_kernel(const Args a, const BwdArgs b) {
  const int lane = threadIdx.x & 31;
  // a token's logits and choices, read one token ahead
  float next[V], w_next = 0.0f, sel_next = 0.0f;
  int id_next = -1;
  auto load = [&](int64_t t) {
    load_token<V, false>(a, t, next);
    if (lane < a.k) {
      id_next = __ldg(b.ids + t * a.k + lane);
      w_next = __ldg(b.weights + t * a.k + lane);
      sel_next = b.dweights ? __ldg(b.dweights + t * a.k + lane) : 0.0f;
    }
  };
  int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (t < a.T) load(t);
  float c[V], chosen = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane * V + i;
    c[i] = e < a.E ? static_cast<float>(__ldg(b.counts + e)) : 0.0f;
    chosen += c[i];
  }
  chosen = fmaxf(warp_sum(chosen), 1.0f);
  const float scale = b.dloss ? __ldg(b.dloss) * static_cast<float>(a.E) / __ldg(b.routed) / chosen : 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] *= scale;
  const int64_t warps_all = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (; t < a.T; t += warps_all) {
    float z[V], e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = next[i];
    int id = id_next;
    float w = w_next, sel = sel_next;
    if (id < 0 || id >= a.E) {
      id = -1;
      sel = 0.0f;
    }
    if (t + warps_all < a.T) load(t + warps_all);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, key_of(z[i]));
    m = __reduce_max_sync(FULL, m);
    if (m == 0 && !takes_part<V>(z)) {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = 0.0f;
      store_token<V>(a, b.dlogits, t, e);
      continue;
    }
    const float zmax = m ? of_key(m) : -INFINITY;
    const float inv = softmax<V>(z, zmax, e);
    // the chosen experts' share, in the lane that holds the choice
    const float p_sel = id >= 0 ? exp_of(load_logit<false>(a.logits, a.f32, t * a.E + id) - zmax) * inv : 0.0f;
    // what the weights add to its logit, and to the sum over the row: none where
    // the weights are over their sum
    float add = p_sel * sel, dot = add;
    if (a.renorm) {
      const float mean = warp_sum(id >= 0 ? sel * w : 0.0f);
      add = id >= 0 ? w * (sel - mean) : 0.0f;
      dot = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      e[i] *= inv;
      dot = fmaf(e[i], c[i], dot);
    }
    dot = warp_sum(dot);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] *= c[i] - dot;
    store_token<V>(a, b.dlogits, t, e);
    __syncwarp();
    // the chosen experts' values over those just written (other lanes' stores,
    // ordered by the warp's barrier)
    if (id >= 0)
      store_logit(b.dlogits, a.f32, t * a.E + id,
                  fmaf(p_sel, static_cast<float>(__ldg(b.counts + id)) * scale - dot, add));
  }
}

// Warps of a forward CTA for E experts.
int fwd_warps(int64_t E) { return E <= 256 ? warps<8>() : E <= 512 ? warps<16>() : warps<32>(); }

// CTAs of the forward: one when a token each is enough for its warps, or two
// with one or two choices each, else one per SM at most.  The second launch
// costs less than a second round of 8 choices (64 tokens of 128 experts: 7.3 us
// against 8.7), more than one of 2 (33 to 64 tokens of 8: 5.9 to 6.2 against 5.0
// to 5.5).
int fwd_ctas(int64_t T, int64_t k, int w, int num_sms) {
  if (T <= (k <= 2 ? 2 * w : w)) return 1;
  const int64_t need = (T + w - 1) / w;
  const int most = num_sms < MAX_CTAS ? num_sms : MAX_CTAS;
  return static_cast<int>(need < most ? need : most);
}

template <int V>
int fwd(const Args& a0, int num_sms, cudaStream_t st, const char** why) {
  Args a = a0;
  const int ctas = fwd_ctas(a.T, a.k, warps<V>(), num_sms);
  a.chunk = a.T > 0 ? (a.T + ctas - 1) / ctas : 1;
  cudaError_t e;
  if (ctas == 1) {
    e = launch_following(route_one_kernel<V>, 1, 32 * warps<V>(), 0, st, a);
  } else {
    route_kernel<V><<<ctas, 32 * warps<V>(), 0, st>>>(a);
    e = cudaGetLastError();
    if (e == cudaSuccess) {
      e = launch_following(rank_kernel<V>, ctas + 1, 32 * rank_warps<V>(), 0, st, a);
    }
  }
  if (e == cudaSuccess) return 0;
  *why = cudaGetErrorString(e);
  return -2;
}

template <int V>
int bwd(const Args& a, const BwdArgs& b, int num_sms, cudaStream_t st, const char** why) {
  const int64_t need = (a.T + 7) / 8;
  static std::atomic<int> fit{0};  // CTAs of an SM, the same on every B200
  int per_sm = fit.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    const cudaError_t q = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, route_bwd_kernel<V>, 256, 0);
    if (q != cudaSuccess) {
      *why = cudaGetErrorString(q);
      return -2;
    }
    fit.store(per_sm, std::memory_order_relaxed);
  }
  const int64_t most = static_cast<int64_t>(num_sms) * per_sm;
  route_bwd_kernel<V><<<static_cast<unsigned>(need < most ? need : most), 256, 0, st>>>(a, b);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  *why = cudaGetErrorString(e);
  return -2;
}

}  // namespace route
}  // namespace gl

static bool vectors(const void* logits, int f32, int64_t E, int v) {
  const int64_t bytes = v * (f32 ? 4 : 2);
  return E % v == 0 && reinterpret_cast<uintptr_t>(logits) % (bytes < 16 ? bytes : 16) == 0;
}

// Experts of a lane.
static int lane_experts(int64_t E) {
  int v = 1;
  while (v * 32 < E) v *= 2;
  return v;
}

// hist and psum of every CTA, then its number of routed tokens; none for one
// CTA whatever the number of choices.
size_t gl_moe_route_ws_bytes(int64_t T, int64_t E) {
  using namespace gl::route;
  if (fwd_ctas(T, GL_MOE_MAX_TOPK, fwd_warps(E), MAX_CTAS) == 1) return 0;
  return static_cast<size_t>(MAX_CTAS) * (2 * static_cast<size_t>(E) + 1) * 4;
}

// Launchers: 0 on a launch, -2 on a launch error (why set).
int gl_launch_moe_route_fwd(const void* logits, int f32, const void* mask, int64_t T, int64_t E, int64_t k,
                            int renorm, int32_t* ids, float* weights, int32_t* counts, int32_t* pos,
                            float* loss, float* routed, void* ws, cudaStream_t st, int num_sms,
                            const char** why) {
  using namespace gl::route;
  const int v = lane_experts(E);
  Args a = {};
  a.logits = logits;
  a.mask = static_cast<const uint8_t*>(mask);
  a.T = T;
  a.E = static_cast<int>(E);
  a.k = static_cast<int>(k);
  a.f32 = f32;
  a.renorm = renorm;
  a.vec = vectors(logits, f32, E, v);
  a.ids = ids;
  a.weights = weights;
  a.counts = counts;
  a.pos = pos;
  a.loss = loss;
  a.routed = routed;
  if (ws) {
    a.hist = static_cast<int*>(ws);
    a.psum = reinterpret_cast<float*>(a.hist + MAX_CTAS * E);
    a.live = reinterpret_cast<int*>(a.psum + MAX_CTAS * E);
  }
  switch (v) {
    case 1: return fwd<1>(a, num_sms, st, why);
    case 2: return fwd<2>(a, num_sms, st, why);
    case 4: return fwd<4>(a, num_sms, st, why);
    case 8: return fwd<8>(a, num_sms, st, why);
    case 16: return fwd<16>(a, num_sms, st, why);
    default: return fwd<32>(a, num_sms, st, why);
  }
}

int gl_launch_moe_route_bwd(const void* logits, int f32, const void* mask, const int32_t* ids,
                            const float* weights, const int32_t* counts, const float* routed,
                            const float* dweights, const float* dloss, int64_t T, int64_t E, int64_t k,
                            int renorm, void* dlogits, cudaStream_t st, int num_sms, const char** why) {
  using namespace gl::route;
  const int v = lane_experts(E);
  Args a = {};
  a.logits = logits;
  a.mask = static_cast<const uint8_t*>(mask);
  a.T = T;
  a.E = static_cast<int>(E);
  a.k = static_cast<int>(k);
  a.f32 = f32;
  a.renorm = renorm;
  a.vec = vectors(logits, f32, E, v) && vectors(dlogits, f32, E, v);
  const BwdArgs b{ids, weights, counts, routed, dweights, dloss, dlogits};
  switch (v) {
    case 1: return bwd<1>(a, b, num_sms, st, why);
    case 2: return bwd<2>(a, b, num_sms, st, why);
    case 4: return bwd<4>(a, b, num_sms, st, why);
    case 8: return bwd<8>(a, b, num_sms, st, why);
    case 16: return bwd<16>(a, b, num_sms, st, why);
    default: return bwd<32>(a, b, num_sms, st, why);
  }
}
