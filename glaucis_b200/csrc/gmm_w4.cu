// Grouped products with 4-bit weights and one fp32 scale per 128 weights of a
// column, for few rows (a decoding batch), and the quantiser of the weights.
//   out[m, n] = sum_b s[g, b, n] * sum_{k in block b} x[m, k] q[g, k, n]
// Format: q in -8..7, stored as the nibble u = q + 8; nibble j of the 32-bit
// word w4[g, i, n] is k = 8 i + j.
//
// With few rows the product reads each weight of the groups in use once and
// computes little with it: it is bound by HBM.  Three things must not get in
// the way: the work of widening 4-bit weights, gaps in the stream of loads, and
// what a call does before its first load.
//   * One launch.  A persistent CTA takes an equal share of all (tile of 8
//     rows, 512 columns, 128 k) units, cut at any k, so no SM waits for another
//     one's longer list.  One thread copies weights, scales and rows of x of the
//     units into a ring of shared-memory stages with TMA, running ahead across
//     tiles; eight warps take 64 columns each (with 32, what a unit costs besides
//     its weights held the product back).
//   * Where a share ends inside a tile's k, its fp32 sums go to the workspace;
//     when its share is done a warp counts its parts in, and whoever completes a
//     job's count adds the parts in order: the result does not depend on which
//     one that is, and nothing waits.  (Counting in at the job's end, amid the
//     loads, stood in their queue: 6 us of 20 for one token.)
//   * Weights go through mma.sync (m16n8k16, bf16 in, fp32 sums) as the 16-row
//     operand, 8 rows of x as the 8 columns: enough rate for a memory-bound
//     product.  (A tcgen05 tile would need the weights widened and written back
//     to shared memory first, and has 128 rows.)
//   * Both operands are exact: x as it was given, and q 2^-6 as a bf16 number,
//     which costs a masked nibble one packed FMA (eight weights: four ANDs, one
//     shift, four FMAs).  Left as they are, u = q + 8, the nibbles would cost no
//     FMA, with 8 sum(x) taken off the sum (one token 16.7 us for 17.9, 128 rows
//     62 for 67); but then an x whose weight is 0 leaves the rounding of 8 x
//     behind: with an outlier of 1e4 among x of unit size errors of 1e-2 in place
//     of 1e-6.
// Sums stay in fp32's range while those of |q x| in a block stay below 2^134.
// Measured in a CUDA graph (K 7168, N 2048, 128 groups): 128 rows in 44 groups 67
// us, 5.1 TB/s of weights and scales (64 us without finishing split jobs, 54.5 us
// without the sums too), 74 at the power cap of a loop; 8 rows in 8 groups 17.9 us
// (15.7, 11.9).
#include "common.cuh"

#include <atomic>

#include "tmap.h"

namespace gl {
namespace w4 {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int ROWS = 8;            // rows of a tile
constexpr int COLS = 512;          // columns of a unit: 64 for each of the
constexpr int WARPS = COLS / 64;   // consumer warps
constexpr int STAGES = 3;          // two CTAs an SM
constexpr int THREADS = 32 * (WARPS + 1);
constexpr int MIN_UNITS = 2;       // a share is no smaller: a part's way through the workspace costs more
// A stage as TMA leaves it: the weights, 32-column strips of 16 words a column;
// the scales; the rows of x, 64 features each, twice.  The 128-byte rows of
// weights and x are swizzled (16-byte chunk c of row r at c ^ (r & 7)).  In a
// 16-byte access phase lanes (gq, t), two gq and four t, read words 2 t + const
// of the weights: chunks gq ^ (2 t + const) are eight different bank groups; and
// of row gq of x the chunks 2 t + const, as many.
constexpr int S_OFF = COLS * 64;
constexpr int X_OFF = S_OFF + COLS * 4;
constexpr int X_BYTES = ROWS * 256;
constexpr int STAGE_BYTES = X_OFF + X_BYTES;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024;  // aligned to 1 KB inside
static_assert(X_OFF % 1024 == 0 && STAGE_BYTES % 1024 == 0, "swizzled rows start at 1 KB");

struct Args {
  const float* s;      // [G, K / 128, N]
  const int* sizes;
  unsigned long long* tags;  // [CTAs, WARPS]: the call's number << 16, plus parts that are there
  float* parts;              // [CTAs, 2, ROWS, COLS]
  unsigned long long nonce;
  int64_t M, N;
  int G, kb, strips;   // kb: K / 128; strips: 512-column strips of N
  void* out;
  int out_f32, zero_tail;
  int* err;
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// q 2^-6 of the nibbles 0 and 4 (lo) or 1 and 5 (hi) of a word, exact: a masked
// nibble u is the bf16 number u 2^-133, or 16 u 2^-133 four bits up (the step
// from the subnormals to the first normal ones, at u = 8, keeps the spacing).
__device__ __forceinline__ uint32_t weights_lo(uint32_t w) {
  return fma_bf16x2(w & 0x000F000Fu, 0x7F007F00u /* 2^127 */, 0xBE00BE00u /* -8 * 2^-6 */);
}

__device__ __forceinline__ uint32_t weights_hi(uint32_t w) {
  return fma_bf16x2(w & 0x00F000F0u, 0x7D007D00u /* 2^123 */, 0xBE00BE00u);
}

__device__ __forceinline__ uint4 lds4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}

__device__ __forceinline__ float4 lds4f(uint32_t addr) {
  const uint4 v = lds4(addr);
  return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}

__device__ __forceinline__ unsigned long long atom_add_acq_rel(unsigned long long* p, unsigned long long v) {
  unsigned long long old;
  asm volatile("atom.acq_rel.gpu.global.add.u64 %0, [%1], %2;" : "=l"(old) : "l"(p), "l"(v) : "memory");
  return old;
}

struct Tile {
  int group, row0, nrows;
};

// The groups' rows and tiles (8 rows of one group), held by a warp: 128
// groups a step, four consecutive ones a lane.  The step last looked at stays
// in registers.
struct Groups {
  const int* sizes;
  int G, M;
  int n[4], rows, tiles;        // the lane's four groups; inclusive sums over the step's lanes
  int rows_before, tiles_before, step;

  // Sizes past M are held at M + 1: sums stay in 32 bits (M <= 2^16, G <= 2^10).
  __device__ __forceinline__ bool load(int g0) {
    const int lane = threadIdx.x & 31;
    step = g0;
    rows = tiles = 0;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int g = g0 + 4 * lane + j;
      n[j] = g < G ? fetch(sizes + g) : 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bad = bad || n[j] < 0;
      n[j] = n[j] < 0 ? 0 : n[j] > M ? M + 1 : n[j];
      rows += n[j];
      tiles += (n[j] + ROWS - 1) / ROWS;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int r = __shfl_up_sync(FULL, rows, o), t = __shfl_up_sync(FULL, tiles, o);
      if (lane >= o) {
        rows += r;
        tiles += t;
      }
    }
    return bad;
  }

  // Number of tiles, and of rows; -1 when the sizes are not a partition of at
  // most M rows.
  __device__ __forceinline__ int count(int& total) {
    bool bad = false;
    rows_before = tiles_before = 0;
    for (int g0 = 0;; g0 += 128) {
      bad = load(g0) || bad;
      const int r = rows_before + __shfl_sync(FULL, rows, 31), t = tiles_before + __shfl_sync(FULL, tiles, 31);
      total = r;
      if (g0 + 128 >= G) return __any_sync(FULL, bad) || r > M ? -1 : t;
      rows_before = r;
      tiles_before = t;
    }
  }

  // Tile `want`, which exists.
  __device__ __forceinline__ Tile find(int want) {
    const int lane = threadIdx.x & 31;
    if (want < tiles_before) {
      rows_before = tiles_before = 0;
      load(0);
    }
    while (want >= tiles_before + __shfl_sync(FULL, tiles, 31)) {
      rows_before += __shfl_sync(FULL, rows, 31);
      tiles_before += __shfl_sync(FULL, tiles, 31);
      load(step + 128);
    }
    const int src = __ffs(__ballot_sync(FULL, want < tiles_before + tiles)) - 1;
    int t0 = tiles_before + tiles, r0 = rows_before + rows;
    Tile f = {0, 0, 0};
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      t0 -= (n[j] + ROWS - 1) / ROWS;
      r0 -= n[j];
      if (want >= t0 && want < t0 + (n[j] + ROWS - 1) / ROWS) {
        const int in = (want - t0) * ROWS;
        f.group = step + 4 * lane + j;
        f.row0 = r0 + in;
        f.nrows = n[j] - in < ROWS ? n[j] - in : ROWS;
      }
    }
    f.group = __shfl_sync(FULL, f.group, src);
    f.row0 = __shfl_sync(FULL, f.row0, src);
    f.nrows = __shfl_sync(FULL, f.nrows, src);
    return f;
  }
};

// The equal shares: unit u = (tile * strips + strip) * kb + block belongs to
// the CTA with start(c) <= u < start(c + 1); the first `longer` of them have
// one unit more.
struct Shares {
  uint32_t each, longer, ctas;
  __device__ __forceinline__ uint32_t start(uint32_t c) const { return c * each + (c < longer ? c : longer); }
  __device__ __forceinline__ uint32_t owner(uint32_t u) const {
    const uint32_t head = longer * (each + 1);
    return u < head ? u / (each + 1) : longer + (u - head) / each;
  }
};

// A CTA's share, unit by unit.
struct Walk {
  Groups groups;
  Tile tile;
  int job, block, at, strip;

  __device__ __forceinline__ void begin(const Args& a, uint32_t u0) {
    job = static_cast<int>(u0 / a.kb);
    block = static_cast<int>(u0 - static_cast<uint32_t>(job) * a.kb);
    at = job / a.strips;
    strip = job - at * a.strips;
    tile = groups.find(at);
  }
  // `more`: a further unit follows
  __device__ __forceinline__ void advance(const Args& a, bool more) {
    if (++block < a.kb) return;
    block = 0;
    ++job;
    if (++strip < a.strips) return;
    strip = 0;
    if (more) tile = groups.find(++at);
  }
};

struct Control {
  uint64_t full[STAGES], empty[STAGES];
  int rows[STAGES];  // rows of the stage's tile; negative where a job ends in this CTA
  int4 job[STAGES];  // then: the job, the tile's first row, its strip
  int4 part[2];      // row0, nrows, strip of the first and the last job, where the CTA has a part only
  Shares shares;
  int tail;          // first row to be zeroed
  int abort;
};

// The lane's sums as four pieces of four columns: piece e is row 2 t + (e & 1)
// of half e >> 1 of the warp's columns.
__device__ __forceinline__ float4 piece(const float (&tot)[4][4], int e) {
  const int h = 2 * (e >> 1), o = e & 1;
  return make_float4(tot[h][o], tot[h][2 + o], tot[h + 1][o], tot[h + 1][2 + o]);
}

__device__ __forceinline__ void store4(const Args& a, int64_t row, int64_t col, const float4& v) {
  const int64_t at = row * a.N + col;
  if (a.out_f32)
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = v;
  else
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
        make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

__device__ __forceinline__ void write_out(const Args& a, const float (&tot)[4][4], int row0, int nrows, int strip) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = 2 * (lane & 3) + (e & 1);
    const int64_t col = static_cast<int64_t>(strip) * COLS + warp * 64 + 32 * (e >> 1) + 4 * (lane >> 2);
    if (r < nrows && col < a.N) store4(a, row0 + static_cast<int64_t>(r), col, piece(tot, e));
  }
}

// Adds the parts of a job in the order of its CTAs: half a warp a row, four
// columns a lane, P pairs of rows from C parts in flight.
template <int P, int C>
__device__ __forceinline__ void add_parts(const Args& a, const int4& job, uint32_t from, uint32_t to,
                                          bool from_last) {
  const int warp = threadIdx.x >> 5, r0 = (threadIdx.x >> 4) & 1, c4 = threadIdx.x & 15;
  const int64_t col = static_cast<int64_t>(job.z) * COLS + warp * 64 + 4 * c4;
  const float* q = a.parts + r0 * COLS + warp * 64 + 4 * c4;
  float4 sum[P];
#pragma unroll
  for (int j = 0; j < P; ++j) sum[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (uint32_t c0 = from; c0 <= to; c0 += C) {
    float4 v[C][P];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t c = c0 + i;
      // the part is the CTA's first; only the first of the job's CTAs can have
      // begun with another job
      const uint32_t slot = 2 * c + (c == from && from_last ? 1 : 0);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        v[i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c <= to && r0 + 2 * j < job.y)
          v[i][j] = __ldcg(reinterpret_cast<const float4*>(q + static_cast<int64_t>(slot) * (ROWS * COLS) +
                                                           2 * j * COLS));
      }
    }
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) {
        sum[j].x += v[i][j].x;
        sum[j].y += v[i][j].y;
        sum[j].z += v[i][j].z;
        sum[j].w += v[i][j].w;
      }
  }
#pragma unroll
  for (int j = 0; j < P; ++j)
    if (r0 + 2 * j < job.y && col < a.N) store4(a, job.x + static_cast<int64_t>(r0 + 2 * j), col, sum[j]);
}

__global__ void __launch_bounds__(THREADS, 2) gmm_w4_kernel(const __grid_constant__ CUtensorMap wmap,
                                                            const __grid_constant__ CUtensorMap xmap,
                                                            const Args a) {
  constexpr int S = STAGES;
  extern __shared__ char smem_raw[];
  __shared__ Control ct;
  const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Abort ab{&ct.abort, a.err};
  Walk walk;
  follow(false);  // the next kernel starts when the loads are under way, not among them
  if (warp == WARPS) {
    walk.groups.sizes = a.sizes;
    walk.groups.G = a.G;
    walk.groups.M = static_cast<int>(a.M);
    int total = 0;
    const int tiles = walk.groups.count(total);
    if (lane == 0) {
      prefetch_tmap(&wmap);
      prefetch_tmap(&xmap);
      ct.abort = 0;
      ct.tail = tiles < 0 ? static_cast<int>(a.M) : total;
      if (tiles < 0 && blockIdx.x == 0) atomicExch(a.err, GL_DEV_BAD_GROUPS);
      const uint32_t units = tiles < 0 ? 0 : static_cast<uint32_t>(tiles) * a.strips * a.kb;
      const uint32_t most = (units + MIN_UNITS - 1) / MIN_UNITS;
      Shares sh;
      sh.ctas = most < gridDim.x ? most : gridDim.x;
      sh.each = sh.ctas ? units / sh.ctas : 0;
      sh.longer = sh.ctas ? units - sh.each * sh.ctas : 0;
      ct.shares = sh;
      for (int i = 0; i < S; ++i) {
        mbar_init(&ct.full[i], 1);
        mbar_init(&ct.empty[i], WARPS);
      }
      fence_mbar_init();
    }
  }
  __syncthreads();
  if (a.zero_tail && warp < WARPS) {  // while the first loads are under way
    const int64_t words = a.N * (a.out_f32 ? 4 : 2) / 16;
    for (int64_t i = ct.tail * words + static_cast<int64_t>(blockIdx.x) * (32 * WARPS) + threadIdx.x; i < a.M * words;
         i += static_cast<int64_t>(gridDim.x) * (32 * WARPS))
      static_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0);
  }
  const Shares sh = ct.shares;
  if (blockIdx.x >= sh.ctas) return;
  const uint32_t u0 = sh.start(blockIdx.x);
  const int units = static_cast<int>(sh.start(blockIdx.x + 1) - u0);

  if (warp == WARPS) {
    // ---- weights, scales and rows of x, and the stage's control words ----
    asm volatile("fence.proxy.async.global;" ::: "memory");  // after follow(): their writes, for the copies' proxy
    walk.begin(a, u0);
    int st = 0, n = 0;
    uint32_t phase = 1;  // the first round of stages is free
    for (; n < units; ++n) {
      if (n >= S && !mbar_wait(&ct.empty[st], phase, ab)) break;
      if (lane == 0) {
        const Tile& tile = walk.tile;
        const int64_t n0 = static_cast<int64_t>(walk.strip) * COLS;
        const uint32_t bytes = static_cast<uint32_t>((a.N - n0 < COLS ? a.N - n0 : COLS) * 4);
        const bool ends = walk.block == a.kb - 1 || n == units - 1;
        ct.rows[st] = ends ? -tile.nrows : tile.nrows;
        if (ends) ct.job[st] = make_int4(walk.job, tile.row0, walk.strip, 0);
        mbar_arrive_expect_tx(&ct.full[st], S_OFF + bytes + X_BYTES);
        char* dst = smem_raw + (smem - smem_u32(smem_raw)) + st * STAGE_BYTES;
        const int64_t kb = static_cast<int64_t>(tile.group) * a.kb + walk.block;
        // columns past N are filled with zeros and counted
        tma_load_3d(dst, &wmap, &ct.full[st], 0, static_cast<int>(kb * 16), walk.strip * (COLS / 32));
        bulk_load(dst + S_OFF, a.s + kb * a.N + n0, bytes, &ct.full[st]);
        // always 8 rows: those past the tile's are other rows of x, or zeros
        tma_load_3d(dst + X_OFF, &xmap, &ct.full[st], 0, tile.row0, 2 * walk.block);
      }
      walk.advance(a, n + 1 < units);
      if (++st == S) {
        st = 0;
        phase ^= 1;
      }
    }
    may_follow();
    // the copies land before the CTA may end, also when it gives up
    for (int i = n > S ? n - S : 0; i < n; ++i) {
      const uint64_t from = global_ns();
      while (!mbar_test(&ct.full[i % S], (i / S) & 1) && global_ns() - from < kWaitNs) {
      }
    }
    return;
  }

  // ---- consumers: 64 columns a warp; lane (gq, t) holds columns 4 gq .. 4 gq
  // + 3 of each half and four of the words k / 8 ----
  const int gq = lane >> 2, t = lane & 3;
  const uint32_t w_even = warp * 4096 + sw128_off(2 * t, gq), w_odd = warp * 4096 + sw128_off(2 * t + 1, gq);
  const uint32_t s_at = S_OFF + warp * 256 + gq * 16;
  const uint32_t x_even = X_OFF + sw128_off(gq, 2 * t), x_odd = X_OFF + sw128_off(gq, 2 * t + 1);
  // The jobs of which this CTA may have a part only, its first (lane 0) and its
  // last (lane 1), and the counts of their parts.  A count is taken over for
  // this call by whoever comes first; each of a job's CTAs looks before it adds
  // to it, so what the workspace held before does not matter, and the last one
  // clears it for a replayed call, whose number is the same.
  const uint32_t first_job = u0 / a.kb, last_job = (u0 + units - 1) / a.kb;
  const uint32_t own_job = lane == 0 ? first_job : last_job;
  const uint32_t own_from = sh.owner(own_job * a.kb), own_to = sh.owner(own_job * a.kb + a.kb - 1);
  const bool own_split = own_from != own_to && (lane == 0 || (lane == 1 && last_job != first_job));
  unsigned long long* const own_tag = a.tags + own_from * WARPS + warp;
  if (own_split) {
    unsigned long long old = *reinterpret_cast<volatile unsigned long long*>(own_tag);
    while (old >> 16 != a.nonce) {
      const unsigned long long seen = atomicCAS(own_tag, old, a.nonce << 16);
      if (seen == old) break;
      old = seen;
    }
  }
  __syncwarp();
  const bool split0 = __shfl_sync(FULL, own_split, 0), split1 = __shfl_sync(FULL, own_split, 1);
  float tot[4][4] = {};  // [column pair][row 2t, 2t + 1 of either column]
  int st = 0;
  uint32_t phase = 0;
  for (int n = 0; n < units; ++n) {
    if (!mbar_wait(&ct.full[st], phase, ab)) return;
    const int meta = ct.rows[st];
    const uint32_t p = smem + st * STAGE_BYTES;
    uint4 w[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h][0] = lds4(p + w_even + h * 2048);
      w[h][1] = lds4(p + w_odd + h * 2048);
      w[h][2] = lds4(p + w_even + h * 2048 + 1024);
      w[h][3] = lds4(p + w_odd + h * 2048 + 1024);
    }
    const float4 s0 = lds4f(p + s_at), s1 = lds4f(p + s_at + 128);
    // 2^6 of the weights
    const float sc[8] = {s0.x * 64.0f, s0.y * 64.0f, s0.z * 64.0f, s0.w * 64.0f,
                         s1.x * 64.0f, s1.y * 64.0f, s1.z * 64.0f, s1.w * 64.0f};
    // Rows past the tile's: a column of the matrix unit's result depends on its
    // own row of x alone, and theirs are not stored.
    const uint4 x[4] = {lds4(p + x_even), lds4(p + x_odd), lds4(p + x_even + 1024), lds4(p + x_odd + 1024)};
    float acc[4][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c[8] = {w[0][i].x, w[0][i].y, w[0][i].z, w[0][i].w,
                             w[1][i].x, w[1][i].y, w[1][i].z, w[1][i].w};
      // the features in the nibbles' order: 0 4, 1 5, 2 6, 3 7
      const uint32_t b0 = __byte_perm(x[i].x, x[i].z, 0x5410), b1 = __byte_perm(x[i].x, x[i].z, 0x7632);
      const uint32_t b2 = __byte_perm(x[i].y, x[i].w, 0x5410), b3 = __byte_perm(x[i].y, x[i].w, 0x7632);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint32_t l = c[2 * h], v = c[2 * h + 1];
        mma(acc[h], weights_lo(l), weights_lo(v), weights_hi(l), weights_hi(v), b0, b1);
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint32_t l = c[2 * h] >> 8, v = c[2 * h + 1] >> 8;
        mma(acc[h], weights_lo(l), weights_lo(v), weights_hi(l), weights_hi(v), b2, b3);
      }
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      tot[h][0] = fmaf(acc[h][0], sc[2 * h], tot[h][0]);
      tot[h][1] = fmaf(acc[h][1], sc[2 * h], tot[h][1]);
      tot[h][2] = fmaf(acc[h][2], sc[2 * h + 1], tot[h][2]);
      tot[h][3] = fmaf(acc[h][3], sc[2 * h + 1], tot[h][3]);
    }
    int4 job = make_int4(0, 0, 0, 0);
    if (meta < 0) job = ct.job[st];
    __syncwarp();
    if (lane == 0) mbar_arrive(&ct.empty[st]);
    if (++st == S) {
      st = 0;
      phase ^= 1;
    }
    if (meta >= 0) continue;

    // the job's end here: its output, or a part of it
    const int nrows = -meta;
    const bool is_first = static_cast<uint32_t>(job.x) == first_job;
    if (is_first ? split0 : split1 && static_cast<uint32_t>(job.x) == last_job) {
      const int slot = is_first ? 0 : 1;
      if (lane == 0) ct.part[slot] = make_int4(job.y, nrows, job.z, 0);  // the same from every warp
      float* part = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * (ROWS * COLS) + warp * 64 + 4 * gq;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (2 * t + (e & 1) < nrows)
          __stcg(reinterpret_cast<float4*>(part + (2 * t + (e & 1)) * COLS + 32 * (e >> 1)), piece(tot, e));
    } else {
      write_out(a, tot, job.y, nrows, job.z);
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) tot[h][0] = tot[h][1] = tot[h][2] = tot[h][3] = 0.0f;
  }

  // the share is done: its parts are counted in, after the warp's stores
  __syncwarp();
  int there = -1;
  if (own_split) there = static_cast<int>(atom_add_acq_rel(own_tag, 1) & 0xFFFF);
  const bool complete = own_split && there == static_cast<int>(own_to - own_from);
  if (complete) *own_tag = 0;
  __syncwarp();  // what the counting lane acquired, for the lanes that read the parts
#pragma unroll
  for (int l = 0; l < 2; ++l) {
    if (!__shfl_sync(FULL, complete, l)) continue;
    const uint32_t job = l == 0 ? first_job : last_job;
    const uint32_t from = __shfl_sync(FULL, own_from, l), to = __shfl_sync(FULL, own_to, l);
    const bool from_last = sh.start(from) / a.kb != job;
    const int4 pj = ct.part[l];
    if (pj.y <= 2)
      add_parts<1, 12>(a, pj, from, to, from_last);
    else if (pj.y <= 4)
      add_parts<2, 6>(a, pj, from, to, from_last);
    else
      add_parts<4, 3>(a, pj, from, to, from_last);
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

// CTAs of the product: two an SM.
int ctas(int num_sms) { return 2 * num_sms; }

// A number of its own for every call of the process (splitmix64, Steele et al. 2014, of a counter:
// nothing that a workspace is likely to hold).
unsigned long long next_nonce() {
  static std::atomic<uint64_t> calls{0};
  uint64_t z = calls.fetch_add(1, std::memory_order_relaxed) * 0x9E3779B97F4A7C15ull + 0xD1B54A32D192ED03ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  z ^= z >> 31;
  return z >> 16 ? z >> 16 : 1;  // 48 bits
}

}  // namespace w4
}  // namespace gl

// The tags and the parts of the shares.
size_t gl_gmm_w4_ws_bytes(int num_sms) {
  using namespace gl::w4;
  return static_cast<size_t>(ctas(num_sms)) * (WARPS * sizeof(unsigned long long) + 2 * ROWS * COLS * sizeof(float));
}

// Launchers: 0 on a launch, -1 on a bad argument, -2 on a launch error (why set).
int gl_launch_gmm_w4(const void* x, const void* w4, const float* s, const int32_t* group_sizes, int64_t G,
                     int64_t M, int64_t K, int64_t N, void* out, int out_f32, int zero_tail, void* ws,
                     int* err, cudaStream_t st, int num_sms, const char** why) {
  using namespace gl::w4;
  const int kb = static_cast<int>(K / 128), n = ctas(num_sms);
  const int64_t strips = (N + COLS - 1) / COLS;
  if ((M / ROWS + (M < G ? M : G)) * strips * kb > 0x7fffffff) {
    *why = "too large a product";
    return -1;
  }
  // 32 columns x words x strips of 32 columns: a box is 16 strips of 16 words
  CUtensorMap wmap, xmap;
  if (!gl_make_tmap_3d(&wmap, CU_TENSOR_MAP_DATA_TYPE_INT32, w4, 32, G * (K / 8), N / 32, N, 32, 32, 16,
                       COLS / 32, CU_TENSOR_MAP_SWIZZLE_128B, why))
    return -1;
  // 64 features x rows x 64-feature pieces: a box is two pieces of 8 rows
  if (!gl_make_tmap_3d(&xmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, 64, M, K / 64, K, 64, 64, ROWS, 2,
                       CU_TENSOR_MAP_SWIZZLE_128B, why))
    return -1;
  unsigned long long* tags = static_cast<unsigned long long*>(ws);
  float* parts = reinterpret_cast<float*>(tags + n * WARPS);
  const Args a{s, group_sizes, tags, parts, next_nonce(), M, N,
               static_cast<int>(G), kb, static_cast<int>(strips), out, out_f32, zero_tail, err};
  if (!gl_set_smem_attr(reinterpret_cast<const void*>(&gmm_w4_kernel), 0, SMEM_BYTES, why)) return -2;
  gl::launch_following(gmm_w4_kernel, n, THREADS, SMEM_BYTES, st, wmap, xmap, a);
  return launched(why);
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
