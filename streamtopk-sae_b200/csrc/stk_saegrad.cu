// Gradient of the top-k SAE over its sparse codes (stk_sae_backward).
//
//   x_hat_b = b_dec + sum_j v_bj W_dec[i_bj],   v_bj = x_b . W_enc[i_bj] + b_enc[i_bj]
//   dv_bj     = g_b . W_dec[i_bj] (+ a given gradient of v)
//   dW_dec[f] = sum over the codes (b, j) of feature f of v_bj g_b
//   dW_enc[f] = ...                                    of dv_bj x_b
//   db_enc[f] = ... of dv_bj        db_dec = sum_b g_b        dX_b = sum_j dv_bj W_enc[i_bj]
//
// The codes are first sorted by feature, codes of one feature by their place in
// (b, j): a radix sort, since sums over an order that atomics left to chance
// would differ from call to call.  Then one kernel walks the features: a
// feature's row of W_dec is read once, the g rows of its codes are gathered
// once for both the dot products dv and the sum dW_dec, and, with dv known, the
// x rows for dW_enc.  Dictionary-sized memory is touched once each: W_dec read,
// dW_dec and dW_enc written.
#include <algorithm>
#include <cmath>

#include "../../include/stk_b200.h"
#include "stk_host.h"
#include "stk_vec.cuh"

namespace stk {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxPart = 256;     // codes of one feature that one warp sums at most; longer lists are split and joined
constexpr int kMinPart = 32;
constexpr int64_t kPartBytes = 256 << 20;  // bound of the workspace for parts' sums (while parts are below kMaxPart)
constexpr int kShort = 8;         // lists up to this length stay in registers
constexpr int kSmallCodes = 8192; // up to this many codes one CTA sorts, while the others zero the gradients
constexpr int kSmallThreads = 1024;
constexpr int kSmallRounds = kSmallCodes / kSmallThreads;
constexpr int kZeroBytes = 8 * 16 * kSmallThreads;  // that a CTA zeroes at a time
constexpr int kSmallBits = 9;     // of a radix digit there
constexpr int kTile = 1024;       // codes per CTA of a radix pass
constexpr int kTileThreads = 256;
constexpr int kTileWarps = kTileThreads / 32;
constexpr int kMaxBits = 11;      // of a radix digit
constexpr int kGradWarps = 4;
constexpr int kGradCtas = 4;      // per SM: with 128 registers a thread; 5, 6 or 8 with fewer measured the same or worse

// A list of more than kShort codes, or a part of one: `first` is the list's
// first row of partial sums in the workspace, `part` < `parts` its place (one part: no such rows).
struct Part {
  int feature, begin, n, part, first, parts;
};

struct Group {
  uint32_t* key[2];
  uint32_t* id[2];
  int* count;      // [bins][tiles] of a pass
  int* total;      // [bins]
  int* start;      // [F + 1] first code of each feature, in sorted order; small: [segments + 1] and
  int* feature;    // [segments]
  int* state;      // [0] segments (small), [1] long lists and parts, [2] rows of partial sums, [3] the next list
  int* arrived;    // [slots] parts that are done, at their list's first row
  Part* part;
  float* part_dec;
  float* part_enc;
  float* part_b;
  float* colsum;   // [chunks][d]
  int* col_arrived;
  float* zeros;    // [d]
};

struct GradArgs {
  const float* g;
  const void* X;
  const void* W_dec;
  const void* W_enc;
  const float* V;
  const int32_t* I;
  const float* gv;
  void* dW_enc;
  float* db_enc;
  void* dW_dec;
  float* db_dec;
  float* dv;
  void* dX;
  int64_t B, F, d, N;
  int k, small, final_buf, log_codes, part;  // part: longest list that is not split
  int chunks;       // row chunks of the column sum of g
  Group grp;
};

// Each kernel of a call is launched while the one before it ends (programmatic
// dependent launch: 471 to 452 us for seven kernels in a row); it touches memory
// only after this.  No kernel lets the next one in before its end: CTAs that wait
// take the place of CTAs that work (452 to 470 us).
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ uint32_t feature_key(const GradArgs& a, int64_t e) {
  const int32_t f = a.I[e];
  const bool ok = f >= 0 && (int64_t)f < a.F;
  if (!ok && a.dv != nullptr) a.dv[e] = 0.f;  // codes that are skipped
  return ok ? (uint32_t)f : (uint32_t)a.F;
}

// ---------------------------------------------------------------------------
// Column sum of g: 128 columns x a chunk of rows per CTA turn, the last chunk
// of a column block to arrive adds all chunks in order.
// ---------------------------------------------------------------------------
template <int WARPS>
__device__ void column_sum(const GradArgs& a, int64_t unit) {
  __shared__ float sm[WARPS][128];
  __shared__ int last;
  const int64_t cb = unit / a.chunks, chunk = unit % a.chunks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rows = (a.B + a.chunks - 1) / a.chunks;
  const int64_t r0 = chunk * rows, r1 = min(a.B, r0 + rows);
  __syncthreads();
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int64_t r = r0 + warp; r < r1; r += WARPS)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t c = cb * 128 + i * 32 + lane;
      acc[i] += c < a.d ? __ldg(&a.g[r * a.d + c]) : 0.f;
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) sm[warp][i * 32 + lane] = acc[i];
  __syncthreads();
  const int64_t c = cb * 128 + threadIdx.x;
  const bool mine = threadIdx.x < 128 && c < a.d;
  float s = 0.f;
  if (mine) {
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += sm[w][threadIdx.x];
    if (a.chunks > 1) a.grp.colsum[chunk * a.d + c] = s;
    else a.db_dec[c] = s;
  }
  if (a.chunks == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&a.grp.col_arrived[cb], 1) == a.chunks - 1;
  __syncthreads();
  if (last && mine) {
    __threadfence();
    s = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.chunks; ++i) s += __ldcg(&a.grp.colsum[i * a.d + c]);
    a.db_dec[c] = s;
  }
}

// ---------------------------------------------------------------------------
// Few codes: CTA 0 sorts them in shared memory and lists the features that
// have any; the other CTAs zero the gradients (most rows stay zero) and sum
// g's columns meanwhile.
// ---------------------------------------------------------------------------
__device__ void zero_fill(void* p, int64_t bytes, int cta, int ctas) {
  // 16-byte streaming stores, eight per thread and 128 KB per CTA in a row; with a CTA for each 128 KB (the launch)
  // 201 MB at 6.4 TB/s, with two CTAs an SM that walk over it at 5.5.
  uint8_t* const b = static_cast<uint8_t*>(p);
  const int64_t head = min(bytes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15));
  const int64_t body = (bytes - head) / 16;
  uint4* const v = reinterpret_cast<uint4*>(b + head);
  constexpr int kTurn = kZeroBytes / 16;
  for (int64_t j = (int64_t)cta * kTurn; j < body; j += (int64_t)ctas * kTurn) {
    if (j + kTurn <= body) {
#pragma unroll
      for (int u = 0; u < 8; ++u) __stcs(&v[j + u * kSmallThreads + threadIdx.x], make_uint4(0, 0, 0, 0));
    } else {
      for (int64_t i = j + threadIdx.x; i < body; i += kSmallThreads) v[i] = make_uint4(0, 0, 0, 0);
    }
  }
  if (cta == 0) {
    if (threadIdx.x < head) b[threadIdx.x] = 0;
    const int64_t tail = head + body * 16 + threadIdx.x;
    if (tail < bytes) b[tail] = 0;
  }
}

__device__ int scan_1024(int v, int* sm, int* total) {  // exclusive, over the 1024 threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = sm[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(kFull, w, o);
      if (lane >= o) w += y;
    }
    sm[lane] = w;
  }
  __syncthreads();
  *total = sm[31];
  return x - v + (warp ? sm[warp - 1] : 0);
}

// Lists a feature's codes as parts of at most a.part.  (The order of the lists,
// which the atomics leave open, has no influence on any sum.)
__device__ void add_long(const GradArgs& a, int feature, int begin, int n) {
  const int parts = (n + a.part - 1) / a.part, at = atomicAdd(&a.grp.state[1], parts);
  int first = 0;
  if (parts > 1) {
    first = atomicAdd(&a.grp.state[2], parts);
    a.grp.arrived[first] = 0;
  }
  for (int p = 0; p < parts; ++p)
    a.grp.part[at + p] = Part{feature, begin + p * a.part, min(a.part, n - p * a.part), p, first, parts};
}

struct SmallSort {
  uint32_t key[kSmallCodes];
  uint16_t id[kSmallCodes];
  uint16_t hist[32 << kSmallBits];  // [digit][warp]: in this order its running sums are the sorted places
  int sm[32];
};

__global__ void __launch_bounds__(kSmallThreads) small_group_kernel(const __grid_constant__ GradArgs a, int key_bits,
                                                                    int64_t dict_bytes) {
  after_previous();
  extern __shared__ uint4 small_smem[];
  if (blockIdx.x > 0) {
    const int cta = blockIdx.x - 1, ctas = gridDim.x - 1;
    if (a.db_dec != nullptr)  // one chunk: no counters, which CTA 0 may not have cleared yet
      for (int64_t u = cta; u < (a.d + 127) / 128; u += ctas) column_sum<kSmallThreads / 32>(a, u);
    if (a.dW_dec != nullptr) zero_fill(a.dW_dec, dict_bytes, cta, ctas);
    if (a.dW_enc != nullptr) zero_fill(a.dW_enc, dict_bytes, ctas - 1 - cta, ctas);
    if (a.db_enc != nullptr) zero_fill(a.db_enc, a.F * 4, cta, ctas);
    return;
  }
  SmallSort& s = *reinterpret_cast<SmallSort*>(small_smem);
  for (int64_t i = threadIdx.x; i < a.d; i += kSmallThreads) a.grp.zeros[i] = 0.f;
  int* const sm = s.sm;
  const int t = threadIdx.x, N = (int)a.N, lane = t & 31, warp = t >> 5;
  const int rounds = (N + kSmallThreads - 1) / kSmallThreads;
  // Warp w has the 32 * rounds codes from there on, 32 in a round.
  const int base = warp * 32 * rounds + lane;
  uint32_t key[kSmallRounds], id[kSmallRounds];
#pragma unroll
  for (int r = 0; r < kSmallRounds; ++r) {
    const int i = base + r * 32;
    id[r] = (uint32_t)i;
    key[r] = r < rounds && i < N ? feature_key(a, i) : 0xffffffffu;
  }
  for (int shift = 0; shift < key_bits; shift += kSmallBits) {
    const int bits = min(kSmallBits, key_bits - shift), places = 32 << bits;
    const uint32_t mask = (1u << bits) - 1u;
    for (int i = t * 8; i < places; i += kSmallThreads * 8) *reinterpret_cast<uint4*>(&s.hist[i]) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint16_t rank[kSmallRounds];
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
      if (r < rounds) {
        const bool in = base + r * 32 < N;
        const uint32_t digit = in ? (key[r] >> shift) & mask : 0xffffffffu;
        const uint32_t same = __match_any_sync(kFull, digit);
        uint16_t* const h = &s.hist[(in ? digit : 0) * 32 + warp];
        const int before = *h;
        __syncwarp();
        if (in && (same & ((1u << lane) - 1u)) == 0u) *h = (uint16_t)(before + __popc(same));
        __syncwarp();
        rank[r] = (uint16_t)(before + __popc(same & ((1u << lane) - 1u)));
      }
    }
    __syncthreads();
    const int per = places / kSmallThreads > 0 ? places / kSmallThreads : 1, first = t * per;
    int sum = 0, total;
    if (first < places)
      for (int i = 0; i < per; ++i) sum += s.hist[first + i];
    int run = scan_1024(sum, sm, &total);
    if (first < places)
      for (int i = 0; i < per; ++i) {
        const int c = s.hist[first + i];
        s.hist[first + i] = (uint16_t)run;
        run += c;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r)
      if (r < rounds && base + r * 32 < N) {
        const int at = s.hist[((key[r] >> shift) & mask) * 32 + warp] + rank[r];
        s.key[at] = key[r];
        s.id[at] = (uint16_t)id[r];
      }
    __syncthreads();
    if (shift + kSmallBits < key_bits)
#pragma unroll
      for (int r = 0; r < kSmallRounds; ++r)
        if (r < rounds && base + r * 32 < N) {
          key[r] = s.key[base + r * 32];
          id[r] = s.id[base + r * 32];
        }
  }
  for (int i = t; i < N; i += kSmallThreads) a.grp.id[0][i] = s.id[i];
  // Features with codes, in order: thread t looks at `rounds` neighbouring codes.
  const int b = min(t * rounds, N), e = min(b + rounds, N);
  int heads = 0, valid = 0;
  for (int i = b; i < e; ++i) {
    const uint32_t f = s.key[i];
    if (f >= (uint32_t)a.F) break;
    ++valid;
    heads += i == 0 || f != s.key[i - 1];
  }
  int nseg, nvalid;
  int at = scan_1024(heads, sm, &nseg);
  scan_1024(valid, sm, &nvalid);
  for (int i = b; i < b + valid; ++i) {
    const uint32_t f = s.key[i];
    if (i == 0 || f != s.key[i - 1]) {
      a.grp.start[at] = i;
      a.grp.feature[at++] = (int)f;
    }
  }
  __syncthreads();
  if (t == 0) {
    a.grp.start[nseg] = nvalid;
    a.grp.state[0] = nseg;
    a.grp.state[1] = a.grp.state[2] = a.grp.state[3] = 0;
  }
  __syncthreads();
  for (int q = t; q < nseg; q += kSmallThreads) {
    const int begin = a.grp.start[q], n = a.grp.start[q + 1] - begin;
    if (n > kShort) add_long(a, a.grp.feature[q], begin, n);
  }
}

// ---------------------------------------------------------------------------
// Many codes: least significant digit radix sort, tiles of 1024 codes.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pass_key(const GradArgs& a, int pass, int64_t i) {
  return pass == 0 ? feature_key(a, i) : a.grp.key[pass & 1][i];
}

__global__ void __launch_bounds__(kTileThreads) radix_count_kernel(const __grid_constant__ GradArgs a, int pass, int shift,
                                                                   int bits, int tiles) {
  after_previous();
  __shared__ int hist[1 << kMaxBits];
  if ((int)blockIdx.x >= tiles) {  // first pass: the CTAs behind the tiles sum g's columns meanwhile
    column_sum<kTileWarps>(a, blockIdx.x - tiles);
    return;
  }
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < bins; i += kTileThreads) hist[i] = 0;
  if (pass == 0 && blockIdx.x == 0) {
    if (threadIdx.x < 4) a.grp.state[threadIdx.x] = 0;
    for (int64_t i = threadIdx.x; i < a.d; i += kTileThreads) a.grp.zeros[i] = 0.f;
  }
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTile;
  for (int i = threadIdx.x; i < kTile && base + i < a.N; i += kTileThreads)
    atomicAdd(&hist[(pass_key(a, pass, base + i) >> shift) & (bins - 1)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += kTileThreads) a.grp.count[(int64_t)i * tiles + blockIdx.x] = hist[i];
}

// Warp per bin: exclusive sums of its counts over the tiles, and the total.
__global__ void __launch_bounds__(256) radix_prefix_kernel(const __grid_constant__ GradArgs a, int bins, int tiles) {
  after_previous();
  const int bin = (int)((blockIdx.x * 256 + threadIdx.x) >> 5), lane = threadIdx.x & 31;
  if (bin >= bins) return;
  int* const c = a.grp.count + (int64_t)bin * tiles;
  int run = 0;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    const int v = t0 + lane < tiles ? c[t0 + lane] : 0;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(kFull, x, o);
      if (lane >= o) x += y;
    }
    if (t0 + lane < tiles) c[t0 + lane] = run + x - v;
    run += __shfl_sync(kFull, x, 31);
  }
  if (lane == 0) a.grp.total[bin] = run;
}

__global__ void __launch_bounds__(kTileThreads) radix_scatter_kernel(const __grid_constant__ GradArgs a, int pass, int shift,
                                                                     int bits) {
  after_previous();
  extern __shared__ int whist[];  // [warps][bins]
  __shared__ int wsum[kTileWarps];
  const int bins = 1 << bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < bins * kTileWarps; i += kTileThreads) whist[i] = 0;
  __syncthreads();
  constexpr int kRounds = kTile / kTileThreads;
  const int64_t base = (int64_t)blockIdx.x * kTile + warp * (kTile / kTileWarps);
  uint32_t key[kRounds];
  int rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * 32 + lane;
    const bool in = i < a.N;
    key[r] = in ? pass_key(a, pass, i) : 0u;
    const uint32_t digit = in ? (key[r] >> shift) & (bins - 1) : 0xffffffffu;
    const uint32_t same = __match_any_sync(kFull, digit);
    int* const h = &whist[warp * bins + (in ? digit : 0)];
    const int before = *h;
    __syncwarp();
    if (in && (same & ((1u << lane) - 1)) == 0) *h = before + __popc(same);
    __syncwarp();
    rank[r] = before + __popc(same & ((1u << lane) - 1));
  }
  __syncthreads();
  // each bin's first place: bins before it, tiles before this one, warps before
  const int per = (bins + kTileThreads - 1) / kTileThreads, b0 = min((int)threadIdx.x * per, bins), b1 = min(b0 + per, bins);
  int sum = 0;
  for (int b = b0; b < b1; ++b) sum += a.grp.total[b];
  int x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) wsum[warp] = x;
  __syncthreads();
  int run = x - sum;
  for (int w = 0; w < warp; ++w) run += wsum[w];
  for (int b = b0; b < b1; ++b) {
    int at = run + a.grp.count[(int64_t)b * gridDim.x + blockIdx.x];
    run += a.grp.total[b];
#pragma unroll
    for (int w = 0; w < kTileWarps; ++w) {
      const int c = whist[w * bins + b];
      whist[w * bins + b] = at;
      at += c;
    }
  }
  __syncthreads();
  uint32_t* const ko = a.grp.key[(pass + 1) & 1];
  uint32_t* const io = a.grp.id[(pass + 1) & 1];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * 32 + lane;
    if (i >= a.N) continue;
    const int at = whist[warp * bins + ((key[r] >> shift) & (bins - 1))] + rank[r];
    ko[at] = key[r];
    io[at] = pass == 0 ? (uint32_t)i : a.grp.id[pass & 1][i];
  }
}

// First code of each feature (binary search in the sorted keys), and the parts
// of features with more than kShort codes.
__global__ void __launch_bounds__(256) bounds_kernel(const __grid_constant__ GradArgs a) {
  after_previous();
  const int64_t f = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (f > a.F) return;
  const uint32_t* const key = a.grp.key[a.final_buf];
  // both searches step by step together: each step is a trip to the L2
  int at[2] = {0, 0};
  for (int step = 1 << a.log_codes; step > 0; step >>= 1)
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (at[q] + step <= (int)a.N && key[at[q] + step - 1] < (uint32_t)(f + q)) at[q] += step;
  a.grp.start[f] = at[0];
  const int n = at[1] - at[0];
  if (f < a.F && n > kShort) add_long(a, (int)f, at[0], n);
}

// ---------------------------------------------------------------------------
// Eight of a slab's 256 columns per lane: neighbours where rows are aligned to
// eight (VEC), else every 32nd.  As four pairs, for fma.rn.f32x2.
// ---------------------------------------------------------------------------
struct F8 {
  uint64_t v[4];
};

// STREAM: read once, which is to leave the L2 to the rows that are gathered.
template <typename T, bool VEC, bool STREAM = false>
__device__ __forceinline__ F8 load_cols(const T* row, int64_t base, int lane, int64_t d) {
  float w[8];
  if constexpr (VEC) {
    const int64_t c = base + lane * 8;
    if (c < d) {
      if constexpr (STREAM) ldcs8(row + c, w);
      else ldg8(row + c, w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t c = base + lane + 32 * i;
      w[i] = c < d ? as_f32(__ldg(row + c)) : 0.f;
    }
  }
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = pair(w[2 * i], w[2 * i + 1]);
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_cols(T* row, int64_t base, int lane, int64_t d, const F8& f) {
  float w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 h = halves(f.v[i]);
    w[2 * i] = h.x;
    w[2 * i + 1] = h.y;
  }
  if constexpr (VEC) {
    const int64_t c = base + lane * 8;
    if (c < d) stcs8(row + c, w);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t c = base + lane + 32 * i;
      if (c < d) row[c] = from_f32<T>(w[i]);
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// N sums over the warp at once; lane l returns the sum of x[l >> 2] (N padded
// to 8 with zeros): halves of the lanes take over halves of the sums.
template <int N>
__device__ __forceinline__ float sum_each(const float (&x)[N], int lane) {
  const auto at = [&](int i) { return i < N ? x[i] : 0.f; };
  float a[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float mine = lane & 16 ? at(i + 4) : at(i), other = lane & 16 ? at(i) : at(i + 4);
    a[i] = mine + __shfl_xor_sync(kFull, other, 16);
  }
  float b[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float mine = lane & 8 ? a[i + 2] : a[i], other = lane & 8 ? a[i] : a[i + 2];
    b[i] = mine + __shfl_xor_sync(kFull, other, 8);
  }
  const float mine = lane & 4 ? b[1] : b[0], other = lane & 4 ? b[0] : b[1];
  float c = mine + __shfl_xor_sync(kFull, other, 4);
  c += __shfl_xor_sync(kFull, c, 2);
  c += __shfl_xor_sync(kFull, c, 1);
  return c;
}

// A list of n <= N codes, lane i < n holding code e, its row and its value:
// rows' addresses, dot products and sums stay in registers over the slabs.
// Lists are rounded up to 1, 2, 4 or 8 codes with a row of zeros: a variant for
// each length took twice the time, waiting for instructions (warps of one SM
// are at different lengths, and the loops of eight variants do not fit the
// instruction cache together).
template <typename T, bool DEC, bool ENC, bool VEC, int N>
__device__ __forceinline__ void short_list(const GradArgs& a, int64_t f, int n, uint32_t e, int row, float value,
                                           float given, int lane) {
  const int64_t mine = lane < n ? (int64_t)row * a.d : -1;
  float dv = given;  // lane i < n: the gradient of code i
  if constexpr (DEC) {
    uint64_t dot[N], v[N];
    const float* g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t off = __shfl_sync(kFull, mine, i);
      const float x = __shfl_sync(kFull, lane < n ? value : 0.f, i);
      g[i] = off >= 0 ? a.g + off : a.grp.zeros;
      v[i] = pair(x, x);
      dot[i] = 0;
    }
    const T* const w_row = static_cast<const T*>(a.W_dec) + f * a.d;
    T* const out = static_cast<T*>(a.dW_dec) + f * a.d;
    // As many slabs at once as the registers hold: all their loads go out before the first sum (375 to 343 us with the
    // same for X below; unrolled loops left each slab's loads behind the stores of the one before).
    constexpr int SG = VEC ? (N >= 8 ? 1 : N >= 2 ? 2 : 4) : 1;
#pragma unroll 1
    for (int64_t base = 0; base < a.d; base += 256 * SG) {
      if (VEC && base + lane * 8 >= a.d) continue;
      F8 w[SG], x[SG][N];
#pragma unroll
      for (int s = 0; s < SG; ++s) {
        w[s] = load_cols<T, VEC, true>(w_row, base + 256 * s, lane, a.d);
#pragma unroll
        for (int i = 0; i < N; ++i) x[s][i] = load_cols<float, VEC>(g[i], base + 256 * s, lane, a.d);
      }
#pragma unroll
      for (int s = 0; s < SG; ++s) {
        F8 acc = {{0, 0, 0, 0}};
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            acc.v[c] = fma2(v[i], x[s][i].v[c], acc.v[c]);
            dot[i] = fma2(w[s].v[c], x[s][i].v[c], dot[i]);
          }
        store_cols<T, VEC>(out, base + 256 * s, lane, a.d, acc);
      }
    }
    float sums[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 h = halves(dot[i]);
      sums[i] = h.x + h.y;
    }
    const float s = sum_each<N>(sums, lane);
    dv += __shfl_sync(kFull, s, (lane & 7) * 4);
    if (a.dv != nullptr && lane < n) a.dv[e] = dv;
  }
  if constexpr (ENC) {
    if (lane >= n) dv = 0.f;
    uint64_t x2[N];
    const T* X[N];
    float b = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t off = __shfl_sync(kFull, mine, i);
      const float x = __shfl_sync(kFull, dv, i);
      X[i] = off >= 0 ? static_cast<const T*>(a.X) + off : reinterpret_cast<const T*>(a.grp.zeros);
      x2[i] = pair(x, x);
      b += x;
    }
    if (lane == 0) a.db_enc[f] = b;
    T* const out = static_cast<T*>(a.dW_enc) + f * a.d;
    // As many slabs at once as make eight rows' pieces: their loads go out together.
    constexpr int SL = VEC && sizeof(T) == 2 ? (N >= 8 ? 1 : N >= 4 ? 2 : 4) : 1;
#pragma unroll 1
    for (int64_t base = 0; base < a.d; base += 256 * SL) {
      if (VEC && base + lane * 8 >= a.d) continue;
      F8 acc[SL];
      if constexpr (VEC && sizeof(T) == 2) {
        uint4 raw[SL][N];
#pragma unroll
        for (int s = 0; s < SL; ++s) {
          const int64_t c = base + 256 * s + lane * 8;
#pragma unroll
          for (int i = 0; i < N; ++i) raw[s][i] = __ldg(reinterpret_cast<const uint4*>(X[i] + (c < a.d ? c : 0)));
        }
#pragma unroll
        for (int s = 0; s < SL; ++s) {
          acc[s] = F8{{0, 0, 0, 0}};
#pragma unroll
          for (int i = 0; i < N; ++i) {
            float w[8];
            unpack8<T>(raw[s][i], w);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[s].v[c] = fma2(x2[i], pair(w[2 * c], w[2 * c + 1]), acc[s].v[c]);
          }
        }
      } else {
        acc[0] = F8{{0, 0, 0, 0}};
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const F8 x = load_cols<T, VEC>(X[i], base, lane, a.d);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[0].v[c] = fma2(x2[i], x.v[c], acc[0].v[c]);
        }
      }
#pragma unroll
      for (int s = 0; s < SL; ++s) store_cols<T, VEC>(out, base + 256 * s, lane, a.d, acc[s]);
    }
  }
}

// A warp's list of more codes, filled up to a multiple of 8 with rows of zeros:
// its rows, values and gradients.
struct List {
  int row[kMaxPart];
  float v[kMaxPart];
  float dv[kMaxPart];
};

// (Inlined: as a function of its own it took 1.9 times the time, 349 to 185 us for
// lists of 512.)  A list of any length up to kMaxPart, slab by slab and eight codes at a time;
// `slot` >= 0: a part of a longer list, whose sums go to the workspace.
template <typename T, bool DEC, bool ENC, bool VEC>
__device__ __forceinline__ void long_list(const GradArgs& a, List& s, int64_t f, int begin, int n, int64_t slot, int lane) {
  const uint32_t* const id = a.grp.id[a.final_buf];
  for (int i = lane; i < ((n + 7) & ~7); i += 32) {
    const uint32_t e = i < n ? id[begin + i] : 0u;
    s.row[i] = i < n ? (int)(e / (uint32_t)a.k) : -1;
    s.v[i] = DEC && i < n ? a.V[e] : 0.f;
    s.dv[i] = a.gv != nullptr && i < n ? a.gv[e] : 0.f;
  }
  __syncwarp();
  if constexpr (DEC) {
    const T* const w_row = static_cast<const T*>(a.W_dec) + f * a.d;
#pragma unroll 1
    for (int64_t base = 0; base < a.d; base += 256) {
      const F8 w = load_cols<T, VEC, true>(w_row, base, lane, a.d);
      F8 acc = {{0, 0, 0, 0}};
#pragma unroll 1
      for (int i = 0; i < n; i += 8) {
        float sums[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int row = s.row[i + q];
          const F8 g = load_cols<float, VEC>(row >= 0 ? a.g + (int64_t)row * a.d : a.grp.zeros, base, lane, a.d);
          const uint64_t v = pair(s.v[i + q], s.v[i + q]);
          uint64_t dot = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            acc.v[c] = fma2(v, g.v[c], acc.v[c]);
            dot = fma2(w.v[c], g.v[c], dot);
          }
          const float2 h = halves(dot);
          sums[q] = h.x + h.y;
        }
        const float sum = sum_each<8>(sums, lane);
        if ((lane & 3) == 0) s.dv[i + (lane >> 2)] += sum;
      }
      if (slot >= 0)
        store_cols<float, VEC>(a.grp.part_dec + slot * a.d, base, lane, a.d, acc);
      else
        store_cols<T, VEC>(static_cast<T*>(a.dW_dec) + f * a.d, base, lane, a.d, acc);
    }
    __syncwarp();
    if (a.dv != nullptr)
      for (int i = lane; i < n; i += 32) a.dv[id[begin + i]] = s.dv[i];
  }
  if constexpr (ENC) {
    float b = 0.f;
    for (int i = lane; i < n; i += 32) b += s.dv[i];
    b = warp_sum(b);
    if (lane == 0) {
      if (slot >= 0) a.grp.part_b[slot] = b;
      else a.db_enc[f] = b;
    }
#pragma unroll 1
    for (int64_t base = 0; base < a.d; base += 256) {
      F8 acc = {{0, 0, 0, 0}};
#pragma unroll 1
      for (int i = 0; i < n; i += 8) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int row = s.row[i + q];
          const F8 x = load_cols<T, VEC>(row >= 0 ? static_cast<const T*>(a.X) + (int64_t)row * a.d
                                                  : reinterpret_cast<const T*>(a.grp.zeros), base, lane, a.d);
          const float dv = row >= 0 ? s.dv[i + q] : 0.f;  // (what a NaN in w made of a row of zeros stays out)
          const uint64_t v = pair(dv, dv);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc.v[c] = fma2(v, x.v[c], acc.v[c]);
        }
      }
      if (slot >= 0)
        store_cols<float, VEC>(a.grp.part_enc + slot * a.d, base, lane, a.d, acc);
      else
        store_cols<T, VEC>(static_cast<T*>(a.dW_enc) + f * a.d, base, lane, a.d, acc);
    }
  }
  __syncwarp();
}

// Adds a slab of a long list's parts, in order.
template <typename T, bool VEC>
__device__ __noinline__ void join_slab(const GradArgs& a, const float* from, T* to, int first, int parts, int64_t base,
                                       int lane) {
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int p = 0; p < parts; ++p) {
    // from L2: other SMs wrote these rows, maybe during this kernel
    const float* const row = from + (int64_t)(first + p) * a.d;
    if constexpr (VEC) {
      const int64_t c = base + lane * 8;
      if (c < a.d) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(row + c)), y = __ldcg(reinterpret_cast<const float4*>(row + c) + 1);
        acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
        acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
      }
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int64_t col = base + lane + 32 * c;
        acc[c] += col < a.d ? __ldcg(row + col) : 0.f;
      }
    }
  }
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = pair(acc[2 * i], acc[2 * i + 1]);
  store_cols<T, VEC>(to, base, lane, a.d, r);
}

template <typename T, bool DEC, bool ENC, bool VEC>
__device__ __forceinline__ void join_at(const GradArgs& a, const Part& p, int64_t base, int lane) {
  if constexpr (DEC)
    join_slab<T, VEC>(a, a.grp.part_dec, static_cast<T*>(a.dW_dec) + (int64_t)p.feature * a.d, p.first, p.parts, base, lane);
  if constexpr (ENC) {
    join_slab<T, VEC>(a, a.grp.part_enc, static_cast<T*>(a.dW_enc) + (int64_t)p.feature * a.d, p.first, p.parts, base, lane);
    if (lane == 0 && base == 0) {
      float b = 0.f;
      for (int q = 0; q < p.parts; ++q) b += __ldcg(&a.grp.part_b[p.first + q]);
      a.db_enc[p.feature] = b;
    }
  }
}

// Many codes: a warp per long list and slab, after the parts.  (One warp for a
// list of 28 parts, the last to arrive, took 30 us at the end of the kernel.)
template <typename T, bool DEC, bool ENC, bool VEC>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ GradArgs a) {
  after_previous();
  const int lane = threadIdx.x & 31;
  if (a.grp.state[2] == 0) return;
  const int64_t slabs = (a.d + 255) / 256, tasks = a.grp.state[1] * slabs;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); t < tasks; t += (int64_t)gridDim.x * 4) {
    const Part p = a.grp.part[t / slabs];
    if (p.parts > 1 && p.part == 0) join_at<T, DEC, ENC, VEC>(a, p, t % slabs * 256, lane);
  }
}

template <typename T, bool DEC, bool ENC, bool VEC>
__global__ void __launch_bounds__(32 * kGradWarps, kGradCtas) sae_grad_kernel(const __grid_constant__ GradArgs a) {
  after_previous();
  __shared__ List lists[kGradWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  List& s = lists[warp];
  const int64_t me = (int64_t)blockIdx.x * kGradWarps + warp, all = (int64_t)gridDim.x * kGradWarps;
  // Long lists first: they take longest, and their joins hide behind the rest.
  const int parts = a.grp.state[1];
  for (int64_t t = me; t < parts; t += all) {
    const Part p = a.grp.part[t];
    long_list<T, DEC, ENC, VEC>(a, s, p.feature, p.begin, p.n, p.parts > 1 ? p.first + p.part : -1, lane);
    if (p.parts == 1 || !a.small) continue;
    // Few codes: the warp that is last to finish a part of the list joins them (a kernel more would cost 2 us).
    __threadfence();
    __syncwarp();
    int done = 0;
    if (lane == 0) done = atomicAdd(&a.grp.arrived[p.first], 1) == p.parts - 1;
    if (!__shfl_sync(kFull, done, 0)) continue;
    __threadfence();
    for (int64_t base = 0; base < a.d; base += 256) join_at<T, DEC, ENC, VEC>(a, p, base, lane);
  }
  const int64_t tasks = a.small ? a.grp.state[0] : a.F;
  const uint32_t* const id = a.grp.id[a.final_buf];
  // The short lists, one after the other to whichever warp is free.  What a list needs is asked for three steps
  // ahead of its sums, since each waits for the one before: its number, its bounds, its codes, their values.
  // (The first two of each warp are its own: with few lists nobody waits for the counter.)
  const auto take = [&]() {
    int q = 0;
    if (lane == 0) q = atomicAdd(&a.grp.state[3], 1);
    return 2 * all + (int64_t)__shfl_sync(kFull, q, 0);
  };
  const auto bounds = [&](int64_t q, int& b, int& m, int64_t& feature) {
    b = m = 0;
    feature = q;
    if (q < tasks) {
      b = a.grp.start[q];
      m = a.grp.start[q + 1] - b;
      if (a.small) feature = a.grp.feature[q];
    }
  };
  int64_t t = all - 1 - me, next_t = t + all, f, next_f;  // (warps with a part more come last)
  int begin, n, next_begin, next_n;
  bounds(t, begin, n, f);
  bounds(next_t, next_begin, next_n, next_f);
  uint32_t e = lane < n ? id[begin + lane] : 0u;
  float v = DEC && lane < n ? a.V[e] : 0.f, given = a.gv != nullptr && lane < n ? a.gv[e] : 0.f;
  while (t < tasks) {
    const uint32_t next_e = lane < next_n ? id[next_begin + lane] : 0u;
    const int64_t after_t = next_t < tasks ? take() : tasks;
    int64_t after_f;
    int after_begin, after_n;
    bounds(after_t, after_begin, after_n, after_f);
    const int row = (int)(e / (uint32_t)a.k);
    if (n == 0) {
      if (!a.small) {
        const F8 zero = {{0, 0, 0, 0}};
        for (int64_t base = 0; base < a.d; base += 256) {
          if constexpr (DEC) store_cols<T, VEC>(static_cast<T*>(a.dW_dec) + f * a.d, base, lane, a.d, zero);
          if constexpr (ENC) store_cols<T, VEC>(static_cast<T*>(a.dW_enc) + f * a.d, base, lane, a.d, zero);
        }
        if (ENC && lane == 0) a.db_enc[f] = 0.f;
      }
    } else if (n == 1) {
      short_list<T, DEC, ENC, VEC, 1>(a, f, n, e, row, v, given, lane);
    } else if (n == 2) {
      short_list<T, DEC, ENC, VEC, 2>(a, f, n, e, row, v, given, lane);
    } else if (n <= 4) {
      short_list<T, DEC, ENC, VEC, 4>(a, f, n, e, row, v, given, lane);
    } else if (n <= kShort) {
      short_list<T, DEC, ENC, VEC, kShort>(a, f, n, e, row, v, given, lane);
    }
    t = next_t, f = next_f, begin = next_begin, n = next_n, e = next_e;
    next_t = after_t, next_f = after_f, next_begin = after_begin, next_n = after_n;
    v = DEC && lane < n ? a.V[e] : 0.f;
    given = a.gv != nullptr && lane < n ? a.gv[e] : 0.f;
  }
}

// dX_b = sum_j dv_bj W_enc[i_bj]: a warp per row and slab of 256 columns.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128) dx_kernel(const __grid_constant__ GradArgs a) {
  after_previous();
  const int lane = threadIdx.x & 31;
  const int64_t slabs = (a.d + 255) / 256;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); t < a.B * slabs; t += (int64_t)gridDim.x * 4) {
    const int64_t b = t / slabs, base = (t % slabs) * 256;
    F8 acc = {{0, 0, 0, 0}};
    for (int j0 = 0; j0 < a.k; j0 += 32) {
      const int left = min(32, a.k - j0);
      int fi = lane < left ? a.I[b * a.k + j0 + lane] : -1;
      if ((uint32_t)fi >= (uint32_t)a.F) fi = -1;
      const float di = fi >= 0 ? a.dv[b * a.k + j0 + lane] : 0.f;
      // codes that are passed over are dropped, so that four rows can be on their way at once
      const uint32_t live = __ballot_sync(kFull, fi >= 0);
      const int codes = __popc(live);
      const int from = lane < codes ? __fns(live, 0, lane + 1) : 0;
      const int ff = __shfl_sync(kFull, fi, from);
      const float dd = __shfl_sync(kFull, di, from);
      int j = 0;
      for (; j + 4 <= codes; j += 4) {
        F8 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          w[q] = load_cols<T, VEC>(static_cast<const T*>(a.W_enc) + (int64_t)__shfl_sync(kFull, ff, j + q) * a.d, base, lane, a.d);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float x = __shfl_sync(kFull, dd, j + q);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc.v[c] = fma2(pair(x, x), w[q].v[c], acc.v[c]);
        }
      }
      for (; j < codes; ++j) {
        const F8 w = load_cols<T, VEC>(static_cast<const T*>(a.W_enc) + (int64_t)__shfl_sync(kFull, ff, j) * a.d, base, lane, a.d);
        const float x = __shfl_sync(kFull, dd, j);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc.v[c] = fma2(pair(x, x), w.v[c], acc.v[c]);
      }
    }
    store_cols<T, VEC>(static_cast<T*>(a.dX) + b * a.d, base, lane, a.d, acc);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
size_t round_up(size_t n) { return (n + 255) & ~(size_t)255; }

struct Plan {
  bool small;
  int key_bits, passes, bits[3], tiles, part, slots, chunks;
  size_t bytes;
};

// Where each array of the workspace lies; with `base` null only the size.
Plan lay_out(int64_t B, int64_t k, int64_t F, int64_t d, char* base, Group* g) {
  Plan p = {};
  const int64_t N = B * k;
  p.small = N <= kSmallCodes;
  int bits = 1;
  while (bits < 31 && ((int64_t)1 << bits) <= F) ++bits;  // the keys 0 .. F
  p.key_bits = bits;
  p.passes = (bits + kMaxBits - 1) / kMaxBits;
  for (int i = 0; i < p.passes; ++i) p.bits[i] = bits / p.passes + (i < bits % p.passes ? 1 : 0);
  p.tiles = (int)((N + kTile - 1) / kTile);
  // Short parts spread a few frequent features over many warps, at the cost of sums that are written and read again.
  // Parts of 32 and of 64 codes, whole gradients in bf16 (a tenth of the codes on 50 features where it says so):
  //   16384 codes, d=768 F=16384, frequent 61, 63 us      33033, d=1032 F=20000, frequent 90, 106
  //   64000, d=1024 F=16384, frequent 88, 106             64000, d=512 F=1024 73, 75
  //   131072, d=1024 F=16384, frequent 130, 132           262144, d=2048 F=65536, frequent 409, 391
  //   262144, d=768 F=4096 187, 174                       524288, d=512 F=1024 326, 271
  // So 64 from 65536 codes on, where there are parts enough for all warps, and longer ones where their sums would take
  // more than kPartBytes of workspace (which parts of kMaxPart may exceed).
  p.part = N < 65536 ? kMinPart : 2 * kMinPart;
  while (p.part < kMaxPart && 2 * (N / p.part) * d > kPartBytes / 8) p.part *= 2;
  p.slots = (int)(2 * (N / p.part));  // lists longer than a part: at most N / part of them, and N / part full parts
  p.chunks = p.small ? 1 : (int)std::min<int64_t>(32, (B + 127) / 128);
  Group none;
  Group& r = g ? *g : none;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* q = base ? base + at : nullptr;
    at += round_up(bytes);
    return static_cast<void*>(q);
  };
  for (int i = 0; i < 2; ++i) {
    r.id[i] = static_cast<uint32_t*>(take(4 * N));
    r.key[i] = static_cast<uint32_t*>(take(p.small ? 0 : 4 * N));
  }
  const size_t bins = (size_t)1 << kMaxBits;
  r.count = static_cast<int*>(take(p.small ? 0 : 4 * bins * p.tiles));
  r.total = static_cast<int*>(take(p.small ? 0 : 4 * bins));
  r.start = static_cast<int*>(take(4 * (size_t)((p.small ? std::min(N, F) : F) + 1)));
  r.feature = static_cast<int*>(take(p.small ? 4 * (size_t)N : 0));
  r.state = static_cast<int*>(take(16));
  r.arrived = static_cast<int*>(take(4 * (size_t)p.slots));
  // lists with more than kShort codes, and one more for each full part
  r.part = static_cast<Part*>(take(sizeof(Part) * (size_t)(N / (kShort + 1) + N / p.part)));
  r.part_dec = static_cast<float*>(take(4 * (size_t)p.slots * d));
  r.part_enc = static_cast<float*>(take(4 * (size_t)p.slots * d));
  r.part_b = static_cast<float*>(take(4 * (size_t)p.slots));
  r.colsum = static_cast<float*>(take(p.chunks > 1 ? 4 * (size_t)p.chunks * d : 0));
  r.col_arrived = static_cast<int*>(take(4 * (size_t)((d + 127) / 128)));
  r.zeros = static_cast<float*>(take(4 * (size_t)d));
  p.bytes = at;
  return p;
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t s, bool after, A... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = after ? 1 : 0;  // the call's first kernel waits for whatever comes before it
  return cudaLaunchKernelEx(&c, kernel, args...);
}

template <typename T, bool DEC, bool ENC, bool VEC>
cudaError_t launch_modes(const GradArgs& a, int sms, cudaStream_t s) {
  const int64_t tasks = a.small ? std::min(a.N, a.F) : a.F;
  const unsigned grid =
      (unsigned)std::max<int64_t>(1, std::min<int64_t>((tasks + kGradWarps - 1) / kGradWarps, sms * kGradCtas));
  cudaError_t e = launch(sae_grad_kernel<T, DEC, ENC, VEC>, grid, 32 * kGradWarps, 0, s, true, a);
  if (e == cudaSuccess && !a.small && a.N > a.part)
    e = launch(join_kernel<T, DEC, ENC, VEC>, (unsigned)sms * 4, 128, 0, s, true, a);
  if (e == cudaSuccess && a.dX != nullptr) {
    const int64_t warps = a.B * ((a.d + 255) / 256);
    e = launch(dx_kernel<T, VEC>, (unsigned)std::min<int64_t>((warps + 3) / 4, sms * 16), 128, 0, s, true, a);
  }
  return e;
}

template <typename T, bool VEC>
cudaError_t launch_main(const GradArgs& a, bool dec, bool enc, int sms, cudaStream_t s) {
  if (dec && enc) return launch_modes<T, true, true, VEC>(a, sms, s);
  return dec ? launch_modes<T, true, false, VEC>(a, sms, s) : launch_modes<T, false, true, VEC>(a, sms, s);
}

template <typename T>
cudaError_t launch_type(const GradArgs& a, bool vec, bool dec, bool enc, int sms, cudaStream_t s) {
  return vec ? launch_main<T, true>(a, dec, enc, sms, s) : launch_main<T, false>(a, dec, enc, sms, s);
}

bool sizes_ok(int64_t B, int64_t k, int64_t F, int64_t d) {
  return B >= 0 && k >= 1 && F >= 1 && d >= 1 && F < 0x7fffffff && d <= (1 << 24) && k <= (1 << 20) &&
         B <= 0x3fffffff / k;
}

}  // namespace
}  // namespace stk

extern "C" int stk_sae_backward_workspace_bytes(int64_t B, int64_t k, int64_t F, int64_t d, size_t* bytes) {
  STK_ENTRY_BEGIN
  using namespace stk;
  if (!bytes) return host_fail(STK_EINVAL, "bytes is NULL");
  if (!sizes_ok(B, k, F, d))
    return host_fail(STK_EINVAL, "stk_sae_backward: need B >= 0, k, F, d >= 1, B * k < 2^30, F < 2^31 - 1, d <= 2^24");
  *bytes = lay_out(B, k, F, d, nullptr, nullptr).bytes;
  return STK_OK;
  STK_ENTRY_END
}

extern "C" int stk_sae_backward(const float* grad_out, const void* X, const void* W_enc, const void* W_dec, const float* V,
                                const int32_t* I, const float* grad_vals, void* dW_enc, float* db_enc, void* dW_dec,
                                float* db_dec, float* dvals, void* dX, int64_t B, int64_t k, int64_t F, int64_t d,
                                int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  STK_ENTRY_BEGIN
  using namespace stk;
  if (dtype != STK_F32 && dtype != STK_F16 && dtype != STK_BF16)
    return host_fail(STK_EINVAL, "stk_sae_backward: X, W_enc and W_dec must be fp32, fp16, or bf16");
  if (!sizes_ok(B, k, F, d))
    return host_fail(STK_EINVAL, "stk_sae_backward: need B >= 0, k, F, d >= 1, B * k < 2^30, F < 2^31 - 1, d <= 2^24");
  const bool dec = dW_dec != nullptr, enc = dW_enc != nullptr;
  if (!dec && !enc) return host_fail(STK_EINVAL, "stk_sae_backward: one of dW_enc and dW_dec is needed");
  if (enc != (db_enc != nullptr)) return host_fail(STK_EINVAL, "stk_sae_backward: dW_enc and db_enc go together");
  if (!dec && (db_dec || dvals)) return host_fail(STK_EINVAL, "stk_sae_backward: db_dec and dvals need dW_dec");
  if (dX && !enc) return host_fail(STK_EINVAL, "stk_sae_backward: dX needs dW_enc");
  if (B > 0 && (!I || (dec && (!grad_out || !W_dec || !V)) || (enc && !X) || (!dec && !grad_vals) ||
                (dX && (!W_enc || (dec && !dvals)))))
    return host_fail(STK_EINVAL, "stk_sae_backward: null pointer");
  const size_t es = dtype == STK_F32 ? 4 : 2;
  for (const void* p : {X, W_enc, W_dec, (const void*)dW_enc, (const void*)dW_dec, (const void*)dX})
    if (!aligned_to(p, es)) return host_fail(STK_EINVAL, "stk_sae_backward: pointer not aligned to its element");
  for (const void* p : {(const void*)grad_out, (const void*)V, (const void*)I, (const void*)grad_vals, (const void*)db_enc,
                        (const void*)db_dec, (const void*)dvals})
    if (!aligned_to(p, 4)) return host_fail(STK_EINVAL, "stk_sae_backward: pointer not aligned to its element");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t dict = (size_t)F * (size_t)d * es;
  if (B == 0) {
    cudaError_t e = cudaSuccess;
    if (enc) e = cudaMemsetAsync(dW_enc, 0, dict, s);
    if (e == cudaSuccess && enc) e = cudaMemsetAsync(db_enc, 0, 4 * (size_t)F, s);
    if (e == cudaSuccess && dec) e = cudaMemsetAsync(dW_dec, 0, dict, s);
    if (e == cudaSuccess && db_dec) e = cudaMemsetAsync(db_dec, 0, 4 * (size_t)d, s);
    return e == cudaSuccess ? STK_OK : host_cuda_fail(e, "cudaMemsetAsync");
  }
  GradArgs a = {};
  const Plan p = lay_out(B, k, F, d, static_cast<char*>(workspace), &a.grp);
  if (!workspace || workspace_bytes < p.bytes)
    return host_fail(STK_ENOSPACE, "stk_sae_backward: workspace too small (stk_sae_backward_workspace_bytes)");
  if (!aligned_to(workspace, 32)) return host_fail(STK_EINVAL, "stk_sae_backward: workspace must be 32-byte aligned");
  a.g = grad_out;
  a.X = X;
  a.W_dec = W_dec;
  a.W_enc = W_enc;
  a.V = V;
  a.I = I;
  a.gv = grad_vals;
  a.dW_enc = dW_enc;
  a.db_enc = db_enc;
  a.dW_dec = dW_dec;
  a.db_dec = db_dec;
  a.dv = dvals;
  a.dX = dX;
  a.B = B;
  a.F = F;
  a.d = d;
  a.N = B * k;
  a.k = (int)k;
  a.small = p.small;
  a.final_buf = p.small ? 0 : p.passes & 1;
  a.chunks = p.chunks;
  a.part = p.part;
  while (((int64_t)2 << a.log_codes) <= a.N) ++a.log_codes;
  int sms = 0;
  if (const int rc = host_device_sms(&sms)) return rc;
  cudaError_t e;
  if (p.small) {
    e = cudaFuncSetAttribute(small_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(SmallSort));
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute");
    const unsigned grid = (unsigned)std::max<int64_t>(2 * sms, 1 + (int64_t)(dict / kZeroBytes));
    e = launch(small_group_kernel, grid, kSmallThreads, sizeof(SmallSort), s, false, a, p.key_bits, (int64_t)dict);
  } else {
    e = cudaFuncSetAttribute(radix_scatter_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             4 * kTileWarps << kMaxBits);
    if (e == cudaSuccess && p.chunks > 1)
      e = cudaMemsetAsync(a.grp.col_arrived, 0, 4 * (size_t)((d + 127) / 128), s);
    if (e != cudaSuccess) return host_cuda_fail(e, "stk_sae_backward");
    for (int pass = 0, shift = 0; pass < p.passes; shift += p.bits[pass++]) {
      const int bins = 1 << p.bits[pass], sums = pass == 0 && db_dec ? (int)((d + 127) / 128 * p.chunks) : 0;
      e = launch(radix_count_kernel, p.tiles + sums, kTileThreads, 0, s, pass > 0, a, pass, shift, p.bits[pass], p.tiles);
      if (e == cudaSuccess) e = launch(radix_prefix_kernel, (bins + 7) / 8, 256, 0, s, true, a, bins, p.tiles);
      if (e == cudaSuccess)
        e = launch(radix_scatter_kernel, p.tiles, kTileThreads, 4 * (size_t)kTileWarps * bins, s, true, a, pass, shift,
                   p.bits[pass]);
      if (e != cudaSuccess) return host_cuda_fail(e, "stk_sae_backward: radix pass launch");
    }
    e = launch(bounds_kernel, (unsigned)(F / 256 + 1), 256, 0, s, true, a);
  }
  if (e != cudaSuccess) return host_cuda_fail(e, "stk_sae_backward: grouping launch");
  if (dX && !dec) a.dv = const_cast<float*>(grad_vals);  // read by dx_kernel alone
  bool vec = d % 8 == 0 && vec_aligned<float>(grad_out);
  for (const void* q : {X, W_enc, W_dec, (const void*)dW_enc, (const void*)dW_dec, (const void*)dX}) vec &= aligned_to(q, 8 * es);
  e = dtype == STK_F32   ? launch_type<float>(a, vec, dec, enc, sms, s)
      : dtype == STK_F16 ? launch_type<__half>(a, vec, dec, enc, sms, s)
                         : launch_type<__nv_bfloat16>(a, vec, dec, enc, sms, s);
  if (e != cudaSuccess) return host_cuda_fail(e, "sae_grad_kernel launch");
  return STK_OK;
  STK_ENTRY_END
}
