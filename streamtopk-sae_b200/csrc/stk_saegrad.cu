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
constexpr int kPart = 256;        // codes of one feature that one warp sums; longer lists are split and joined
constexpr int kSmallCodes = 8192; // up to this many codes one CTA sorts, while the others zero the gradients
constexpr int kSmallThreads = 1024;
constexpr int kTile = 2048;       // codes per CTA of a radix pass
constexpr int kTileThreads = 256;
constexpr int kTileWarps = kTileThreads / 32;
constexpr int kMaxBits = 11;      // of a radix digit
constexpr int kGradWarps = 4;

struct Part {
  int feature, begin, n, slot, first, parts;
};

struct Group {
  uint32_t* key[2];
  uint32_t* id[2];
  int* count;      // [bins][tiles] of a pass
  int* total;      // [bins]
  int* start;      // [F + 1] first code of each feature, in sorted order; small: [segments + 1] and
  int* feature;    // [segments]
  int* state;      // [0] segments, [1] parts
  int* arrived;    // [slots] parts that are done, at their list's first slot
  Part* part;
  float* part_dec;
  float* part_enc;
  float* part_b;
  float* colsum;   // [chunks][d]
  int* col_arrived;
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
  int k, small, final_buf;
  int chunks;       // row chunks of the column sum of g
  Group grp;
};

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
__device__ void column_sum(const GradArgs& a, int64_t unit) {
  __shared__ float sm[8][128];
  __shared__ int last;
  const int64_t cb = unit / a.chunks, chunk = unit % a.chunks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = min((int)blockDim.x / 32, 8);
  const int64_t rows = (a.B + a.chunks - 1) / a.chunks;
  const int64_t r0 = chunk * rows, r1 = min(a.B, r0 + rows);
  __syncthreads();
  if (warp < warps) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t r = r0 + warp; r < r1; r += warps)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t c = cb * 128 + i * 32 + lane;
        if (c < a.d) acc[i] += a.g[r * a.d + c];
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) sm[warp][i * 32 + lane] = acc[i];
  }
  __syncthreads();
  const int64_t c = cb * 128 + threadIdx.x;
  const bool mine = threadIdx.x < 128 && c < a.d;
  float s = 0.f;
  if (mine) {
    for (int w = 0; w < warps; ++w) s += sm[w][threadIdx.x];
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
    for (int i = 0; i < a.chunks; ++i) s += __ldcg(&a.grp.colsum[i * a.d + c]);
    a.db_dec[c] = s;
  }
}

// ---------------------------------------------------------------------------
// Few codes: CTA 0 sorts them in shared memory and lists the features that
// have any; the other CTAs zero the gradients (most rows stay zero) and sum
// g's columns meanwhile.
// ---------------------------------------------------------------------------
__device__ void zero_fill(void* p, int64_t bytes, int64_t i, int64_t n) {
  // p is at least 4-byte aligned where it is not 16-byte aligned only for 2-byte elements: go by bytes at the edges
  uint8_t* const b = static_cast<uint8_t*>(p);
  const int64_t head = min(bytes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15));
  const int64_t body = (bytes - head) / 16;
  uint4* const v = reinterpret_cast<uint4*>(b + head);
  for (int64_t j = i; j < body; j += n) v[j] = make_uint4(0, 0, 0, 0);
  for (int64_t j = i; j < head; j += n) b[j] = 0;
  for (int64_t j = head + body * 16 + i; j < bytes; j += n) b[j] = 0;
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

__global__ void __launch_bounds__(kSmallThreads) small_group_kernel(const __grid_constant__ GradArgs a, int padded,
                                                                    int64_t dict_bytes) {
  extern __shared__ uint64_t codes[];
  __shared__ int sm[33];
  if (blockIdx.x > 0) {
    const int64_t i = (int64_t)(blockIdx.x - 1) * blockDim.x + threadIdx.x, n = (int64_t)(gridDim.x - 1) * blockDim.x;
    if (a.dW_dec != nullptr) zero_fill(a.dW_dec, dict_bytes, i, n);
    if (a.dW_enc != nullptr) zero_fill(a.dW_enc, dict_bytes, i, n);
    if (a.db_enc != nullptr) zero_fill(a.db_enc, a.F * 4, i, n);
    if (a.db_dec != nullptr)  // one chunk: no counters, which CTA 0 may not have cleared yet
      for (int64_t u = blockIdx.x - 1; u < (a.d + 127) / 128; u += gridDim.x - 1) column_sum(a, u);
    return;
  }
  const int t = threadIdx.x, N = (int)a.N;
  for (int i = t; i < padded; i += kSmallThreads)
    codes[i] = i < N ? ((uint64_t)feature_key(a, i) << 32) | (uint32_t)i : ~0ull;
  for (int size = 2; size <= padded; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int i = t; i < padded / 2; i += kSmallThreads) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const uint64_t x = codes[lo], y = codes[hi];
        if ((x > y) == ((lo & size) == 0)) {
          codes[lo] = y;
          codes[hi] = x;
        }
      }
    }
  __syncthreads();
  for (int i = t; i < N; i += kSmallThreads) a.grp.id[0][i] = (uint32_t)codes[i];
  // Features with codes, in order: thread t looks at `per` neighbouring codes.
  const int per = (N + kSmallThreads - 1) / kSmallThreads;
  const int b = min(t * per, N), e = min(b + per, N);
  int heads = 0, valid = 0;
  for (int i = b; i < e; ++i) {
    const uint32_t f = (uint32_t)(codes[i] >> 32);
    if (f >= (uint32_t)a.F) break;
    ++valid;
    heads += i == 0 || f != (uint32_t)(codes[i - 1] >> 32);
  }
  int nseg, nvalid;
  int at = scan_1024(heads, sm, &nseg);
  scan_1024(valid, sm, &nvalid);
  for (int i = b; i < b + valid; ++i) {
    const uint32_t f = (uint32_t)(codes[i] >> 32);
    if (i == 0 || f != (uint32_t)(codes[i - 1] >> 32)) {
      a.grp.start[at] = i;
      a.grp.feature[at++] = (int)f;
    }
  }
  __syncthreads();
  if (t == 0) {
    a.grp.start[nseg] = nvalid;
    a.grp.state[0] = nseg;
    sm[32] = 0;
  }
  __syncthreads();
  for (int s = t; s < nseg; s += kSmallThreads) {
    const int begin = a.grp.start[s], n = a.grp.start[s + 1] - begin;
    if (n <= kPart) continue;
    const int parts = (n + kPart - 1) / kPart, first = atomicAdd(&sm[32], parts);
    for (int p = 0; p < parts; ++p)
      a.grp.part[first + p] = Part{a.grp.feature[s], begin + p * kPart, min(kPart, n - p * kPart), first + p, first, parts};
    a.grp.arrived[first] = 0;
  }
  __syncthreads();
  if (t == 0) a.grp.state[1] = sm[32];
}

// ---------------------------------------------------------------------------
// Many codes: least significant digit radix sort, tiles of 2048 codes.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pass_key(const GradArgs& a, int pass, int64_t i) {
  return pass == 0 ? feature_key(a, i) : a.grp.key[pass & 1][i];
}

__global__ void __launch_bounds__(kTileThreads) radix_count_kernel(const __grid_constant__ GradArgs a, int pass, int shift,
                                                                   int bits) {
  __shared__ int hist[1 << kMaxBits];
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < bins; i += kTileThreads) hist[i] = 0;
  if (pass == 0 && blockIdx.x == 0) {
    if (threadIdx.x < 2) a.grp.state[threadIdx.x] = 0;
    for (int64_t i = threadIdx.x; i < (a.d + 127) / 128; i += kTileThreads) a.grp.col_arrived[i] = 0;
  }
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTile;
  for (int i = threadIdx.x; i < kTile && base + i < a.N; i += kTileThreads)
    atomicAdd(&hist[(pass_key(a, pass, base + i) >> shift) & (bins - 1)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += kTileThreads) a.grp.count[(int64_t)i * gridDim.x + blockIdx.x] = hist[i];
}

// Warp per bin: exclusive sums of its counts over the tiles, and the total.
__global__ void __launch_bounds__(256) radix_prefix_kernel(const __grid_constant__ GradArgs a, int bins, int tiles) {
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
// of features with more than kPart codes.
__global__ void __launch_bounds__(256) bounds_kernel(const __grid_constant__ GradArgs a) {
  const int64_t f = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (f > a.F) return;
  const uint32_t* const key = a.grp.key[a.final_buf];
  int at[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    int lo = 0, hi = (int)a.N;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (key[mid] < (uint32_t)(f + q)) lo = mid + 1;
      else hi = mid;
    }
    at[q] = lo;
  }
  a.grp.start[f] = at[0];
  const int n = at[1] - at[0];
  if (f == a.F || n <= kPart) return;
  const int parts = (n + kPart - 1) / kPart, first = atomicAdd(&a.grp.state[1], parts);
  for (int p = 0; p < parts; ++p)
    a.grp.part[first + p] = Part{(int)f, at[0] + p * kPart, min(kPart, n - p * kPart), first + p, first, parts};
  a.grp.arrived[first] = 0;
}

__global__ void __launch_bounds__(256) column_sum_kernel(const __grid_constant__ GradArgs a) { column_sum(a, blockIdx.x); }

// ---------------------------------------------------------------------------
// Eight of a slab's 256 columns per lane: neighbours where rows are 16-byte
// aligned (VEC), else every 32nd.
// ---------------------------------------------------------------------------
template <typename T, bool VEC>
__device__ __forceinline__ void load_cols(const T* row, int64_t base, int lane, int64_t d, float (&w)[8]) {
  if constexpr (VEC) {
    const int64_t c = base + lane * 8;
    if (c < d) {
      load8(row + c, w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t c = base + lane + 32 * i;
      w[i] = c < d ? as_f32(row[c]) : 0.f;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_cols(T* row, int64_t base, int lane, int64_t d, const float (&w)[8]) {
  if constexpr (VEC) {
    const int64_t c = base + lane * 8;
    if (c < d) store8(row + c, w);
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

// A warp's list of codes: its rows, values and gradients.
struct List {
  int row[kPart];
  float v[kPart];
  float dv[kPart];
};

template <typename T, bool DEC, bool ENC, bool VEC>
__device__ __forceinline__ void run_list(const GradArgs& a, List& s, int64_t f, int begin, int n, int slot, int lane) {
  const uint32_t* const id = a.grp.id[a.final_buf];
  for (int i = lane; i < n; i += 32) {
    const uint32_t e = id[begin + i];
    s.row[i] = (int)(e / (uint32_t)a.k);
    s.v[i] = DEC ? a.V[e] : 0.f;
    s.dv[i] = a.gv != nullptr ? a.gv[e] : 0.f;
  }
  __syncwarp();
  if constexpr (DEC) {
    const T* const w_row = static_cast<const T*>(a.W_dec) + f * a.d;
    for (int64_t base = 0; base < a.d; base += 256) {
      float w[8], acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      load_cols<T, VEC>(w_row, base, lane, a.d, w);
      for (int i = 0; i < n; i += 4) {
        float x[4][8], dot[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (i + q < n) {
            load_cols<float, VEC>(a.g + (int64_t)s.row[i + q] * a.d, base, lane, a.d, x[q]);
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) x[q][c] = 0.f;
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float v = i + q < n ? s.v[i + q] : 0.f;
          dot[q] = 0.f;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            acc[c] = fmaf(v, x[q][c], acc[c]);
            dot[q] = fmaf(w[c], x[q][c], dot[q]);
          }
        }
        // four sums over the warp at once: lane 16 a + 8 b ends with the sum of dot[2 a + b]
        const bool up = lane & 16, mid = lane & 8;
        float p0 = (up ? dot[2] : dot[0]) + __shfl_xor_sync(kFull, up ? dot[0] : dot[2], 16);
        float p1 = (up ? dot[3] : dot[1]) + __shfl_xor_sync(kFull, up ? dot[1] : dot[3], 16);
        float p = (mid ? p1 : p0) + __shfl_xor_sync(kFull, mid ? p0 : p1, 8);
        p += __shfl_xor_sync(kFull, p, 4);
        p += __shfl_xor_sync(kFull, p, 2);
        p += __shfl_xor_sync(kFull, p, 1);
        const int at = i + (lane >> 3);
        if ((lane & 7) == 0 && at < n) s.dv[at] += p;
      }
      if (slot >= 0)
        store_cols<float, VEC>(a.grp.part_dec + (int64_t)slot * a.d, base, lane, a.d, acc);
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
    for (int64_t base = 0; base < a.d; base += 256) {
      float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < n; i += 4) {
        float x[4][8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (i + q < n) {
            load_cols<T, VEC>(static_cast<const T*>(a.X) + (int64_t)s.row[i + q] * a.d, base, lane, a.d, x[q]);
          } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) x[q][c] = 0.f;
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float v = i + q < n ? s.dv[i + q] : 0.f;
#pragma unroll
          for (int c = 0; c < 8; ++c) acc[c] = fmaf(v, x[q][c], acc[c]);
        }
      }
      if (slot >= 0)
        store_cols<float, VEC>(a.grp.part_enc + (int64_t)slot * a.d, base, lane, a.d, acc);
      else
        store_cols<T, VEC>(static_cast<T*>(a.dW_enc) + f * a.d, base, lane, a.d, acc);
    }
  }
  __syncwarp();
}

// Adds a long list's parts in order, once the last of them is done.
template <typename T, bool VEC>
__device__ __noinline__ void join_parts(const GradArgs& a, const float* from, T* to, int first, int parts, int lane) {
  for (int64_t base = 0; base < a.d; base += 256) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < parts; ++p) {
      // from L2: other SMs wrote these rows during this kernel
      const float* const row = from + (int64_t)(first + p) * a.d;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int64_t col = VEC ? base + lane * 8 + c : base + lane + 32 * c;
        if (col < a.d) acc[c] += __ldcg(row + col);
      }
    }
    store_cols<T, VEC>(to, base, lane, a.d, acc);
  }
}

template <typename T, bool DEC, bool ENC, bool VEC>
__global__ void __launch_bounds__(32 * kGradWarps) sae_grad_kernel(const __grid_constant__ GradArgs a) {
  __shared__ List lists[kGradWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  List& s = lists[warp];
  const int64_t me = (int64_t)blockIdx.x * kGradWarps + warp, all = (int64_t)gridDim.x * kGradWarps;
  // Parts of long lists first: they take longest, and the joins hide behind the rest.
  const int parts = a.grp.state[1];
  for (int64_t t = me; t < parts; t += all) {
    const Part p = a.grp.part[t];
    run_list<T, DEC, ENC, VEC>(a, s, p.feature, p.begin, p.n, p.slot, lane);
    __threadfence();
    __syncwarp();
    int done = 0;
    if (lane == 0) done = atomicAdd(&a.grp.arrived[p.first], 1) == p.parts - 1;
    if (!__shfl_sync(kFull, done, 0)) continue;
    __threadfence();
    if constexpr (DEC)
      join_parts<T, VEC>(a, a.grp.part_dec, static_cast<T*>(a.dW_dec) + (int64_t)p.feature * a.d, p.first, p.parts, lane);
    if constexpr (ENC) {
      join_parts<T, VEC>(a, a.grp.part_enc, static_cast<T*>(a.dW_enc) + (int64_t)p.feature * a.d, p.first, p.parts, lane);
      if (lane == 0) {
        float b = 0.f;
        for (int q = 0; q < p.parts; ++q) b += __ldcg(&a.grp.part_b[p.first + q]);
        a.db_enc[p.feature] = b;
      }
    }
  }
  const int64_t tasks = a.small ? a.grp.state[0] : a.F;
  // The other way round, so that warps with a part more have a feature less.
  for (int64_t t = all - 1 - me; t < tasks; t += all) {
    const int begin = a.grp.start[t], n = a.grp.start[t + 1] - begin;
    if (n > kPart) continue;
    const int64_t f = a.small ? a.grp.feature[t] : t;
    run_list<T, DEC, ENC, VEC>(a, s, f, begin, n, -1, lane);
  }
}

// dX_b = sum_j dv_bj W_enc[i_bj]: a warp per row and slab of 256 columns.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128) dx_kernel(const __grid_constant__ GradArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t slabs = (a.d + 255) / 256;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); t < a.B * slabs; t += (int64_t)gridDim.x * 4) {
    const int64_t b = t / slabs, base = (t % slabs) * 256;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < a.k; j0 += 32) {
      const int left = min(32, a.k - j0);
      int fi = lane < left ? a.I[b * a.k + j0 + lane] : -1;
      if ((uint32_t)fi >= (uint32_t)a.F) fi = -1;
      const float di = fi >= 0 ? a.dv[b * a.k + j0 + lane] : 0.f;
#pragma unroll 4
      for (int j = 0; j < left; ++j) {
        const int f = __shfl_sync(kFull, fi, j);
        const float dv = __shfl_sync(kFull, di, j);
        if (f < 0) continue;
        float w[8];
        load_cols<T, VEC>(static_cast<const T*>(a.W_enc) + (int64_t)f * a.d, base, lane, a.d, w);
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = fmaf(dv, w[c], acc[c]);
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
  int passes, bits[3], tiles, slots, chunks;
  size_t bytes;
};

// Where each array of the workspace lies; with `base` null only the size.
Plan lay_out(int64_t B, int64_t k, int64_t F, int64_t d, char* base, Group* g) {
  Plan p = {};
  const int64_t N = B * k;
  p.small = N <= kSmallCodes;
  int bits = 1;
  while (bits < 31 && ((int64_t)1 << bits) <= F) ++bits;  // the keys 0 .. F
  p.passes = (bits + kMaxBits - 1) / kMaxBits;
  for (int i = 0; i < p.passes; ++i) p.bits[i] = bits / p.passes + (i < bits % p.passes ? 1 : 0);
  p.tiles = (int)((N + kTile - 1) / kTile);
  p.slots = (int)(2 * (N / kPart));  // lists longer than kPart: at most N / kPart of them, and N / kPart full parts
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
  r.state = static_cast<int*>(take(8));
  r.arrived = static_cast<int*>(take(4 * (size_t)p.slots));
  r.part = static_cast<Part*>(take(sizeof(Part) * (size_t)p.slots));
  r.part_dec = static_cast<float*>(take(4 * (size_t)p.slots * d));
  r.part_enc = static_cast<float*>(take(4 * (size_t)p.slots * d));
  r.part_b = static_cast<float*>(take(4 * (size_t)p.slots));
  r.colsum = static_cast<float*>(take(p.chunks > 1 ? 4 * (size_t)p.chunks * d : 0));
  r.col_arrived = static_cast<int*>(take(4 * (size_t)((d + 127) / 128)));
  p.bytes = at;
  return p;
}

template <typename T, bool VEC>
void launch_main(const GradArgs& a, bool dec, bool enc, int sms, cudaStream_t s) {
  const int64_t tasks = a.small ? std::min(a.N, a.F) : a.F;
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>((tasks + kGradWarps - 1) / kGradWarps, sms * 6));
  if (dec && enc)
    sae_grad_kernel<T, true, true, VEC><<<grid, 32 * kGradWarps, 0, s>>>(a);
  else if (dec)
    sae_grad_kernel<T, true, false, VEC><<<grid, 32 * kGradWarps, 0, s>>>(a);
  else
    sae_grad_kernel<T, false, true, VEC><<<grid, 32 * kGradWarps, 0, s>>>(a);
  if (a.dX != nullptr) {
    const int64_t warps = a.B * ((a.d + 255) / 256);
    dx_kernel<T, VEC><<<(unsigned)std::min<int64_t>((warps + 3) / 4, sms * 16), 128, 0, s>>>(a);
  }
}

template <typename T>
void launch_type(const GradArgs& a, bool vec, bool dec, bool enc, int sms, cudaStream_t s) {
  if (vec) launch_main<T, true>(a, dec, enc, sms, s);
  else launch_main<T, false>(a, dec, enc, sms, s);
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
  if (!aligned_to(workspace, 16)) return host_fail(STK_EINVAL, "stk_sae_backward: workspace must be 16-byte aligned");
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
  int sms = 0;
  if (const int rc = host_device_sms(&sms)) return rc;
  cudaError_t e;
  if (p.small) {
    int padded = 2;
    while (padded < a.N) padded <<= 1;
    e = cudaFuncSetAttribute(small_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmallCodes * 8);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute");
    small_group_kernel<<<1 + 2 * sms, kSmallThreads, 8 * (size_t)padded, s>>>(a, padded, (int64_t)dict);
  } else {
    e = cudaFuncSetAttribute(radix_scatter_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             4 * kTileWarps << kMaxBits);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute");
    for (int pass = 0, shift = 0; pass < p.passes; shift += p.bits[pass++]) {
      const int bins = 1 << p.bits[pass];
      radix_count_kernel<<<p.tiles, kTileThreads, 0, s>>>(a, pass, shift, p.bits[pass]);
      radix_prefix_kernel<<<(bins + 7) / 8, 256, 0, s>>>(a, bins, p.tiles);
      radix_scatter_kernel<<<p.tiles, kTileThreads, 4 * (size_t)kTileWarps * bins, s>>>(a, pass, shift, p.bits[pass]);
    }
    bounds_kernel<<<(unsigned)(F / 256 + 1), 256, 0, s>>>(a);
    if (db_dec) column_sum_kernel<<<(unsigned)((d + 127) / 128 * p.chunks), 256, 0, s>>>(a);
  }
  e = cudaGetLastError();
  if (e != cudaSuccess) return host_cuda_fail(e, "stk_sae_backward: grouping launch");
  if (dX && !dec) a.dv = const_cast<float*>(grad_vals);  // read by dx_kernel alone
  bool vec = d % 8 == 0 && aligned_to(grad_out, 16);
  for (const void* q : {X, W_enc, W_dec, (const void*)dW_enc, (const void*)dW_dec, (const void*)dX}) vec &= aligned_to(q, 16);
  if (dtype == STK_F32) launch_type<float>(a, vec, dec, enc, sms, s);
  if (dtype == STK_F16) launch_type<__half>(a, vec, dec, enc, sms, s);
  if (dtype == STK_BF16) launch_type<__nv_bfloat16>(a, vec, dec, enc, sms, s);
  e = cudaGetLastError();
  if (e != cudaSuccess) return host_cuda_fail(e, "sae_grad_kernel launch");
  return STK_OK;
  STK_ENTRY_END
}
