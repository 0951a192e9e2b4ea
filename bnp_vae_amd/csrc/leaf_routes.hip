// From responsibilities to rows in leaf order and back: the k likeliest leaves of every frame, the stable counting
// sort of the (frame, choice) slots by leaf, the copy of frames' rows into that order and the weighted sum back, each
// with its gradient.  All of it is bound by memory; no kernel here adds with atomics on floating-point values, so
// every result has the same bits on every launch.
#include "layers_common.h"

namespace bnpvi {

// ------------------------------------------------------------------------------------------------------------------
// Top leaves.  A row is read once, 16 bytes a lane where it is aligned; LPR lanes share a row (a wave holds 64 / LPR
// rows), each keeps its own K best in order, then K rounds of a maximum over the LPR lanes take the best heads off.
// Ties: a lane visits its columns in ascending order and only a larger value moves an earlier one down; between
// lanes the lowest column among the equal heads wins.  What is not a finite positive number is never taken.
// Bound by the read of phi: 1M x 64, k = 2 in 61 us (272 MB, 4.5 TB/s), 150k x 512, k = 4 in 67 us (312 MB, 4.7 TB/s).
template <int K>
struct Best {
  float v[K];
  int i[K];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      v[j] = 0.f;
      i[j] = 0x7fffffff;
    }
  }
  __device__ __forceinline__ void add(float x, int col) {
    if (!(x > v[K - 1]) || !(x < __builtin_inff())) return;
    v[K - 1] = x;
    i[K - 1] = col;
#pragma unroll
    for (int j = K - 1; j > 0; --j) {
      const bool up = v[j] > v[j - 1];
      const float a = v[j - 1], b = v[j];
      const int ia = i[j - 1], ib = i[j];
      v[j - 1] = up ? b : a;
      v[j] = up ? a : b;
      i[j - 1] = up ? ib : ia;
      i[j] = up ? ia : ib;
    }
  }
  __device__ __forceinline__ void pop() {
#pragma unroll
    for (int j = 0; j + 1 < K; ++j) {
      v[j] = v[j + 1];
      i[j] = i[j + 1];
    }
    v[K - 1] = 0.f;
    i[K - 1] = 0x7fffffff;
  }
};

template <int K, int LPR, int VEC>
__global__ __launch_bounds__(256) void top_leaves_kernel(const float* __restrict__ phi, int64_t ldphi, int64_t N, int L, int k,
                                                         int renorm, int32_t* __restrict__ leaf, float* __restrict__ weight,
                                                         float* __restrict__ total) {
  constexpr int RPB = 256 / LPR;
  const int sub = threadIdx.x % LPR, r = threadIdx.x / LPR;
  for (int64_t n0 = (int64_t)blockIdx.x * RPB; n0 < N; n0 += (int64_t)gridDim.x * RPB) {
    const int64_t n = n0 + r;
    const bool live = n < N;
    Best<K> best;
    best.clear();
    if (live) {
      const float* row = phi + n * ldphi;
      for (int c = sub * VEC; c < L; c += LPR * VEC) {
        if (VEC == 4) {
          const f32x4 q = *reinterpret_cast<const f32x4*>(row + c);    // c + 3 < ldphi: columns from L on are skipped
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < L) best.add(q[e], c + e);
        } else {
          best.add(row[c], c);
        }
      }
    }
    float myv = 0.f;
    int myi = -1;
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (j < k) {
        const float m = lanes_max<LPR>(best.v[0]);
        const int at = lanes_min<LPR>(best.v[0] == m ? best.i[0] : 0x7fffffff);
        if (best.i[0] == at) best.pop();      // columns are distinct: one lane of the row holds it (or all are empty)
        if (sub == j) {                       // K <= 8 <= LPR: one lane a choice
          myv = m;
          myi = m > 0.f ? at : -1;
        }
        sum += (double)m;
      }
    }
    if (live) {
      if (sub < k) {
        leaf[n * k + sub] = myi;
        weight[n * k + sub] = renorm ? (sum > 0.0 ? (float)((double)myv / sum) : 0.f) : myv;
      }
      if (total != nullptr && sub == 0) total[n] = (float)sum;
    }
  }
}

// The gradient writes every column of every row: bound by those stores, which pass the caches, and by the wait for the
// few values of a row in front of them, so a lane takes R rows at once (1M x 64, k = 2: 63 us for 280 MB, 4.4 TB/s).
template <int K, int LPR, int VEC>
__global__ __launch_bounds__(256) void top_leaves_bwd_kernel(const int32_t* __restrict__ leaf, const float* __restrict__ weight,
                                                             const float* __restrict__ total, const float* __restrict__ dweight,
                                                             int64_t N, int k, int renorm, float* __restrict__ dphi, int64_t ld,
                                                             int cols) {
  constexpr int RPB = 256 / LPR, R = K <= 2 ? 4 : K <= 4 ? 2 : 1;
  const int sub = threadIdx.x % LPR, r = threadIdx.x / LPR;
  for (int64_t n0 = (int64_t)blockIdx.x * RPB * R + r; n0 < N; n0 += (int64_t)gridDim.x * RPB * R) {
    int at[R][K];
    float g[R][K], w[R][K], s[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t n = n0 + i * RPB;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const bool on = j < k && n < N;
        at[i][j] = on ? leaf[n * k + j] : -1;
        g[i][j] = on ? dweight[n * k + j] : 0.f;
        w[i][j] = on && renorm ? weight[n * k + j] : 0.f;
      }
      s[i] = renorm && n < N ? total[n] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t n = n0 + i * RPB;
      if (n >= N) break;
      if (renorm) {
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) dot = at[i][j] >= 0 ? fmaf(g[i][j], w[i][j], dot) : dot;
#pragma unroll
        for (int j = 0; j < K; ++j) g[i][j] = s[i] > 0.f ? (g[i][j] - dot) / s[i] : 0.f;
      }
      float* row = dphi + n * ld;
      for (int c = sub * VEC; c < cols; c += LPR * VEC) {
        f32x4 q = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const int e = at[i][j] - c;          // leaves differ, so at most one lands on each column
          q[0] = e == 0 ? g[i][j] : q[0];
          if (VEC == 4) {
            q[1] = e == 1 ? g[i][j] : q[1];
            q[2] = e == 2 ? g[i][j] : q[2];
            q[3] = e == 3 ? g[i][j] : q[3];
          }
        }
        if (VEC == 4)
          __builtin_nontemporal_store(q, reinterpret_cast<f32x4*>(row + c));
        else
          row[c] = q[0];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Stable counting sort of M slots by leaf, slots without a leaf behind the last one (bin L).  A workgroup owns a
// contiguous chunk, each of its W waves a contiguous part of it.  Counting is order-free (integer LDS adds).  Placing
// keeps the order: a wave takes 64 slots at a time, finds the lanes that hold the same leaf by one ballot per bit of
// the leaf number, and the lowest of them advances that leaf's place in the wave's own LDS row -- no wave writes
// another's row, so nothing is added atomically and the result is the stable order itself.  Bound by launches and the
// waits between the steps: 524k slots, 64 leaves 6 + 5 + 12 us (count, scan, place); 900k slots, 7776 leaves 6 + 9 + 30.
__device__ __forceinline__ int bin_of(int32_t l, int L) { return (uint32_t)l < (uint32_t)L ? l : L; }

__global__ __launch_bounds__(1024) void leaf_count_kernel(const int32_t* __restrict__ leaf, int64_t M, int L, int64_t chunk,
                                                         int32_t* __restrict__ hist) {
  extern __shared__ int32_t cnt[];
  const int B = L + 1;
  for (int i = threadIdx.x; i < B; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * chunk, hi = min(M, lo + chunk);
  for (int64_t s = lo + threadIdx.x; s < hi; s += blockDim.x) atomicAdd(&cnt[bin_of(leaf[s], L)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < B; i += blockDim.x) hist[(int64_t)blockIdx.x * B + i] = cnt[i];
}

// hist[b][bin] -> slots of that bin in the chunks before b; start[bin] = slots of the lower bins of its 64, sums[i] =
// slots of the i-th 64 bins.  64 bins a workgroup, 16 waves that share the chunks.
__global__ __launch_bounds__(1024) void leaf_scan_kernel(int32_t* __restrict__ hist, int nb, int B, int32_t* __restrict__ start,
                                                         int32_t* __restrict__ sums) {
  __shared__ int32_t part[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int bin = blockIdx.x * 64 + lane;
  const int per = (nb + 15) / 16, b0 = min(nb, w * per), b1 = min(nb, b0 + per);
  int32_t sum = 0;
  if (bin < B) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += hist[(int64_t)b * B + bin];
  }
  part[w][lane] = sum;
  __syncthreads();
  int32_t run = 0;
  for (int i = 0; i < w; ++i) run += part[i][lane];
  if (w == 15) {
    const int32_t all = run + sum;
    int32_t inc = all;
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    if (bin < B) start[bin] = inc - all;
    if (lane == 63) sums[blockIdx.x] = inc;
  }
  if (bin < B) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
      const int32_t h = hist[(int64_t)b * B + bin];
      hist[(int64_t)b * B + bin] = run;
      run += h;
    }
  }
}

// Exclusive scan of a[0 .. n) in LDS by the whole workgroup; red: one int per wave.
__device__ void scan_in_lds(int32_t* a, int n, int32_t* red) {
  const int T = blockDim.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int per = (n + T - 1) / T, i0 = min(n, t * per), i1 = min(n, i0 + per);
  int32_t sum = 0;
  for (int i = i0; i < i1; ++i) sum += a[i];
  int32_t inc = sum;
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t o = __shfl_up(inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 63) red[w] = inc;
  __syncthreads();
  int32_t run = inc - sum;
  for (int i = 0; i < w; ++i) run += red[i];
  for (int i = i0; i < i1; ++i) {
    const int32_t v = a[i];
    a[i] = run;
    run += v;
  }
  __syncthreads();
}

// LDS: base[W][B] | sums[max(B, bins of 64)] | red[16].  The first W waves place, all of them do the work over the bins.
// One workgroup (hist == nullptr) does the whole sort: counts, scan, places.
__global__ __launch_bounds__(1024) void leaf_place_kernel(const int32_t* __restrict__ leaf, int64_t M, int L, int64_t chunk, int bits,
                                                          int W, const int32_t* __restrict__ hist, const int32_t* __restrict__ start,
                                                          const int32_t* __restrict__ sums, int32_t* __restrict__ place,
                                                          int32_t* __restrict__ order, int32_t* __restrict__ offsets) {
  extern __shared__ int32_t lds[];
  const int B = L + 1, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int nsum = (B + 63) / 64;
  int32_t* mine = lds + (size_t)w * B;
  int32_t* firsts = lds + (size_t)W * B;               // of the bins (one workgroup) or of each 64 bins
  int32_t* red = firsts + (hist != nullptr ? nsum : B);
  const int64_t lo = (int64_t)blockIdx.x * chunk, hi = min(M, lo + chunk);
  const int64_t per = ((hi - lo + W - 1) / W + 63) / 64 * 64;
  const int64_t s0 = w < W ? min(hi, lo + w * per) : hi, s1 = min(hi, s0 + per);
  for (int i = threadIdx.x; i < W * B; i += blockDim.x) lds[i] = 0;
  if (hist != nullptr)
    for (int i = threadIdx.x; i < nsum; i += blockDim.x) firsts[i] = sums[i];
  __syncthreads();
  for (int64_t s = s0 + lane; s < s1; s += 64) atomicAdd(&mine[bin_of(leaf[s], L)], 1);
  __syncthreads();
  if (hist != nullptr) {
    scan_in_lds(firsts, nsum, red);
  } else {
    for (int i = threadIdx.x; i < B; i += blockDim.x) {
      int32_t sum = 0;
      for (int v = 0; v < W; ++v) sum += lds[(size_t)v * B + i];
      firsts[i] = sum;
    }
    __syncthreads();
    scan_in_lds(firsts, B, red);
  }
#pragma unroll 2
  for (int i = threadIdx.x; i < B; i += blockDim.x) {
    const int32_t at = hist != nullptr ? firsts[i >> 6] + start[i] : firsts[i];
    if (blockIdx.x == 0) offsets[i] = at;            // offsets[L] = slots with a leaf = first place without one
    int32_t run = at + (hist != nullptr ? hist[(int64_t)blockIdx.x * B + i] : 0);
    for (int v = 0; v < W; ++v) {
      const int32_t c = lds[(size_t)v * B + i];
      lds[(size_t)v * B + i] = run;
      run += c;
    }
  }
  __syncthreads();
  for (int64_t s = s0; s < s1; s += 64) {
    const int64_t at = s + lane;
    const bool live = at < s1;
    const int bin = live ? bin_of(leaf[at], L) : 0;
    uint64_t peers = __ballot(live);
    for (int b = 0; b < bits; ++b) {
      const uint64_t one = __ballot((bin >> b) & 1);
      peers &= ((bin >> b) & 1) ? one : ~one;
    }
    if (live) {
      const int rank = __popcll(peers & ((1ull << lane) - 1));
      const int32_t from = *(volatile int32_t*)&mine[bin];
      const int32_t p = from + rank;
      if (rank == 0) *(volatile int32_t*)&mine[bin] = from + (int32_t)__popcll(peers);
      place[at] = p;
      order[p] = (int32_t)at;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Frames of a workgroup that takes `rpb` at a time.  With `runs` every XCD has a contiguous run of them: neighbours in leaf
// order are about L / k frames apart, and where their rows share 128-byte lines they meet in one XCD's L2 (300k frames,
// k = 3, 100 floats, 64 leaves: to the leaves 137 -> 120 us, backward 263 -> 242).  Rows of whole lines share none, and go
// faster with the XCDs side by side (262k frames, k = 2, 256 bf16: 77 us to the leaves, 86 in runs); rows too far apart for
// the L2's 4 MB gain nothing (7776 leaves: the whole exchange 299 us, 303 in runs).
static bool in_runs(int64_t L, int64_t pitch_bytes) { return pitch_bytes % 128 != 0 && L * pitch_bytes <= (2 << 20); }

struct Frames {
  int64_t first, end, step;
  __device__ __forceinline__ Frames(int64_t N, int rpb, bool runs) {
    const uint32_t xcds = runs && gridDim.x >= 8 ? 8 : 1, xcd = blockIdx.x % xcds;
    const int64_t per = (N + (int64_t)xcds * rpb - 1) / ((int64_t)xcds * rpb) * rpb;
    first = xcd * per + (int64_t)(blockIdx.x / xcds) * rpb;
    end = min(N, (xcd + 1) * per);
    step = (int64_t)((gridDim.x + xcds - 1 - xcd) / xcds) * rpb;
  }
};

// A row is read and written in pieces of 16 bytes whatever its width and wherever it starts (global memory takes any
// address): the last piece ends with the row and shares elements with the one before it, both write the same values there.
// 1M rows of 37 floats: 130 us to the leaves and 171 us back one float a lane, 61 and 73 us in pieces.  Rows
// shorter than a piece are copied in pieces of 4 bytes, if they have so many, and computed element by element.
//
// Bound by memory: 262k x 256 bf16, k = 2 to the leaves in 65 us (403 MB), back in 87 (4.6 TB/s), backward in 133 (671 MB,
// 5.0 TB/s; part of it lies in the memory-side cache).
//
// Rows into leaf order.  A frame's row is read once and written to its k places; rows of slots without a leaf, which
// lie from offsets[L] on, are zeroed.  tx lanes share a row, a piece of `V` a lane.
template <typename V>
__global__ __launch_bounds__(256) void rows_to_leaves_kernel(const char* __restrict__ x, int64_t ldx, int64_t N, int k, int row, int tx,
                                                             const int32_t* __restrict__ place, const int32_t* __restrict__ kept_at,
                                                             char* __restrict__ xs, int64_t ldxs, bool runs) {
  const int sub = threadIdx.x % tx, r = threadIdx.x / tx, rpb = 256 / tx;
  const int32_t kept = *kept_at;
  const int64_t M = N * k;
  const Frames f(N, rpb, runs);
  for (int64_t n = f.first + r; n < f.end; n += f.step) {
    const int32_t* pl = place + n * k;
    for (int i = sub * (int)sizeof(V); i < row; i += tx * (int)sizeof(V)) {
      const int c = min(i, row - (int)sizeof(V));
      const V v = *reinterpret_cast<const V*>(x + n * ldx + c);
      for (int j = 0; j < k; ++j) {
        const int32_t p = pl[j];
        if ((uint32_t)p < (uint64_t)M) *reinterpret_cast<V*>(xs + (int64_t)p * ldxs + c) = p < kept ? v : V{};
      }
    }
  }
}

// y[n] = sum_j w[n][j] ys[place[n][j]] over the slots with a leaf (w = 1 where `weight` is null: the gradient of the
// copy above); fp32 sums in the order of j, one rounding.  E elements a lane: a piece, or one.
template <typename T, int E>
__global__ __launch_bounds__(256) void rows_from_leaves_kernel(const T* __restrict__ ys, int64_t ldys, const int32_t* __restrict__ place,
                                                               const float* __restrict__ weight, const int32_t* __restrict__ kept_at,
                                                               int64_t N, int k, int D, int tx, T* __restrict__ y, int64_t ldy, bool runs) {
  const int sub = threadIdx.x % tx, r = threadIdx.x / tx, rpb = 256 / tx;
  const int32_t kept = (int32_t)max((int64_t)0, min((int64_t)*kept_at, N * k));          // no read goes behind the rows
  const Frames f(N, rpb, runs);
  for (int64_t n = f.first + r; n < f.end; n += f.step) {
    for (int i = sub * E; i < D; i += tx * E) {
      const int c = min(i, D - E);
      float acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      for (int j0 = 0; j0 < k; j0 += 4) {          // four rows under way at once, added in order
        float v[4][E], w[4];
        bool in[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int32_t p = j0 + j < k ? place[n * k + j0 + j] : -1;
          in[j] = (uint32_t)p < (uint32_t)kept;
          w[j] = in[j] ? (weight != nullptr ? weight[n * k + j0 + j] : 1.f) : 0.f;
          if (in[j]) load_piece<T, E>(ys + (int64_t)p * ldys + c, v[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (in[j]) {
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(w[j], v[j][e], acc[e]);
          }
      }
      store_piece<T, E>(y + n * ldy + c, acc);
    }
  }
}

// dys[place[n][j]] = w[n][j] dy[n], dweight[n][j] = <dy[n], ys[place[n][j]]>; zeros for slots without a leaf.  The tx
// lanes of a row add their parts of the inner product in a fixed order, each element once.
template <typename T, int E>
__global__ __launch_bounds__(256) void rows_from_leaves_bwd_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ ys,
                                                                   int64_t ldys, const int32_t* __restrict__ place,
                                                                   const float* __restrict__ weight, const int32_t* __restrict__ kept_at,
                                                                   int64_t N, int k, int D, int tx, T* __restrict__ dys, int64_t lddys,
                                                                   float* __restrict__ dweight, bool runs) {
  const int sub = threadIdx.x % tx, r = threadIdx.x / tx, rpb = 256 / tx;
  const int32_t kept = *kept_at;
  const int64_t M = N * k;
  const Frames f(N, rpb, runs);
  for (int64_t n0 = f.first; n0 < f.end; n0 += f.step) {          // the same turns for every lane: the sums below use all of a row's
    const int64_t n = n0 + r;
    for (int j = 0; j < k; ++j) {
      float dot = 0.f;
      if (n < f.end) {
        const int32_t p = place[n * k + j];
        const bool in = (uint32_t)p < (uint32_t)kept;
        const float w = in ? weight[n * k + j] : 0.f;
        if ((uint32_t)p < (uint64_t)M) {
          for (int i = sub * E; i < D; i += tx * E) {
            const int c = min(i, D - E), again = i - c;          // elements that the piece before has too
            float g[E], o[E];
            load_piece<T, E>(dy + n * lddy + c, g);
            if (in) {
              float v[E];
              load_piece<T, E>(ys + (int64_t)p * ldys + c, v);
#pragma unroll
              for (int e = 0; e < E; ++e) dot = e < again ? dot : fmaf(g[e], v[e], dot);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = in ? w * g[e] : 0.f;
            if (dys != nullptr) store_piece<T, E>(dys + (int64_t)p * lddys + c, o);
          }
        }
      }
      for (int d = 1; d < tx; d <<= 1) dot += __shfl_xor(dot, d);
      if (n < f.end && sub == 0 && dweight != nullptr) dweight[n * k + j] = dot;
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
static int grid_for(const bnpvi_ctx* ctx, int64_t blocks) {
  const int64_t most = (int64_t)ctx->num_cu * 32;         // 8 resident workgroups of 256 per CU, four turns
  return (int)(blocks < 1 ? 1 : blocks < most ? blocks : most);
}

template <int LPR, int VEC>
static void launch_top(const bnpvi_ctx* ctx, const float* phi, int64_t ld, int64_t N, int L, int k, int renorm, int32_t* leaf,
                       float* weight, float* total, hipStream_t s) {
  const int g = grid_for(ctx, ceil_div(N, 256 / LPR));
  if (k == 1)
    top_leaves_kernel<1, LPR, VEC><<<g, 256, 0, s>>>(phi, ld, N, L, k, renorm, leaf, weight, total);
  else if (k == 2)
    top_leaves_kernel<2, LPR, VEC><<<g, 256, 0, s>>>(phi, ld, N, L, k, renorm, leaf, weight, total);
  else if (k <= 4)
    top_leaves_kernel<4, LPR, VEC><<<g, 256, 0, s>>>(phi, ld, N, L, k, renorm, leaf, weight, total);
  else
    top_leaves_kernel<8, LPR, VEC><<<g, 256, 0, s>>>(phi, ld, N, L, k, renorm, leaf, weight, total);
}

template <int K>
static void launch_top_bwd(const bnpvi_ctx* ctx, const int32_t* leaf, const float* weight, const float* total, const float* dweight,
                           int64_t N, int k, int renorm, float* dphi, int64_t ld, int cols, bool vec, hipStream_t s) {
  if (vec && cols <= 32)
    top_leaves_bwd_kernel<K, 8, 4><<<grid_for(ctx, ceil_div(N, 32)), 256, 0, s>>>(leaf, weight, total, dweight, N, k, renorm, dphi, ld, cols);
  else if (vec && cols <= 128)
    top_leaves_bwd_kernel<K, 16, 4><<<grid_for(ctx, ceil_div(N, 16)), 256, 0, s>>>(leaf, weight, total, dweight, N, k, renorm, dphi, ld, cols);
  else if (vec)
    top_leaves_bwd_kernel<K, 64, 4><<<grid_for(ctx, ceil_div(N, 4)), 256, 0, s>>>(leaf, weight, total, dweight, N, k, renorm, dphi, ld, cols);
  else
    top_leaves_bwd_kernel<K, 64, 1><<<grid_for(ctx, ceil_div(N, 4)), 256, 0, s>>>(leaf, weight, total, dweight, N, k, renorm, dphi, ld, cols);
}

// lanes that share a row of `n` accesses: a power of two up to a wave
static int lanes_for(int64_t n) {
  int tx = 1;
  while (tx < 64 && tx < n) tx <<= 1;
  return tx;
}

template <typename T>
static void launch_from(const bnpvi_ctx* ctx, const T* ys, int64_t ldys, const int32_t* place, const float* weight,
                        const int32_t* kept, int L, int64_t N, int k, int D, T* y, int64_t ldy, hipStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const int tx = lanes_for(D >= E ? ceil_div(D, E) : D);
  const int g = grid_for(ctx, ceil_div(N, 256 / tx));
  const bool runs = in_runs(L, ldys * sizeof(T));
  if (D >= E)
    rows_from_leaves_kernel<T, E><<<g, 256, 0, s>>>(ys, ldys, place, weight, kept, N, k, D, tx, y, ldy, runs);
  else
    rows_from_leaves_kernel<T, 1><<<g, 256, 0, s>>>(ys, ldys, place, weight, kept, N, k, D, tx, y, ldy, runs);
}

template <typename T>
static void launch_from_bwd(const bnpvi_ctx* ctx, const T* dy, int64_t lddy, const T* ys, int64_t ldys, const int32_t* place,
                            const float* weight, const int32_t* kept, int L, int64_t N, int k, int D, T* dys, int64_t lddys, float* dweight,
                            hipStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const int tx = lanes_for(D >= E ? ceil_div(D, E) : D);
  const int g = grid_for(ctx, ceil_div(N, 256 / tx));
  const bool runs = in_runs(L, ldys * sizeof(T));
  if (D >= E)
    rows_from_leaves_bwd_kernel<T, E><<<g, 256, 0, s>>>(dy, lddy, ys, ldys, place, weight, kept, N, k, D, tx, dys, lddys, dweight, runs);
  else
    rows_from_leaves_bwd_kernel<T, 1><<<g, 256, 0, s>>>(dy, lddy, ys, ldys, place, weight, kept, N, k, D, tx, dys, lddys, dweight, runs);
}

}  // namespace bnpvi

using namespace bnpvi;

extern "C" {

int bnpvi_top_leaves_max(void) { return kTopMax; }

int bnpvi_top_leaves(bnpvi_ctx* ctx, const float* phi, int64_t ldphi, int64_t N, int L, int k, int renormalize, int32_t* leaf,
                     float* weight, float* total, void* stream) {
  BNPVI_REQUIRE(ctx != nullptr, "bnpvi_top_leaves: ctx is NULL");
  BNPVI_REQUIRE(N >= 0 && N < (int64_t(1) << 33), "bnpvi_top_leaves: N=%lld", (long long)N);
  BNPVI_REQUIRE(L >= 1 && ldphi >= L, "bnpvi_top_leaves: L=%d, ldphi=%lld (a row holds at least L columns)", L, (long long)ldphi);
  BNPVI_REQUIRE(k >= 1 && k <= kTopMax && k <= L, "bnpvi_top_leaves: k=%d (1 .. min(%d, L=%d))", k, kTopMax, L);
  if (N == 0) return BNPVI_OK;
  BNPVI_REQUIRE(phi && leaf && weight, "bnpvi_top_leaves: NULL device pointer");
  OnDevice on(ctx->device);
  BNPVI_HIP(on.status());
  hipStream_t s = (hipStream_t)stream;
  // 16-byte loads read up to column roundup(L, 4) - 1 of a row, so the pitch has to cover it
  const bool vec = ldphi % 4 == 0 && ((uintptr_t)phi & 15) == 0;
  if (vec) {
    if (L <= 32)
      launch_top<8, 4>(ctx, phi, ldphi, N, L, k, renormalize, leaf, weight, total, s);
    else if (L <= 1024)      // four rows a wave: the rounds cost the same for one row or four (150k x 512, k = 4: 99 us one row a wave)
      launch_top<16, 4>(ctx, phi, ldphi, N, L, k, renormalize, leaf, weight, total, s);
    else
      launch_top<64, 4>(ctx, phi, ldphi, N, L, k, renormalize, leaf, weight, total, s);
  } else {
    if (L <= 32)
      launch_top<16, 1>(ctx, phi, ldphi, N, L, k, renormalize, leaf, weight, total, s);
    else
      launch_top<64, 1>(ctx, phi, ldphi, N, L, k, renormalize, leaf, weight, total, s);
  }
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

int bnpvi_top_leaves_backward(bnpvi_ctx* ctx, const int32_t* leaf, const float* weight, const float* total, const float* dweight,
                              int64_t N, int L, int k, int renormalize, float* dphi, int64_t lddphi, int cols, void* stream) {
  BNPVI_REQUIRE(ctx != nullptr, "bnpvi_top_leaves_backward: ctx is NULL");
  BNPVI_REQUIRE(N >= 0 && N < (int64_t(1) << 33), "bnpvi_top_leaves_backward: N=%lld", (long long)N);
  BNPVI_REQUIRE(k >= 1 && k <= kTopMax && k <= L, "bnpvi_top_leaves_backward: k=%d (1 .. min(%d, L=%d))", k, kTopMax, L);
  BNPVI_REQUIRE(cols >= L && lddphi >= cols, "bnpvi_top_leaves_backward: L=%d, cols=%d, lddphi=%lld", L, cols, (long long)lddphi);
  if (N == 0) return BNPVI_OK;
  BNPVI_REQUIRE(leaf && dweight && dphi && (!renormalize || (weight && total)), "bnpvi_top_leaves_backward: NULL device pointer");
  OnDevice on(ctx->device);
  BNPVI_HIP(on.status());
  hipStream_t s = (hipStream_t)stream;
  const bool vec = lddphi % 4 == 0 && cols % 4 == 0 && ((uintptr_t)dphi & 15) == 0;
  if (k == 1)
    launch_top_bwd<1>(ctx, leaf, weight, total, dweight, N, k, renormalize, dphi, lddphi, cols, vec, s);
  else if (k == 2)
    launch_top_bwd<2>(ctx, leaf, weight, total, dweight, N, k, renormalize, dphi, lddphi, cols, vec, s);
  else if (k <= 4)
    launch_top_bwd<4>(ctx, leaf, weight, total, dweight, N, k, renormalize, dphi, lddphi, cols, vec, s);
  else
    launch_top_bwd<8>(ctx, leaf, weight, total, dweight, N, k, renormalize, dphi, lddphi, cols, vec, s);
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

// ---- sort: sizes of one call ---------------------------------------------------------------------------------------
struct SortPlan {
  bool single;                 // one workgroup, one launch, no workspace: its LDS holds the firsts of all bins too
  int waves, threads, bits, nb;
  int64_t chunk;
  size_t lds;
};

static SortPlan sort_plan(int64_t M, int L) {
  SortPlan p;
  p.single = false;
  const int B = L + 1, nsum = (B + 63) / 64;
  p.bits = 1;
  while ((int64_t(1) << p.bits) < B) ++p.bits;
  if (M <= 8192 && (size_t)17 * B * 4 + 64 <= (size_t)kMaxLdsBytes) {
    // a minibatch: one workgroup, one launch (8192 slots, 512 leaves: 13.6 us, three launches 17.8; 16000: 22 and 17.9), of 16
    // waves but for the smallest (1000 slots, 512 leaves: 6.1 us, four waves 8.2; 256 slots, 25 leaves: 4.7 and 3.9)
    p.single = true;
    p.nb = 1;
    p.waves = M <= 512 && L <= 256 ? 4 : 16;
    p.threads = p.waves * 64;
    p.chunk = M < 1 ? 1 : M;
    p.lds = ((size_t)(p.waves + 1) * B + 16) * 4;
    return p;
  }
  // The counters of all placing waves have to fit the LDS.  Work over many bins is shared by 16 waves.
  p.waves = (size_t)(4 * B + nsum + 16) * 4 <= (size_t)kMaxLdsBytes ? 4 : 2;
  p.threads = B > 1024 ? 1024 : 256;
  // chunks of 2048 slots, longer where that makes more than 1024 of them, or -- where a chunk's counters outweigh its
  // slots -- more than one a CU (900k slots, 7776 leaves: 89 us with chunks of 7936, one for 43 % of the CUs)
  int64_t c = 2048;
  const int64_t most = B > 2048 ? 256 : 1024;
  if (ceil_div(M, c) > most) c = ceil_div(M, most);
  p.chunk = (c + 255) / 256 * 256;
  p.nb = (int)std::max<int64_t>(1, ceil_div(M, p.chunk));
  p.lds = ((size_t)p.waves * B + nsum + 16) * 4;
  return p;
}

int bnpvi_leaf_sort_max_leaves(void) { return kSortMaxLeaves; }

int64_t bnpvi_leaf_sort_workspace(int64_t M, int L) {
  if (M < 0 || M > INT32_MAX || L < 1 || L > kSortMaxLeaves) return -1;
  const SortPlan p = sort_plan(M, L);
  return p.single ? 0 : ((int64_t)(p.nb + 1) * (L + 1) + (L + 64) / 64) * 4;
}

int bnpvi_leaf_sort(bnpvi_ctx* ctx, const int32_t* leaf, int64_t M, int L, int32_t* place, int32_t* order, int32_t* offsets,
                    void* work, int64_t work_bytes, void* stream) {
  BNPVI_REQUIRE(ctx != nullptr, "bnpvi_leaf_sort: ctx is NULL");
  BNPVI_REQUIRE(M >= 0 && M <= INT32_MAX, "bnpvi_leaf_sort: M=%lld slots (0 .. 2^31 - 1)", (long long)M);
  BNPVI_REQUIRE(L >= 1 && L <= kSortMaxLeaves, "bnpvi_leaf_sort: L=%d (1 .. %d)", L, kSortMaxLeaves);
  BNPVI_REQUIRE(offsets && (M == 0 || (leaf && place && order)), "bnpvi_leaf_sort: NULL device pointer");
  const int64_t need = bnpvi_leaf_sort_workspace(M, L);
  BNPVI_REQUIRE(work_bytes >= need && (need == 0 || work != nullptr), "bnpvi_leaf_sort: workspace of %lld bytes, %lld needed",
                (long long)work_bytes, (long long)need);
  OnDevice on(ctx->device);
  BNPVI_HIP(on.status());
  hipStream_t s = (hipStream_t)stream;
  const SortPlan p = sort_plan(M, L);
  const int B = L + 1;
  static LdsLimit place_limit, count_limit;
  BNPVI_HIP(place_limit.raise((const void*)leaf_place_kernel, ctx->device));
  if (p.single) {
    leaf_place_kernel<<<1, p.threads, p.lds, s>>>(leaf, M, L, p.chunk, p.bits, p.waves, nullptr, nullptr, nullptr, place, order, offsets);
  } else {
    BNPVI_HIP(count_limit.raise((const void*)leaf_count_kernel, ctx->device));
    int32_t* hist = (int32_t*)work;
    int32_t* start = hist + (size_t)p.nb * B;
    int32_t* sums = start + B;
    leaf_count_kernel<<<p.nb, p.threads, (size_t)B * 4, s>>>(leaf, M, L, p.chunk, hist);
    leaf_scan_kernel<<<(B + 63) / 64, 1024, 0, s>>>(hist, p.nb, B, start, sums);
    leaf_place_kernel<<<p.nb, p.threads, p.lds, s>>>(leaf, M, L, p.chunk, p.bits, p.waves, hist, start, sums, place, order, offsets);
  }
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

static int check_rows(const char* what, bnpvi_ctx* ctx, int dtype, int64_t N, int k, int D, int L) {
  BNPVI_REQUIRE(ctx != nullptr, "%s: ctx is NULL", what);
  BNPVI_REQUIRE(dtype_bytes(dtype) > 0, "%s: dtype %d unknown", what, dtype);
  BNPVI_REQUIRE(k >= 1 && N >= 0 && N <= INT32_MAX / k, "%s: N=%lld, k=%d (N k below 2^31)", what, (long long)N, k);
  BNPVI_REQUIRE(D >= 1 && D <= (1 << 28), "%s: D=%d", what, D);
  BNPVI_REQUIRE(L >= 1, "%s: L=%d", what, L);
  return BNPVI_OK;
}

int bnpvi_rows_to_leaves(bnpvi_ctx* ctx, int dtype, const void* x, int64_t ldx, int64_t N, int k, int D, const int32_t* place,
                         const int32_t* offsets, int L, void* xs, int64_t ldxs, void* stream) {
  const int rc = check_rows("bnpvi_rows_to_leaves", ctx, dtype, N, k, D, L);
  if (rc) return rc;
  BNPVI_REQUIRE(ldx >= D && ldxs >= D, "bnpvi_rows_to_leaves: row pitch %lld / %lld below D=%d", (long long)ldx, (long long)ldxs, D);
  if (N == 0) return BNPVI_OK;
  BNPVI_REQUIRE(x && place && offsets && xs, "bnpvi_rows_to_leaves: NULL device pointer");
  OnDevice on(ctx->device);
  BNPVI_HIP(on.status());
  hipStream_t s = (hipStream_t)stream;
  const int e = dtype_bytes(dtype);
  const int64_t lx = ldx * e, ls = ldxs * e;
  const int row = D * e, tx = lanes_for(row >= 16 ? ceil_div(row, 16) : row >= 4 ? ceil_div(row, 4) : 1);
  const int g = grid_for(ctx, ceil_div(N, 256 / tx));
  const int32_t* kept = offsets + L;
  const bool runs = in_runs(L, ls);
  if (row >= 16)
    rows_to_leaves_kernel<u32x4_anywhere><<<g, 256, 0, s>>>((const char*)x, lx, N, k, row, tx, place, kept, (char*)xs, ls, runs);
  else if (row >= 4)
    rows_to_leaves_kernel<u32_anywhere><<<g, 256, 0, s>>>((const char*)x, lx, N, k, row, tx, place, kept, (char*)xs, ls, runs);
  else
    rows_to_leaves_kernel<uint16_t><<<g, 256, 0, s>>>((const char*)x, lx, N, k, row, tx, place, kept, (char*)xs, ls, runs);
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

int bnpvi_rows_from_leaves(bnpvi_ctx* ctx, int dtype, const void* ys, int64_t ldys, const int32_t* place, const float* weight,
                           const int32_t* offsets, int L, int64_t N, int k, int D, void* y, int64_t ldy, void* stream) {
  const int rc = check_rows("bnpvi_rows_from_leaves", ctx, dtype, N, k, D, L);
  if (rc) return rc;
  BNPVI_REQUIRE(ldys >= D && ldy >= D, "bnpvi_rows_from_leaves: row pitch %lld / %lld below D=%d", (long long)ldys, (long long)ldy, D);
  if (N == 0) return BNPVI_OK;
  BNPVI_REQUIRE(ys && place && offsets && y, "bnpvi_rows_from_leaves: NULL device pointer");
  OnDevice on(ctx->device);
  BNPVI_HIP(on.status());
  hipStream_t s = (hipStream_t)stream;
  const int32_t* kept = offsets + L;
  if (dtype == BNPVI_F32)
    launch_from<float>(ctx, (const float*)ys, ldys, place, weight, kept, L, N, k, D, (float*)y, ldy, s);
  else if (dtype == BNPVI_BF16)
    launch_from<bf16_t>(ctx, (const bf16_t*)ys, ldys, place, weight, kept, L, N, k, D, (bf16_t*)y, ldy, s);
  else
    launch_from<f16_t>(ctx, (const f16_t*)ys, ldys, place, weight, kept, L, N, k, D, (f16_t*)y, ldy, s);
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

int bnpvi_rows_from_leaves_backward(bnpvi_ctx* ctx, int dtype, const void* dy, int64_t lddy, const void* ys, int64_t ldys,
                                    const int32_t* place, const float* weight, const int32_t* offsets, int L, int64_t N, int k, int D,
                                    void* dys, int64_t lddys, float* dweight, void* stream) {
  const int rc = check_rows("bnpvi_rows_from_leaves_backward", ctx, dtype, N, k, D, L);
  if (rc) return rc;
  BNPVI_REQUIRE(lddy >= D && ldys >= D && (dys == nullptr || lddys >= D),
                "bnpvi_rows_from_leaves_backward: row pitch %lld / %lld / %lld below D=%d", (long long)lddy, (long long)ldys,
                (long long)lddys, D);
  if (N == 0) return BNPVI_OK;
  BNPVI_REQUIRE(dy && ys && place && weight && offsets, "bnpvi_rows_from_leaves_backward: NULL device pointer");
  if (dys == nullptr && dweight == nullptr) return BNPVI_OK;
  if (dys == nullptr) lddys = 0;
  OnDevice on(ctx->device);
  BNPVI_HIP(on.status());
  hipStream_t s = (hipStream_t)stream;
  const int32_t* kept = offsets + L;
  if (dtype == BNPVI_F32)
    launch_from_bwd<float>(ctx, (const float*)dy, lddy, (const float*)ys, ldys, place, weight, kept, L, N, k, D, (float*)dys, lddys,
                           dweight, s);
  else if (dtype == BNPVI_BF16)
    launch_from_bwd<bf16_t>(ctx, (const bf16_t*)dy, lddy, (const bf16_t*)ys, ldys, place, weight, kept, L, N, k, D, (bf16_t*)dys, lddys,
                            dweight, s);
  else
    launch_from_bwd<f16_t>(ctx, (const f16_t*)dy, lddy, (const f16_t*)ys, ldys, place, weight, kept, L, N, k, D, (f16_t*)dys, lddys,
                           dweight, s);
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

}  // extern "C"
