// Entry points of the dense product (dense_kernels.h) and the passes around its matrix kernel: the row tiles of the
// groups, dz = dy act'(z) with the bias gradient's partial sums, and the sums over partial results.
#include "dense_kernels.h"

namespace bnpvi {

// ---- row tiles of the groups ---------------------------------------------------------------------------------------
// map[t] = {group, first row, end row}; rows in front of the first and behind the last group make tiles of group -1,
// unused entries are empty.  first[g] = first tile of group g (first[G] = their number).  One workgroup: a scan of the
// groups' tile counts, then every tile finds its group by bisection.
__device__ __forceinline__ int64_t clamp_row(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// Exclusive scan of one value per thread over the workgroup of 1024; the sum of all in `total`.
__device__ int32_t scan_threads(int32_t v, int32_t* red, int32_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int32_t inc = v;
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t o = __shfl_up(inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 63) red[w] = inc;
  __syncthreads();
  int32_t run = inc - v;
  total = 0;
  for (int i = 0; i < 16; ++i) {
    if (i < w) run += red[i];
    total += red[i];
  }
  __syncthreads();
  return run;
}

__device__ void row_tiles(const int32_t* __restrict__ offsets, int G, int64_t M, int tile, int64_t ntiles, int4* __restrict__ map,
                          int32_t* __restrict__ first, int32_t* start, int32_t* red) {
  const int t = threadIdx.x;
  const int per = (G + 1023) / 1024, g0 = min(G, t * per), g1 = min(G, g0 + per);
  int32_t sum = 0, used;
  for (int g = g0; g < g1; ++g) {
    const int64_t lo = clamp_row(offsets[g], 0, M), hi = clamp_row(offsets[g + 1], lo, M);
    sum += (int32_t)((hi - lo + tile - 1) / tile);
  }
  int32_t run = scan_threads(sum, red, used);
  for (int g = g0; g < g1; ++g) {
    const int64_t lo = clamp_row(offsets[g], 0, M), hi = clamp_row(offsets[g + 1], lo, M);
    start[g] = run;
    run += (int32_t)((hi - lo + tile - 1) / tile);
  }
  if (t == 0) start[G] = used;
  __syncthreads();
  if (first != nullptr)
    for (int g = t; g <= G; g += 1024) first[g] = start[g];
  const int64_t head = clamp_row(offsets[0], 0, M), tail = clamp_row(offsets[G], 0, M);
  const int64_t nhead = (head + tile - 1) / tile;
  for (int64_t i = t; i < ntiles; i += 1024) {
    int4 m = {-1, 0, 0, 0};
    if (i < used) {
      int lo = 0, hi = G;                    // the last group that starts at or before tile i; empty groups share a start
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= i)
          lo = mid;
        else
          hi = mid;
      }
      const int64_t r0 = clamp_row(offsets[lo], 0, M), r1 = clamp_row(offsets[lo + 1], r0, M);
      const int64_t r = r0 + (i - start[lo]) * tile;
      if (r >= r0 && r < r1) {               // always, where the offsets ascend
        m.x = lo;
        m.y = (int)r;
        m.z = (int)(r + tile < r1 ? r + tile : r1);
      }
    } else {
      const int64_t j = i - used;
      const int64_t r0 = j < nhead ? j * tile : tail + (j - nhead) * tile, r1 = j < nhead ? head : M;
      if (r0 < r1) {
        m.y = (int)r0;
        m.z = (int)(r0 + tile < r1 ? r0 + tile : r1);
      }
    }
    map[i] = m;
  }
}

// ---- pieces of the groups' sums (dW) ---------------------------------------------------------------------------------
// Groups differ in length, and dW's tiles all have their group's: a group of more than `piece` frames is summed in pieces,
// whose partial results lie in `part`s of their own and are added in order afterwards.  map[e] = {group, first frame, end
// frame, part or -1}, the longest first by 64ths of a piece, and every second eight of them backwards: every eighth entry --
// one XCD's share -- is a like mixture.  (Entries of one 64th lie in any order; nothing is added in it.)  sums[i] = {group,
// first part, parts} of the groups in pieces; count = {entries, groups in pieces}.
constexpr int kLengths = 65;

__device__ void sum_pieces(const int32_t* __restrict__ offsets, int G, int64_t M, int64_t piece, int entries, int most, int4* __restrict__ map,
                           int4* __restrict__ sums, int32_t* __restrict__ count, int32_t* at, int32_t* red) {
  const int t = threadIdx.x;
  const int per = (G + 1023) / 1024, g0 = min(G, t * per), g1 = min(G, g0 + per);
  int32_t parts = 0, split = 0;
  auto look = [&](int g, int64_t& lo, int32_t& n, int64_t& left, int& shorter, bool& tail) {
    lo = clamp_row(offsets[g], 0, M);
    const int64_t len = clamp_row(offsets[g + 1], lo, M) - lo;
    n = (int32_t)(len / piece);
    left = len - n * piece;
    tail = left > 0 || len == 0;
    shorter = 64 - (int)(64 * left / piece);          // 0: a full piece
  };
  int64_t lo, left;
  int32_t n, used, all, unused;
  int shorter;
  bool tail;
  for (int i = t; i < kLengths; i += 1024) at[i] = 0;
  __syncthreads();
  for (int g = g0; g < g1; ++g) {
    look(g, lo, n, left, shorter, tail);
    if (n) atomicAdd(&at[0], n);
    if (tail) atomicAdd(&at[shorter], 1);
    if (n + tail > 1) {
      parts += n + tail;
      ++split;
    }
  }
  __syncthreads();
  const int32_t before = scan_threads(t < kLengths ? at[t] : 0, red, used);
  if (t < kLengths) at[t] = before;
  int32_t at_part = scan_threads(parts, red, unused), at_split = scan_threads(split, red, all);
  if ((uint32_t)used > (uint32_t)entries) used = entries;
  if (t == 0) {
    count[0] = used;
    count[1] = all < most ? all : most;
  }
  auto put = [&](int32_t rank, const int4& m) {
    const int32_t turn = rank >> 3, at_rank = (turn & 1) && 8 * turn + 8 <= used ? 8 * turn + 7 - (rank & 7) : rank;
    if ((uint32_t)rank < (uint32_t)used) map[at_rank] = m;
  };
  for (int g = g0; g < g1; ++g) {
    look(g, lo, n, left, shorter, tail);
    // the bounds hold wherever the offsets ascend; others are not followed out of the workspace
    const bool many = n + tail > 1 && (uint32_t)at_part < (uint32_t)(2 * most) && n + tail <= 2 * most - at_part;
    int32_t rank = n ? atomicAdd(&at[0], n) : 0;
    for (int32_t i = 0; i < n; ++i) put(rank + i, int4{g, (int)(lo + i * piece), (int)(lo + (i + 1) * piece), many ? at_part + i : -1});
    if (tail) put(atomicAdd(&at[shorter], 1), int4{g, (int)(lo + n * piece), (int)(lo + n * piece + left), many ? at_part + n : -1});
    if (many) {
      if ((uint32_t)at_split < (uint32_t)most) sums[at_split] = int4{g, at_part, n + tail, 0};
      ++at_split;
      at_part += n + tail;
    }
  }
}

// All maps of a call in one launch, a workgroup each.
struct MapArgs {
  const int32_t* offsets;
  int G;
  int64_t M;
  int tile[2];                 // row tiles: two maps at most
  int64_t ntiles[2];
  int4* map[2];
  int32_t* first[2];
  int64_t piece;               // pieces of the sums
  int entries, most;
  int4* pieces;
  int4* sums;
  int32_t* count;
};

__global__ __launch_bounds__(1024) void maps_kernel(const MapArgs a) {
  extern __shared__ int32_t start[];        // [G + 1 or kLengths] | [16]
  int32_t* red = start + max(a.G + 1, kLengths);
  if (blockIdx.x < 2) {
    if (a.map[blockIdx.x] != nullptr)
      row_tiles(a.offsets, a.G, a.M, a.tile[blockIdx.x], a.ntiles[blockIdx.x], a.map[blockIdx.x], a.first[blockIdx.x], start, red);
  } else if (a.pieces != nullptr) {
    sum_pieces(a.offsets, a.G, a.M, a.piece, a.entries, a.most, a.pieces, a.sums, a.count, start, red);
  }
}

// ---- dz, residual gradient, partial sums of the bias gradient --------------------------------------------------------
// One workgroup: a row tile (of one group) x 256 columns.  dz = dy * d, rounded once, or PAIR: in 16 bits in two parts
// hi + lo (dense_kernels.h): |dz - hi - lo| is at most 2^-16 of |dz| in bf16, 2^-22 in fp16 (where lo's smallest step adds
// 2^-25, half of dy's own).  hi stays finite where dz is -- a dz behind fp16's largest value, which is up to 1.13 dy, is 65504
// and the rest of it.  The bias gradient adds the unrounded products: per thread over its rows, then the eight row threads
// of a column in order, into `part`, or into `db` where one tile has all rows.  dres (or nullptr): dy, 0 in the rows of no
// group.  Bound by memory: 131072 x 512 in bf16 takes 130 us for 671 MB (5.1 TB/s).
template <typename T>
__device__ __forceinline__ void two_parts(float v, T& hi, T& lo) {
  constexpr float most = std::is_same<T, bf16_t>::value ? 3.3895313892515355e38f : 65504.f;
  const bool finite = fabsf(v) < __builtin_inff();
  hi = (T)(finite ? fminf(fmaxf(v, -most), most) : v);
  lo = (T)(finite ? v - (float)hi : 0.f);
}

constexpr int kDzRows = 128;

template <typename T, bool PAIR>
__global__ __launch_bounds__(256) void dz_kernel(const T* __restrict__ dy, int64_t lddy, const float* __restrict__ d, int64_t ldd,
                                                 const int4* __restrict__ map, int64_t M, int n, T* __restrict__ dz, int64_t lddz,
                                                 T* __restrict__ dres, int64_t lddres, float* __restrict__ part,
                                                 T* __restrict__ db) {
  constexpr int CT = 32, E = 8;              // threads across, columns a thread
  __shared__ float sums[8][CT * E + 1];
  const int tx = threadIdx.x % CT, ty = threadIdx.x / CT;
  int64_t r0 = (int64_t)blockIdx.x * kDzRows, r1 = min(M, r0 + kDzRows);
  int g = 0;
  if (map != nullptr) {
    const int4 m = map[blockIdx.x];
    g = m.x;
    r0 = m.y;
    r1 = m.z;
  }
  const int c = ((int)blockIdx.y * CT + tx) * E, inside = n - c;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (inside > 0 || (PAIR && dz != nullptr && 2 * c < lddz)) {
#pragma unroll 2
    for (int64_t r = r0 + ty; r < r1; r += 8) {
      float v[E], o[E];
      if (g < 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
        if (dres != nullptr) store_any<false, T, E>(dres + r * lddres + c, inside, o);
        continue;
      }
      load_any<T, E>(dy + r * lddy + c, inside, v);
      if (dres != nullptr) store_any<false, T, E>(dres + r * lddres + c, inside, v);
      if (d != nullptr) {
        load_any<float, E>(d + r * ldd + c, inside, o);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] *= o[e];
        if (dz != nullptr) {
          if constexpr (PAIR) {          // zeros behind column n up to the end of its 32
            union {
              u32x4 u;
              T t[E];
            } hi, lo;
#pragma unroll
            for (int e = 0; e < E; ++e) two_parts<T>(v[e], hi.t[e], lo.t[e]);
            T* at = dz + r * lddz + (c / 32) * 64 + c % 32;
            *reinterpret_cast<u32x4*>(at) = hi.u;
            *reinterpret_cast<u32x4*>(at + 32) = lo.u;
          } else {                       // zeros behind column n up to a whole 16 bytes
            store_any<false, T, E>(dz + r * lddz + c, (int)(lddz - c), v);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += v[e];
    }
  }
  if (part == nullptr && db == nullptr) return;
#pragma unroll
  for (int e = 0; e < E; ++e) sums[ty][tx * E + e] = acc[e];
  __syncthreads();
  for (int i = threadIdx.x; i < CT * E; i += 256) {
    const int col = (int)blockIdx.y * CT * E + i;
    if (col < n) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += sums[k][i];
      if (db != nullptr)
        db[col] = (T)s;
      else
        part[(int64_t)blockIdx.x * n + col] = s;
    }
  }
}

// ---- rows copied to a pitch of whole 16 bytes, zeros behind their end ------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void pad_rows_kernel(const T* __restrict__ src, int64_t ld, int64_t group, int64_t per_group, int64_t rows,
                                                       int width, int pieces, T* __restrict__ dst) {
  constexpr int PER = 16 / (int)sizeof(T);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * pieces; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / pieces, g = r / per_group;
    const int c = (int)(i - r * pieces) * PER, inside = width - c;
    const T* p = src + g * group + (r - g * per_group) * ld + c;
    union {
      u32x4 u;
      T t[PER];
    } q;
    if (inside >= PER) {
      const u32x4_anywhere v = *reinterpret_cast<const u32x4_anywhere*>(p);
      q.u = u32x4{v[0], v[1], v[2], v[3]};
    } else {
      q.u = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (e < inside) q.t[e] = p[e];
    }
    reinterpret_cast<u32x4*>(dst)[i] = q.u;
  }
}

// db[g] = sum over the group's row tiles, 16 interleaved partial sums per column, added in order
template <typename T>
__global__ __launch_bounds__(1024) void db_kernel(const float* __restrict__ part, const int32_t* __restrict__ first, int64_t tiles, int n,
                                                  T* __restrict__ db) {
  __shared__ float sums[16][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, g = blockIdx.y, col = blockIdx.x * 64 + tx;
  const int64_t t0 = first != nullptr ? clamp_row(first[g], 0, tiles) : 0;
  const int64_t t1 = first != nullptr ? clamp_row(first[g + 1], t0, tiles) : tiles;
  float acc = 0.f;
  if (col < n)
    #pragma unroll 8
    for (int64_t t = t0 + ty; t < t1; t += 16) acc += part[t * n + col];
  sums[ty][tx] = acc;
  __syncthreads();
  if (ty == 0 && col < n) {
#pragma unroll
    for (int k = 1; k < 16; ++k) acc += sums[k][tx];
    db[(int64_t)g * n + col] = (T)acc;
  }
}

// ---- sums over the splits of the reduce axis, in order, of dW and behind it of db ---------------------------------------
struct SumArgs {
  const float* slab[2];
  void* out[2];
  int64_t elems[2];
};

template <typename T>
__global__ __launch_bounds__(256) void split_sum_kernel(const SumArgs a, int splits) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.elems[0] + a.elems[1]; i += (int64_t)gridDim.x * 256) {
    const bool two = i >= a.elems[0];
    const int64_t elems = a.elems[two], e = two ? i - a.elems[0] : i;
    const float* p = a.slab[two] + e;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < splits; ++k) s += p[k * elems];
    reinterpret_cast<T*>(a.out[two])[e] = (T)s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void piece_sum_kernel(const SumArgs a, const int4* __restrict__ sums, const int32_t* __restrict__ count) {
  for (int g = blockIdx.y; g < count[1]; g += gridDim.y) {
    const int4 m = sums[g];
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.elems[0] + a.elems[1]; i += (int64_t)gridDim.x * 256) {
      const bool two = i >= a.elems[0];
      const int64_t elems = a.elems[two], e = two ? i - a.elems[0] : i;
      const float* p = a.slab[two] + m.y * elems + e;
      float s = 0.f;
#pragma unroll 4
      for (int k = 0; k < m.z; ++k) s += p[k * elems];
      reinterpret_cast<T*>(a.out[two])[m.x * elems + e] = (T)s;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void split_epilogue_kernel(const float* __restrict__ slab, int splits, const GemmArgs a) {
  const int64_t elems = a.rows * a.cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < elems; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / a.cols, col = i % a.cols;
    float z = 0.f;
    for (int k = 0; k < splits; ++k) z += slab[k * elems + i];
    if (a.bias != nullptr) z += (float)reinterpret_cast<const T*>(a.bias)[col];
    float v[1] = {z}, d[1];
    activate<sizeof(T) == 2, 1>(a.act, v, d);
    float y = v[0];
    if (a.res != nullptr) y += (float)reinterpret_cast<const T*>(a.res)[row * a.ldres + col];
    if (a.dact != nullptr) a.dact[row * a.lddact + col] = d[0];
    reinterpret_cast<T*>(a.C)[row * a.ldc + col] = (T)y;
  }
}

// ---- up to eight rows: products with vectors ---------------------------------------------------------------------------
// Bound by the weight's bytes (one frame: by the wait for them): a wave a column, 16 bytes a lane of its row of W, or four
// waves where rows are long and columns too few for all CUs, whose sums meet in LDS (8 x 4096 -> 1024 bf16: 6.5 us, one
// wave 7.4; 4 x 4096 -> 4096: 12.6, one wave 8.8; fp32 4 x 4096 -> 4096: 17.1 and 16.7, one row 11.9 and 13.1).
// The matrix kernel takes 32 rows whatever their number and parts of the sum to fill the chip (8 x 4096 -> 32: 14.7 us in
// bf16 and 22.5 in fp32, here 6.8 and 6.2), but reads x once a tile, where every column here reads all of it: 8 x 4096 ->
// 4096 in fp32 takes 23.5 us there and would take 34.4 here, six rows 23.3 and 23.5.
static bool as_vectors(int64_t M, int64_t K, int64_t n, int G) { return G == 0 && (M <= 4 || (M <= 8 && (double)M * K * n <= 1.0e8)); }

template <typename T>
struct Piece {
  static constexpr int kPer = 16 / (int)sizeof(T);
  union {
    u32x4_anywhere u;
    T t[kPer];
  } v;
  __device__ __forceinline__ void load(const T* p, int inside) {
    if (inside >= kPer) {
      v.u = *reinterpret_cast<const u32x4_anywhere*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) v.t[e] = e < inside ? p[e] : (T)0.f;
    }
  }
};
// acc + <a, b>, for 16 bits by the instruction that adds two products of a pair to an fp32 sum
template <typename T>
__device__ __forceinline__ float dot(const Piece<T>& a, const Piece<T>& b, float acc) {
#pragma unroll
  for (int e = 0; e < Piece<T>::kPer; e += sizeof(T) == 4 ? 1 : 2) {
    if constexpr (sizeof(T) == 4) {
      acc = fmaf(a.v.t[e], b.v.t[e], acc);
    } else {
      typedef T two __attribute__((ext_vector_type(2)));
      const two p = {a.v.t[e], a.v.t[e + 1]}, q = {b.v.t[e], b.v.t[e + 1]};
      if constexpr (std::is_same<T, bf16_t>::value)
        acc = __builtin_amdgcn_fdot2_f32_bf16(p, q, acc, false);
      else
        acc = __builtin_amdgcn_fdot2(p, q, acc, false);
    }
  }
  return acc;
}

template <typename T, int M, int WPC>
__global__ __launch_bounds__(256) void gemv_kernel(const GemmArgs a) {
  constexpr int PER = Piece<T>::kPer;
  __shared__ float sums[4][M];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, part = wave % WPC;
  const int64_t col = (int64_t)blockIdx.x * (4 / WPC) + wave / WPC;
  float acc[M];
#pragma unroll
  for (int m = 0; m < M; ++m) acc[m] = 0.f;
  if (col < a.cols) {
    const T* w = reinterpret_cast<const T*>(a.S) + col * a.lds;
    const T* x = reinterpret_cast<const T*>(a.R);
#pragma unroll 4
    for (int64_t k = (part * 64 + lane) * PER; k < a.K; k += WPC * 64 * PER) {
      const int inside = a.K - k < PER ? (int)(a.K - k) : PER;
      Piece<T> pw, px;
      pw.load(w + k, inside);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        px.load(x + m * a.ldr + k, inside);
        acc[m] = dot(px, pw, acc[m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
    for (int d = 32; d > 0; d >>= 1) acc[m] += __shfl_xor(acc[m], d);
  if (lane == 0) {
#pragma unroll
    for (int m = 0; m < M; ++m) sums[wave][m] = acc[m];
  }
  __syncthreads();
  const int m = lane;
  if (part != 0 || m >= M || col >= a.cols) return;
  float z[1] = {0.f}, d[1];
#pragma unroll
  for (int p = 0; p < WPC; ++p) z[0] += sums[wave + p][m];
  if (a.bias != nullptr) z[0] += (float)reinterpret_cast<const T*>(a.bias)[col];
  activate<sizeof(T) == 2, 1>(a.act, z, d);
  if (a.res != nullptr) z[0] += (float)reinterpret_cast<const T*>(a.res)[m * a.ldres + col];
  if (a.dact != nullptr) a.dact[m * a.lddact + col] = d[0];
  reinterpret_cast<T*>(a.C)[m * a.ldc + col] = (T)z[0];
}

template <typename T, int M>
static void launch_gemv(const GemmArgs& a, hipStream_t s) {
  if (a.K * (int64_t)sizeof(T) > 2048 && (sizeof(T) == 4 || a.cols < 2048))
    gemv_kernel<T, M, 4><<<(unsigned)a.cols, 256, 0, s>>>(a);
  else
    gemv_kernel<T, M, 1><<<(unsigned)ceil_div(a.cols, 4), 256, 0, s>>>(a);
}

template <typename T>
static void gemv(const GemmArgs& a, hipStream_t s) {
  switch (a.rows) {
    case 1:
      return launch_gemv<T, 1>(a, s);
    case 2:
      return launch_gemv<T, 2>(a, s);
    case 3:
      return launch_gemv<T, 3>(a, s);
    case 4:
      return launch_gemv<T, 4>(a, s);
    case 5:
      return launch_gemv<T, 5>(a, s);
    case 6:
      return launch_gemv<T, 6>(a, s);
    case 7:
      return launch_gemv<T, 7>(a, s);
    default:
      return launch_gemv<T, 8>(a, s);
  }
}

// ---- sizes of one call -----------------------------------------------------------------------------------------------
struct GemmPlan {
  int tile, splits;
  int64_t row_tiles;
  int col_tiles;
  size_t slab;                 // bytes
  int64_t piece;               // kDw with groups: frames of a piece, entries of its map and parts at most
  int64_t entries, parts;
};

static void tile_size(int tile, int& br, int& bc) {
  if (tile == kTile256) {
    br = bc = 256;
    return;
  }
  br = tile == kTile128 || tile == kTileTall ? 128 : tile == kTile64 ? 64 : 32;
  bc = tile == kTile128 || tile == kTileFlat ? 128 : tile == kTile64 ? 64 : 32;
}

// rows x cols of output, `K` summed; grouped: G groups along the rows (kFwd, kDx) or along the sum (kDw); direct: all
// operands' rows start on 16 bytes; pair: R in two parts, 32 k's a stage.
//
// The tile and the number of parts of the sum are the cheapest by what was measured.  A stage of 128 bytes of k takes a
// workgroup the microseconds below, by how many of them share a CU (8192^3 in 16 bits: 64 / 128 / 256 wide tiles make 384 /
// 560 / 760 outputs a nanosecond and stage, so the large tile wins wherever it fills the chip; fp32 is bound by its matrix
// rate), and a tile its first load and its epilogue.  65536 x 4096 -> 256: 207 us in tiles of 128, 173 in tiles of 256;
// 16384 x 512 -> 512: 15 us in tiles of 128, 22 in tiles of 256; 256 leaves of 200 rows, 512 -> 512: 80 and 102.
// Splitting the sum costs a launch and two passes over the parts.  Transposing reads cost the large tile's stages a tenth
// more (8192^3: 922 / 1044 / 1002 us forward, dx, dW).
//
// Narrow results take the tall tile (50000 x 1024 -> 32: 19 us in bf16 and 55 in fp32, tiles of 64: 22 and 81), few rows the
// flat one, and so do small leaves, whose last tile is half empty on average (256 leaves of 40 / 96 / 128 rows, 512 -> 512 in
// bf16: 39 / 52 / 67 us, tiles of 64 or 128: 41 / 57 / 62; fp32, of 40 / 200 rows: 122 / 332 us and 144 / 342).
//
// dW with groups: leaves are unequal, and a launch waits for its longest tile.  A leaf longer than `piece` frames is summed
// in pieces; the shorter they are the evener the end (half a piece is idle on average), the more partial results pass
// through memory.
static GemmPlan gemm_plan(int kind, int dtype, int64_t rows, int64_t cols, int64_t K, bool grouped, int G, bool direct, bool pair = false) {
  GemmPlan p;
  const int e = dtype_bytes(dtype), bk = pair ? 32 : 128 / e;
  const bool by_rows = grouped && kind != kDw;
  const bool by_sum = grouped && kind == kDw;
  const int64_t per_group = by_rows ? ceil_div(rows, G) : rows;
  p.piece = p.entries = p.parts = 0;
  p.splits = 1;
  if (cols <= 32 && per_group > 32 && !pair) {
    p.tile = kTileTall;
  } else if (per_group <= (by_rows ? (e == 4 ? 256 : 96) : 32)) {
    p.tile = kTileFlat;
  } else {
    p.tile = kTile64;
  }
  // kTile128, kTile64 (also for the narrow ones), kTile256; up to four workgroups a CU
  static const double k16[3][4] = {{0.9, 1.3, 1.3, 1.3}, {0.5, 0.6, 0.72, 0.84}, {1.83, 1.83, 1.83, 1.83}};
  static const double k32[3][4] = {{1.8, 3.5, 3.5, 3.5}, {0.6, 1.0, 1.5, 1.92}, {0, 0, 0, 0}};
  const double tile_cost[] = {5.0, 3.5, kind == kFwd ? 12.0 : kind == kDx ? 9.0 : 8.0};
  static const int kPerCu[] = {2, 4, 1};
  auto row_of = [](int tile) { return tile == kTile128 ? 0 : tile == kTile256 ? 2 : 1; };
  const int64_t stages = std::max<int64_t>(1, ceil_div(K, bk));
  auto tiles_of = [&](int tile) {
    int br, bc;
    tile_size(tile, br, bc);
    return (ceil_div(rows, br) + (by_rows ? G / 2 : 0)) * ceil_div(cols, bc);
  };
  // whole turns of a full chip and one of what is left, which has the CUs to itself
  auto cost = [&](int tile, int64_t s) {
    const int r = row_of(tile);
    const int64_t n = tiles_of(tile) * s, whole = n / (kPerCu[r] * kNumCU), rest = ceil_div(n % (kPerCu[r] * kNumCU), kNumCU);
    auto turn = [&](int64_t each) {
      return (double)ceil_div(stages, s) * (e == 4 ? k32 : k16)[r][each - 1] * (r == 2 ? 1.0 + 0.08 * kind : 1.0) + tile_cost[r];
    };
    return whole * turn(kPerCu[r]) + (rest ? turn(rest) : 0.0) + (s > 1 ? 4.0 + 8.0 * s * rows * cols / 4.0e6 : 0.0);
  };
  // groups of the sum, `len` stages a piece: the work, the pieces' first loads and epilogues, half a piece at the end, the
  // parts -- nearly all pieces where they are shorter than a leaf is on average, else those of the long leaves
  auto cost_of_pieces = [&](int tile, int64_t len) {
    const int r = row_of(tile);
    const double slots = (double)kPerCu[r] * kNumCU, tiles = (double)tiles_of(tile), work = tiles * (double)(stages + G / 2) / slots;
    const double full = (double)stages / (double)len, stage = (e == 4 ? k32 : k16)[r][kPerCu[r] - 1] * (r == 2 ? 1.16 : 1.0);
    const double parts = stages >= len * G ? full + G / 2 : 0.3 * full;
    return work * stage + (full + G) * tiles / slots * tile_cost[r] + 0.5 * len * stage + 4.0 + 8.0 * parts * rows * cols / 4.0e6;
  };
  const int64_t most = grouped ? 1 : std::min<int64_t>(64, std::max<int64_t>(1, stages / 2));
  const int tried[] = {p.tile, kTile128, kTile256};
  double best = 1e300;
  int tile = p.tile;
  for (int i = 0; i < (p.tile == kTile64 ? (direct && e == 2 ? 3 : 2) : 1); ++i) {
    if (by_sum) {
      const int r = row_of(tried[i]);
      const int64_t even = std::max<int64_t>(8, tiles_of(tried[i]) * stages / (kPerCu[r] * kNumCU));
      for (int64_t len = std::max<int64_t>(8, even / 2); len <= 8 * even; len *= 2) {
        const double c = cost_of_pieces(tried[i], len);
        if (c < best * 0.98) {
          best = c;
          tile = tried[i];
          p.piece = len * bk;
        }
      }
      continue;
    }
    for (int64_t s = 1; s <= most; s *= 2) {
      const double c = cost(tried[i], s);
      if (c < best * 0.98) {
        best = c;
        tile = tried[i];
        p.splits = (int)s;
      }
    }
  }
  p.tile = tile;
  if (const char* f = dev_getenv(kind == kFwd ? "BNPVI_TILE_FWD" : kind == kDx ? "BNPVI_TILE_DX" : "BNPVI_TILE_DW")) p.tile = atoi(f);
  if (const char* f = dev_getenv(kind == kFwd ? "BNPVI_SPLIT_FWD" : kind == kDx ? "BNPVI_SPLIT_DX" : "BNPVI_SPLIT_DW")) p.splits = atoi(f);
  if (const char* f = dev_getenv("BNPVI_PIECE_DW"); f && by_sum) p.piece = atoi(f) * bk;
  int br, bc;
  tile_size(p.tile, br, bc);
  p.row_tiles = ceil_div(rows, br) + (by_rows ? G + 2 : 0);
  p.col_tiles = (int)ceil_div(cols, bc);
  p.slab = p.splits > 1 ? (size_t)p.splits * rows * cols * 4 : 0;
  if (by_sum) {
    p.entries = K / p.piece + G;                                 // every group has one entry at least, and one that is not full
    p.parts = K > p.piece ? 2 * (K / p.piece) : 0;               // a group of more than a piece has two at most per full one
    p.slab = (size_t)p.parts * rows * cols * 4;
  }
  return p;
}

static size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// What a call's work and workspace go by: sizes, which operands lie on 16 bytes (`aligned`), and for a backward pass what it is
// given and asked for.
struct Call {
  int dtype;
  int64_t M, K, n;
  int G;
  bool x_lies, w_lies, dy_lies;
  bool dact, dx, dw, db, dres;
  bool step;                   // dact holds 0 and 1 only
};

struct ForwardPlan {
  GemmPlan gemm;
  bool direct, copy;           // the product loads straight into LDS; operands that do not lie are copied first
  int64_t Kp;                  // pitch of the copies, whole 16 bytes
  size_t map, slab, x, w, bytes;      // byte offsets of the workspace's parts, 0 bytes each where the call has no use for them
};

struct BackwardPlan {
  GemmPlan dx, dw;
  bool dx_direct, dw_direct, copy;
  bool pair;                   // dz in two 16-bit parts
  bool write_dz, dz_pass;      // dz is not dy; a pass over dy is needed
  bool db_in_dw, db_in_dz;
  int64_t dz_tiles, Kp, dz_pitch;     // pitches: of copies of x and W, of dz or of the copy of dy in its place
  size_t dz_map, dz_first, dx_map, dw_map, dw_sums, dw_count, part, dz, slab, db_slab, x, w, bytes;
};

static size_t take(size_t& at, size_t bytes) {
  const size_t o = at;
  at += up256(bytes);
  return o;
}

// Copying pays where the products are large: through registers they run at 0.3 PFLOP/s where straight loads reach 0.65
// (dW: 0.17 against 0.75; 32768 x 1023 -> 1021 in bf16: 225 / 267 / 399 us forward, dx, dW through registers, 107 / 90 / 90
// from rows of 1024, 30 us for the copy), and cost a launch and two passes over the operand.
static bool copy_pays(double flops_fwd, double flops_bwd, int e, int64_t M, int64_t Kp, int64_t weights) {
  return flops_fwd * 1.7e-9 + flops_bwd * 3.1e-9 > 10.0 + 2.0 * e * ((double)M * Kp + (double)weights * Kp) / 4.7e6;
}

static int64_t whole_pieces(int64_t width, int e) { return (width * e + 15) / 16 * 16 / e; }

static ForwardPlan forward_plan(const Call& c) {
  ForwardPlan p;
  const int e = dtype_bytes(c.dtype);
  const int64_t weights = c.n * (c.G > 0 ? c.G : 1);
  const bool lie = c.x_lies && c.w_lies, vector = as_vectors(c.M, c.K, c.n, c.G);
  p.Kp = whole_pieces(c.K, e);
  p.copy = !lie && !vector && copy_pays(2.0 * c.M * c.K * c.n, 0, e, c.M, p.Kp, weights);
  p.direct = lie || p.copy;
  p.gemm = gemm_plan(kFwd, c.dtype, c.M, c.n, c.K, c.G > 0, c.G, p.direct);
  size_t at = 0;
  p.map = take(at, c.G > 0 ? p.gemm.row_tiles * sizeof(int4) : 0);
  p.slab = take(at, vector ? 0 : p.gemm.slab);
  p.x = take(at, p.copy && !c.x_lies ? (size_t)c.M * p.Kp * e : 0);
  p.w = take(at, p.copy && !c.w_lies ? (size_t)weights * p.Kp * e : 0);
  p.bytes = at;
  return p;
}

static BackwardPlan backward_plan(const Call& c) {
  BackwardPlan p = {};
  const int e = dtype_bytes(c.dtype);
  const int64_t weights = c.n * (c.G > 0 ? c.G : 1);
  const bool grouped = c.G > 0, products = c.dx || c.dw;
  p.pair = c.dact && e == 2 && !c.step;          // dy times 0 or 1 is its 16 bits
  p.write_dz = c.dact && products;
  // dz is dy, or lies in the workspace
  const bool dz_lies = p.write_dz || c.dy_lies, w_lies = !c.dx || c.w_lies, x_lies = !c.dw || c.x_lies;
  p.Kp = whole_pieces(c.K, e);
  p.copy = c.M > 0 && products && !(dz_lies && w_lies && x_lies) &&
           copy_pays(0, 4.0 * c.M * c.K * c.n, e, c.M, whole_pieces(c.K + c.n + 16 / e, e), weights);
  p.dx_direct = p.copy || (dz_lies && w_lies);
  p.dw_direct = p.copy || (dz_lies && x_lies);
  if (c.dx) p.dx = gemm_plan(kDx, c.dtype, c.M, c.K, c.n, grouped, c.G, p.dx_direct, p.pair);
  if (c.dw) p.dw = gemm_plan(kDw, c.dtype, c.n, c.K, c.M, grouped, c.G, p.dw_direct, p.pair);
  // Without an activation the products read dy itself and dW's kernel adds up its rows for the bias on the way
  // (16385 x 64 -> 4096 fp32: 70 us of 450 were a pass over dy for that).  With one, dW's kernel sees 16 bits of dz in
  // two parts, so that there only fp32 does the same.
  p.db_in_dw = c.db && c.dw && (!c.dact || c.dtype == BNPVI_F32) && p.dw.tile != kTile256;
  p.dz_pass = p.write_dz || (c.db && !p.db_in_dw) || c.dres;
  p.dz_tiles = ceil_div(c.M, kDzRows) + (grouped ? c.G + 2 : 0);
  p.db_in_dz = c.db && !p.db_in_dw && !grouped && p.dz_tiles == 1 && c.M > 0;          // a launch less
  p.dz_pitch = p.pair ? (c.n + 31) / 32 * 64 : whole_pieces(c.n, e);
  size_t at = 0;
  p.dz_map = take(at, grouped && p.dz_pass ? p.dz_tiles * sizeof(int4) : 0);
  p.dz_first = take(at, grouped && p.dz_pass ? (size_t)(c.G + 1) * 4 : 0);
  p.dx_map = take(at, grouped && c.dx ? p.dx.row_tiles * sizeof(int4) : 0);
  p.dw_map = take(at, (size_t)p.dw.entries * sizeof(int4));
  p.dw_sums = take(at, (size_t)p.dw.parts / 2 * sizeof(int4));
  p.dw_count = take(at, grouped || c.M > 0 ? 8 : 0);          // also where it is not used: no call with rows goes without a workspace
  p.part = take(at, c.db && !p.db_in_dw && !p.db_in_dz ? (size_t)p.dz_tiles * c.n * 4 : 0);
  p.dz = take(at, p.write_dz || (p.copy && !dz_lies) ? (size_t)c.M * p.dz_pitch * e : 0);
  p.slab = take(at, std::max(p.dx.slab, p.dw.slab));
  p.db_slab = take(at, p.db_in_dw ? (size_t)(grouped ? p.dw.parts : p.dw.splits > 1 ? p.dw.splits : 0) * c.n * 4 : 0);
  p.x = take(at, p.copy && !x_lies ? (size_t)c.M * p.Kp * e : 0);
  p.w = take(at, p.copy && !w_lies ? (size_t)weights * p.Kp * e : 0);
  p.bytes = at;
  return p;
}

template <typename T>
static void pad_rows(const void* src, int64_t ld, int64_t group, int64_t per_group, int64_t rows, int64_t width, int64_t pitch, void* dst,
                     hipStream_t s) {
  const int pieces = (int)(pitch * sizeof(T) / 16);
  pad_rows_kernel<T><<<(unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows * pieces, 256), 8192)), 256, 0, s>>>(
      (const T*)src, ld, group, per_group, rows, (int)width, pieces, (T*)dst);
}

static void pad_rows(int dtype, const void* src, int64_t ld, int64_t group, int64_t per_group, int64_t rows, int64_t width, int64_t pitch,
                     void* dst, hipStream_t s) {
  if (dtype_bytes(dtype) == 4)
    pad_rows<uint32_t>(src, ld, group, per_group, rows, width, pitch, dst, s);
  else
    pad_rows<uint16_t>(src, ld, group, per_group, rows, width, pitch, dst, s);
}

// Every row of the operand starts on 16 bytes and its contiguous extent is whole pieces of them.
static bool aligned(const void* p, int64_t ld, int64_t group, int64_t extent, int e) {
  return (((uint64_t)(uintptr_t)p | (uint64_t)(ld * e) | (uint64_t)(group * e) | (uint64_t)(extent * e)) & 15) == 0;
}

static int run_gemm(int kind, int dtype, const GemmPlan& p, bool direct, bool pair, GemmArgs& a, const bnpvi_ctx* ctx, hipStream_t s) {
  a.row_tiles = (int)p.row_tiles;
  a.col_tiles = p.col_tiles;
  a.splits = p.splits;
  return dtype == BNPVI_F32    ? launch_gemm_f32(kind, p.tile, direct, pair, a, ctx, s)
         : dtype == BNPVI_BF16 ? launch_gemm_bf16(kind, p.tile, direct, pair, a, ctx, s)
                               : launch_gemm_f16(kind, p.tile, direct, pair, a, ctx, s);
}

static int launch_maps(const MapArgs& a, int device, hipStream_t s) {
  static LdsLimit limit;
  const size_t lds = (size_t)(std::max(a.G + 1, kLengths) + 16) * 4;
  if (lds > 64 * 1024) BNPVI_HIP(limit.raise((const void*)maps_kernel, device));
  maps_kernel<<<a.pieces ? 3 : a.map[1] ? 2 : 1, 1024, lds, s>>>(a);
  BNPVI_LAUNCH_CHECK();
  return BNPVI_OK;
}

static unsigned flat_grid(int64_t elems) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(elems, 256), 4096)); }

template <typename T>
static void launch_dz(bool pair, const void* dy, int64_t lddy, const void* d, int64_t ldd, const int4* map, int64_t M, int n, int64_t tiles,
                      void* dz, int64_t lddz, void* dres, int64_t lddres, float* part, void* db, hipStream_t s) {
  const dim3 grid((unsigned)tiles, (unsigned)ceil_div(n, 256));
  if constexpr (sizeof(T) == 2) {
    if (pair) {
      dz_kernel<T, true><<<grid, 256, 0, s>>>((const T*)dy, lddy, (const float*)d, ldd, map, M, n, (T*)dz, lddz, (T*)dres, lddres, part, (T*)db);
      return;
    }
  }
  dz_kernel<T, false><<<grid, 256, 0, s>>>((const T*)dy, lddy, (const float*)d, ldd, map, M, n, (T*)dz, lddz, (T*)dres, lddres, part, (T*)db);
}

template <typename T>
static void launch_db(const float* part, const int32_t* first, int64_t tiles, int n, int G, void* db, hipStream_t s) {
  db_kernel<T><<<dim3((unsigned)ceil_div(n, 64), (unsigned)G), 1024, 0, s>>>(part, first, tiles, n, (T*)db);
}

template <typename T>
static void launch_sums(const SumArgs& a, const GemmPlan& p, bool grouped, const int4* sums, const int32_t* count, hipStream_t s) {
  const int64_t elems = a.elems[0] + a.elems[1];
  if (grouped)
    piece_sum_kernel<T><<<dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(elems, 256), 1024)),
                               (unsigned)std::min<int64_t>(p.parts / 2, 64)),
                          256, 0, s>>>(a, sums, count);
  else
    split_sum_kernel<T><<<flat_grid(elems), 256, 0, s>>>(a, p.splits);
}

constexpr int64_t kMaxPitchBytes = int64_t(1) << 22;       // 256 rows of a tile stay below 2^31 bytes

static int check_dense(const char* what, bnpvi_ctx* ctx, int dtype, int64_t M, int64_t K, int64_t n, int G, const int32_t* offsets) {
  BNPVI_REQUIRE(ctx != nullptr, "%s: ctx is NULL", what);
  BNPVI_REQUIRE(dtype_bytes(dtype) > 0, "%s: dtype %d unknown", what, dtype);
  BNPVI_REQUIRE(M >= 0 && M <= INT32_MAX, "%s: M=%lld rows (0 .. 2^31 - 1)", what, (long long)M);
  BNPVI_REQUIRE(K >= 1 && K <= (1 << 20) && n >= 1 && n <= (1 << 20), "%s: K=%lld, n=%lld (1 .. 2^20)", what, (long long)K, (long long)n);
  BNPVI_REQUIRE(G >= 0 && G <= kSortMaxLeaves, "%s: G=%d groups (0 .. %d)", what, G, kSortMaxLeaves);
  BNPVI_REQUIRE((G > 0) == (offsets != nullptr), "%s: G=%d groups need offsets, and only they do", what, G);
  return BNPVI_OK;
}

static bool pitch_fits(int64_t ld, int64_t width, int dtype) {
  return ld >= width && ld * dtype_bytes(dtype) <= kMaxPitchBytes;
}

static bool sizes_fit(int dtype, int64_t M, int64_t K, int64_t n, int G) {
  return dtype_bytes(dtype) > 0 && M >= 0 && M <= INT32_MAX && K >= 1 && K <= (1 << 20) && n >= 1 && n <= (1 << 20) && G >= 0 && G <= kSortMaxLeaves;
}

}  // namespace bnpvi

using namespace bnpvi;

extern "C" {

int64_t bnpvi_dense_workspace_for(int dtype, int64_t M, int64_t K, int64_t n, int G, int call) {
  if (!sizes_fit(dtype, M, K, n, G)) return -1;
  auto has = [call](int bit) { return (call & bit) != 0; };
  const Call c = {dtype, M, K, n, G, !has(BNPVI_DENSE_X_OFF), !has(BNPVI_DENSE_W_OFF), !has(BNPVI_DENSE_DY_OFF), has(BNPVI_DENSE_DACT),
                  has(BNPVI_DENSE_DX), has(BNPVI_DENSE_DW), has(BNPVI_DENSE_DB), has(BNPVI_DENSE_DRES), has(BNPVI_DENSE_STEP)};
  return (int64_t)(has(BNPVI_DENSE_BACKWARD) ? backward_plan(c).bytes : forward_plan(c).bytes);
}

int64_t bnpvi_dense_workspace(int dtype, int64_t M, int64_t K, int64_t n, int G, int backward) {
  if (!sizes_fit(dtype, M, K, n, G)) return -1;
  // enough for every call of these sizes: wherever its operands lie, with and without an activation, with db in dW's pass or
  // not (a call that asks for less needs no more)
  int64_t most = 0;
  for (int off = 0; off < 8; ++off)
    for (int given = 0; given < (backward ? 8 : 1); ++given) {
      const int call = (off & 1 ? BNPVI_DENSE_X_OFF : 0) | (off & 2 ? BNPVI_DENSE_W_OFF : 0) | (off & 4 ? BNPVI_DENSE_DY_OFF : 0);
      const int asked = BNPVI_DENSE_BACKWARD | BNPVI_DENSE_DX | BNPVI_DENSE_DB | BNPVI_DENSE_DRES | (given & 1 ? BNPVI_DENSE_DACT : 0) |
                        (given & 2 ? 0 : BNPVI_DENSE_DW) | (given & 4 ? BNPVI_DENSE_STEP : 0);
      most = std::max(most, bnpvi_dense_workspace_for(dtype, M, K, n, G, backward ? call | asked : call));
    }
  return most;
}

int bnpvi_dense(bnpvi_ctx* ctx, int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t w_group, const void* bias,
                int64_t bias_group, int activation, const void* residual, int64_t ldres, const int32_t* offsets, int G, int64_t M,
                int64_t K, int64_t n, void* y, int64_t ldy, void* dact, int64_t lddact, void* work, int64_t work_bytes, void* stream) {
  const int rc = check_dense("bnpvi_dense", ctx, dtype, M, K, n, G, offsets);
  if (rc) return rc;
  BNPVI_REQUIRE(activation >= BNPVI_ACT_NONE && activation <= BNPVI_ACT_GELU, "bnpvi_dense: activation %d unknown", activation);
  BNPVI_REQUIRE(pitch_fits(ldx, K, dtype) && pitch_fits(ldw, K, dtype),
                "bnpvi_dense: pitches x %lld, w %lld for K=%lld (at least K, at most 4 MiB)", (long long)ldx, (long long)ldw, (long long)K);
  BNPVI_REQUIRE(ldy >= n && (!residual || ldres >= n) && (!dact || lddact >= n), "bnpvi_dense: pitch of y, residual or dact below n=%lld",
                (long long)n);
  if (M == 0) return BNPVI_OK;
  BNPVI_REQUIRE(x && w && y, "bnpvi_dense: NULL device pointer");
  const int e = dtype_bytes(dtype);
  Call c = {dtype, M, K, n, G};
  c.x_lies = aligned(x, ldx, 0, K, e);
  c.w_lies = aligned(w, ldw, G > 1 ? w_group : 0, K, e);
  const ForwardPlan p = forward_plan(c);
  BNPVI_REQUIRE(work_bytes >= (int64_t)p.bytes && (p.bytes == 0 || (work && (uintptr_t)work % 256 == 0)),
                "bnpvi_dense: workspace of %lld bytes (aligned to 256), %lld needed", (long long)work_bytes, (long long)p.bytes);
  OnDevice on(ctx->device);
  BNPVI_HIP(on.status());
  hipStream_t s = (hipStream_t)stream;
  char* wk = (char*)work;
  GemmArgs a = {};
  a.R = x;
  a.ldr = ldx;
  a.S = w;
  a.lds = ldw;
  a.s_group = G > 1 ? w_group : 0;
  a.rows = M;
  a.cols = n;
  a.K = K;
  a.C = y;
  a.ldc = ldy;
  a.bias = bias;
  a.bias_group = G > 1 ? bias_group : 0;
  a.res = residual;
  a.ldres = ldres;
  a.dact = (float*)dact;
  a.lddact = lddact;
  a.act = activation;
  if (as_vectors(M, K, n, G)) {
    if (dtype == BNPVI_F32)
      gemv<float>(a, s);
    else if (dtype == BNPVI_BF16)
      gemv<bf16_t>(a, s);
    else
      gemv<f16_t>(a, s);
    BNPVI_LAUNCH_CHECK();
    return BNPVI_OK;
  }
  if (G > 0) {
    int bc;
    MapArgs m = {};
    m.offsets = offsets;
    m.G = G;
    m.M = M;
    tile_size(p.gemm.tile, m.tile[0], bc);
    m.ntiles[0] = p.gemm.row_tiles;
    m.map[0] = (int4*)(wk + p.map);
    const int r = launch_maps(m, ctx->device, s);
    if (r) return r;
    a.map = (const int4*)(wk + p.map);
  }
  if (p.gemm.slab) a.slab = (float*)(wk + p.slab);
  if (p.copy) {
    const int64_t groups = G > 0 ? G : 1;
    if (!c.x_lies) {
      pad_rows(dtype, x, ldx, 0, M, M, K, p.Kp, wk + p.x, s);
      a.R = wk + p.x;
      a.ldr = p.Kp;
    }
    if (!c.w_lies) {
      pad_rows(dtype, w, ldw, w_group, n, groups * n, K, p.Kp, wk + p.w, s);
      a.S = wk + p.w;
      a.lds = p.Kp;
      a.s_group = G > 1 ? n * p.Kp : 0;
    }
    BNPVI_LAUNCH_CHECK();
  }
  const int r = run_gemm(kFwd, dtype, p.gemm, p.direct, false, a, ctx, s);
  if (r) return r;
  if (p.gemm.slab) {
    const unsigned g = flat_grid(M * n);
    if (dtype == BNPVI_F32)
      split_epilogue_kernel<float><<<g, 256, 0, s>>>(a.slab, p.gemm.splits, a);
    else if (dtype == BNPVI_BF16)
      split_epilogue_kernel<bf16_t><<<g, 256, 0, s>>>(a.slab, p.gemm.splits, a);
    else
      split_epilogue_kernel<f16_t><<<g, 256, 0, s>>>(a.slab, p.gemm.splits, a);
    BNPVI_LAUNCH_CHECK();
  }
  return BNPVI_OK;
}

int bnpvi_dense_backward_act(bnpvi_ctx* ctx, int dtype, int activation, const void* dy, int64_t lddy, const void* dact, int64_t lddact,
                             const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t w_group, const int32_t* offsets, int G,
                             int64_t M, int64_t K, int64_t n, void* dx, int64_t lddx, void* dw, void* db, void* dres, int64_t lddres,
                             void* work, int64_t work_bytes, void* stream) {
  const int rc = check_dense("bnpvi_dense_backward", ctx, dtype, M, K, n, G, offsets);
  if (rc) return rc;
  BNPVI_REQUIRE(activation >= -1 && activation <= BNPVI_ACT_GELU, "bnpvi_dense_backward: activation %d unknown", activation);
  BNPVI_REQUIRE(pitch_fits(lddy, n, dtype) && (!dact || lddact >= n) && (!dx || (pitch_fits(ldw, K, dtype) && lddx >= K)) &&
                    (!dw || pitch_fits(ldx, K, dtype)) && (!dres || lddres >= n),
                "bnpvi_dense_backward: a row pitch is below its width, or above 4 MiB");
  const int e = dtype_bytes(dtype);
  Call c = {dtype, M, K, n, G};
  c.x_lies = aligned(x, ldx, 0, K, e);
  c.w_lies = aligned(w, ldw, G > 1 ? w_group : 0, K, e);
  c.dy_lies = aligned(dy, lddy, 0, n, e);
  c.dact = dact != nullptr;
  c.dx = dx != nullptr;
  c.dw = dw != nullptr;
  c.db = db != nullptr;
  c.dres = dres != nullptr;
  c.step = dact && activation == BNPVI_ACT_RELU;
  const BackwardPlan p = backward_plan(c);
  BNPVI_REQUIRE(work_bytes >= (int64_t)p.bytes && (p.bytes == 0 || (work && (uintptr_t)work % 256 == 0)),
                "bnpvi_dense_backward: workspace of %lld bytes (aligned to 256), %lld needed", (long long)work_bytes, (long long)p.bytes);
  BNPVI_REQUIRE(M == 0 || (dy && (!dx || w) && (!dw || x)), "bnpvi_dense_backward: NULL device pointer");
  OnDevice on(ctx->device);
  BNPVI_HIP(on.status());
  hipStream_t s = (hipStream_t)stream;
  const int groups = G > 0 ? G : 1;
  char* wk = (char*)work;
  int r = BNPVI_OK;
  const int4* dz_map = nullptr;
  int32_t* first = nullptr;
  const bool none = M == 0;
  if (G > 0) {
    MapArgs m = {};
    int bc;
    m.offsets = offsets;
    m.G = G;
    m.M = M;
    if (p.dz_pass) {
      first = (int32_t*)(wk + p.dz_first);
      dz_map = (const int4*)(wk + p.dz_map);
      m.tile[0] = kDzRows;
      m.ntiles[0] = p.dz_tiles;
      m.map[0] = (int4*)(wk + p.dz_map);
      m.first[0] = first;
    }
    if (dx && !none) {
      tile_size(p.dx.tile, m.tile[1], bc);
      m.ntiles[1] = p.dx.row_tiles;
      m.map[1] = (int4*)(wk + p.dx_map);
    }
    if (dw) {
      m.piece = p.dw.piece;
      m.entries = (int)p.dw.entries;
      m.most = (int)(p.dw.parts / 2);
      m.pieces = (int4*)(wk + p.dw_map);
      m.sums = (int4*)(wk + p.dw_sums);
      m.count = (int32_t*)(wk + p.dw_count);
    }
    r = launch_maps(m, ctx->device, s);
    if (r) return r;
  }
  const void* dz = dy;
  int64_t lddz = lddy;
  void* db_in_dz = p.db_in_dz ? db : nullptr;
  float* part = db && !p.db_in_dw && !p.db_in_dz ? (float*)(wk + p.part) : nullptr;
  if (p.dz_pass && !none) {
    void* out = p.write_dz ? (void*)(wk + p.dz) : nullptr;
    const auto launch = dtype == BNPVI_F32 ? launch_dz<float> : dtype == BNPVI_BF16 ? launch_dz<bf16_t> : launch_dz<f16_t>;
    launch(p.pair, dy, lddy, dact, lddact, dz_map, M, (int)n, p.dz_tiles, out, p.dz_pitch, dres, lddres, part, db_in_dz, s);
    BNPVI_LAUNCH_CHECK();
    if (p.write_dz) {
      dz = out;
      lddz = p.dz_pitch;
    }
  }
  if (db && !p.db_in_dw && !p.db_in_dz) {
    const int64_t tiles = none ? 0 : p.dz_tiles;
    if (dtype == BNPVI_F32)
      launch_db<float>(part, first, tiles, (int)n, groups, db, s);
    else if (dtype == BNPVI_BF16)
      launch_db<bf16_t>(part, first, tiles, (int)n, groups, db, s);
    else
      launch_db<f16_t>(part, first, tiles, (int)n, groups, db, s);
    BNPVI_LAUNCH_CHECK();
  }
  const int64_t wg = G > 1 ? w_group : 0;
  const void *xs = x, *ws = w;
  int64_t ldxs = ldx, ldws = ldw, wgs = wg;
  if (p.copy) {
    if (!p.write_dz && !c.dy_lies) {
      pad_rows(dtype, dy, lddy, 0, M, M, n, p.dz_pitch, wk + p.dz, s);
      dz = wk + p.dz;
      lddz = p.dz_pitch;
    }
    if (dx && !c.w_lies) {
      pad_rows(dtype, w, ldw, w_group, n, groups * n, K, p.Kp, wk + p.w, s);
      ws = wk + p.w;
      ldws = p.Kp;
      wgs = G > 1 ? n * p.Kp : 0;
    }
    if (dw && !c.x_lies) {
      pad_rows(dtype, x, ldx, 0, M, M, K, p.Kp, wk + p.x, s);
      xs = wk + p.x;
      ldxs = p.Kp;
    }
    BNPVI_LAUNCH_CHECK();
  }
  if (dx && !none) {
    GemmArgs a = {};
    a.R = dz;
    a.ldr = lddz;
    a.S = ws;
    a.lds = ldws;
    a.s_group = wgs;
    a.rows = M;
    a.cols = K;
    a.K = n;
    a.C = dx;
    a.ldc = lddx;
    if (G > 0) a.map = (const int4*)(wk + p.dx_map);
    if (p.dx.slab) a.slab = (float*)(wk + p.slab);
    r = run_gemm(kDx, dtype, p.dx, p.dx_direct, p.pair, a, ctx, s);
    if (r) return r;
    if (p.dx.slab) {
      // no epilogue: a plain sum over the splits into rows of pitch lddx
      GemmArgs b = a;
      b.act = BNPVI_ACT_NONE;
      const unsigned g = flat_grid(M * K);
      if (dtype == BNPVI_F32)
        split_epilogue_kernel<float><<<g, 256, 0, s>>>(a.slab, p.dx.splits, b);
      else if (dtype == BNPVI_BF16)
        split_epilogue_kernel<bf16_t><<<g, 256, 0, s>>>(a.slab, p.dx.splits, b);
      else
        split_epilogue_kernel<f16_t><<<g, 256, 0, s>>>(a.slab, p.dx.splits, b);
      BNPVI_LAUNCH_CHECK();
    }
  }
  if (dw) {
    GemmArgs a = {};
    a.R = dz;
    a.ldr = lddz;
    a.S = xs;
    a.lds = ldxs;
    a.rows = n;
    a.cols = K;
    a.K = M;
    if (G > 0) {
      a.map = (const int4*)(wk + p.dw_map);
      a.used = (const int32_t*)(wk + p.dw_count);
      a.entries = (int)p.dw.entries;
    }
    a.C = dw;
    a.ldc = K;
    a.c_group = n * K;
    if (p.dw.slab) a.slab = (float*)(wk + p.slab);
    if (p.db_in_dw) {
      a.db = db;
      if (p.dw.slab) a.db_slab = (float*)(wk + p.db_slab);
    }
    r = run_gemm(kDw, dtype, p.dw, p.dw_direct, p.pair, a, ctx, s);
    if (r) return r;
    if (p.dw.slab) {
      const int4* sums = (const int4*)(wk + p.dw_sums);
      const int32_t* count = (const int32_t*)(wk + p.dw_count);
      const SumArgs b = {{a.slab, a.db_slab}, {dw, db}, {n * K, p.db_in_dw ? n : 0}};
      if (dtype == BNPVI_F32)
        launch_sums<float>(b, p.dw, G > 0, sums, count, s);
      else if (dtype == BNPVI_BF16)
        launch_sums<bf16_t>(b, p.dw, G > 0, sums, count, s);
      else
        launch_sums<f16_t>(b, p.dw, G > 0, sums, count, s);
      BNPVI_LAUNCH_CHECK();
    }
  }
  return BNPVI_OK;
}

int bnpvi_dense_backward(bnpvi_ctx* ctx, int dtype, const void* dy, int64_t lddy, const void* dact, int64_t lddact, const void* x,
                         int64_t ldx, const void* w, int64_t ldw, int64_t w_group, const int32_t* offsets, int G, int64_t M, int64_t K,
                         int64_t n, void* dx, int64_t lddx, void* dw, void* db, void* dres, int64_t lddres, void* work,
                         int64_t work_bytes, void* stream) {
  return bnpvi_dense_backward_act(ctx, dtype, -1, dy, lddy, dact, lddact, x, ldx, w, ldw, w_group, offsets, G, M, K, n, dx, lddx, dw, db, dres,
                                  lddres, work, work_bytes, stream);
}

}  // extern "C"
