// Dense product y = r + act(x W^T + b), its gradients, and the same per leaf on rows sorted by leaf.
//
// One matrix kernel C[row][col] = sum_k R(row, k) S(col, k) serves three products:
//     forward   rows of x,  columns = rows of W,   sum over the input width     R, S contiguous along k
//     dx        rows of dz, columns of W,          sum over the output width    R along k, S along its columns
//     dW        columns of dz, columns of x,       sum over the frames          R, S along their columns
// An operand that is contiguous along k ("KM") lies in LDS as [row][128 bytes of k], one contiguous along its
// rows / columns ("MM") as [k][row].  Either way a stage of a B-row operand is 128 B bytes in pieces of 16, which
// reach the LDS without passing through registers (buffer loads to LDS; a piece outside the matrix takes an offset
// behind the descriptor's range and arrives as zeros).  The loader cannot pad, so conflicts are avoided by permuting
// the pieces it fetches: KM piece c of row r sits at c ^ (r & 7); 16-bit MM 32-byte unit u of row k at u ^ (k mod
// units).  Fragments: KM one 16-byte LDS read; 16-bit MM two transposing 8-byte reads; fp32 MM four 4-byte reads.
// Operands whose rows do not start on 16 bytes take the same way through registers in narrower pieces.
//
// Products: v_mfma_f32_32x32x16 (bf16, f16) and v_mfma_f32_32x32x2_f32, fp32 accumulation.  S is the first operand of
// the instruction, so a lane ends with four consecutive columns of one row, and after an exchange between lanes with
// eight: the epilogue reads and writes 16-byte pieces of rows without another pass through LDS.
#pragma once

#include "layers_common.h"

namespace bnpvi {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8v __attribute__((ext_vector_type(8)));
typedef __fp16 f16x4s __attribute__((ext_vector_type(4)));

// The derivative of the activation is kept for the backward pass in a type that does not add to the error of the
// 16-bit gradients: fp16 (half a step 2^-12, 2^-25 absolute below 2^-14) beside bf16's 2^-9, fp32 beside fp16 and fp32.
template <typename T>
struct Deriv {
  typedef float type;
};
template <>
struct Deriv<bf16_t> {
  typedef f16_t type;
};

enum { kFwd = 0, kDx = 1, kDw = 2 };
enum { kTile128 = 0, kTile64 = 1, kTileFlat = 2, kTileTall = 3, kTile256 = 4 };      // 128x128, 64x64, 32x128, 128x32, 256x256

struct GemmArgs {
  const void* R;
  const void* S;
  int64_t ldr, lds;            // pitches in elements
  int64_t rows, cols, K;       // rows of C (all groups), columns, reduce extent (kDw with groups: all frames)
  int64_t s_group, c_group;    // elements between the groups' S (kFwd, kDx) or C (kDw)
  const int32_t* offsets;      // groups' bounds (kDw) or nullptr
  const int4* map;             // row tiles {group, first row, end row} (kFwd, kDx with groups) or nullptr
  int G, splits;
  int64_t row_tiles;
  int col_tiles;
  int rv, sv;                  // elements per access of R and S where a row does not start on 16 bytes
  int cvec;                    // C, residual and derivative take 16-byte accesses
  void* C;
  int64_t ldc;
  const void* bias;
  int64_t bias_group;
  const void* res;
  int64_t ldres;
  void* dact;
  int64_t lddact;
  int act;
  float* slab;                 // [group x split][rows][cols] partial sums, or nullptr
};

// act(z) and act'(z).  16-bit results (FAST) take the hardware's exp2 and reciprocal (1 ulp each) and the normal
// distribution function from formula 7.1.26 of Abramowitz and Stegun (|error| of erf below 1.5e-7), whose
// exp(-z^2 / 2) the derivative of gelu needs anyway: 2^-11 of the largest error a rounding makes.  The accurate
// functions took as long as the product itself (gelu, 33.5M values: 90 of 195 us).
template <bool FAST>
__device__ __forceinline__ float exp_of(float v) {
  return FAST ? __builtin_amdgcn_exp2f(v * 1.4426950408889634f) : expf(v);
}
template <bool FAST>
__device__ __forceinline__ float inverse(float v) {
  return FAST ? __builtin_amdgcn_rcpf(v) : 1.f / v;
}

// v: z -> act(z), d: act'(z)
template <bool FAST, int E>
__device__ __forceinline__ void activate(int act, float (&v)[E], float (&d)[E]) {
  const float inf = __builtin_inff();
  if (act == BNPVI_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < E; ++i) d[i] = 1.f;
  } else if (act == BNPVI_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      d[i] = v[i] > 0.f ? 1.f : 0.f;
      v[i] = v[i] < 0.f ? 0.f : v[i];
    }
  } else if (act == BNPVI_ACT_SOFTSIGN) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float z = v[i], q = inverse<FAST>(1.f + fabsf(z));
      v[i] = fabsf(z) < inf ? z * q : (z != z ? z : copysignf(1.f, z));
      d[i] = q * q;
    }
  } else if (act == BNPVI_ACT_TANH) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      // with e = exp(-2 |z|): tanh = (1 - e) / (1 + e), 1 - tanh^2 = 4 e / (1 + e)^2 without cancellation near 1
      const float z = v[i], e = exp_of<FAST>(-2.f * fabsf(z)), q = inverse<FAST>(1.f + e);
      v[i] = FAST ? (fabsf(z) < 0.02f ? z * (1.f - z * z * (1.f / 3.f)) : copysignf((1.f - e) * q, z)) : tanhf(z);
      d[i] = 4.f * e * q * q;
    }
  } else if (act == BNPVI_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float z = v[i], e = exp_of<FAST>(-fabsf(z)), q = inverse<FAST>(1.f + e);     // never overflows
      const float s = z >= 0.f ? q : e * q;
      v[i] = z == -inf ? 0.f : z * s;
      d[i] = fabsf(z) < inf ? s * (1.f + z * (1.f - s)) : s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float z = v[i], e = exp_of<FAST>(-0.5f * z * z);
      float c;
      if (FAST) {
        const float t = inverse<true>(1.f + 0.3275911f * 0.70710678f * fabsf(z));
        const float p = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
        const float h = 0.5f * p * e;                                          // of the tail beyond |z|
        c = z >= 0.f ? 1.f - h : (z != z ? z : h);
      } else {
        c = 0.5f * erfcf(-0.70710678118654752f * z);
      }
      v[i] = z == -inf ? 0.f : z * c;
      d[i] = fabsf(z) < inf ? c + z * (0.39894228040143268f * e) : c;
    }
  }
}

// ---- loaders -------------------------------------------------------------------------------------------------------
constexpr uint32_t kOutside = 0x90000000u;           // behind every descriptor's range: reads as zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x80000000u, 0x00027000);
}
__device__ __forceinline__ void buffer_to_lds(__amdgpu_buffer_rsrc_t r, char* l, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)l, 16, off, 0, 0, 0);
}

// Where the 16-byte pieces of one operand stage come from.  B rows (KM) or columns (MM), P pieces a lane.
template <typename T, bool KM, int B, int THREADS>
struct Source {
  static constexpr int kP = B * 8 / THREADS;
  static constexpr int kPer = 16 / (int)sizeof(T);                 // elements of a piece
  static constexpr int kBK = 128 / (int)sizeof(T);                 // k's of a stage
  static constexpr int kRow = KM ? 8 : B * (int)sizeof(T) / 16;    // pieces of an LDS row
  static constexpr int kUnits = B / 16;                            // 32-byte units of a 16-bit MM row
  static_assert(B * 8 % THREADS == 0, "whole pieces per lane");

  const char* base;      // first element of the tile's rows (KM) / columns (MM) at k = 0
  int64_t pitch;         // bytes
  int n, k;              // rows / columns left in the matrix, k's of this workgroup
  int row[kP], piece[kP];

  __device__ __forceinline__ void init(const void* p, int64_t ld, int left, int kext) {
    base = reinterpret_cast<const char*>(p);
    pitch = ld * (int64_t)sizeof(T);
    n = left;
    k = kext;
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      const int i = q * THREADS + threadIdx.x;
      const int r = i / kRow, c = i % kRow;
      row[q] = r;
      if (KM)
        piece[q] = c ^ (r & 7);
      else if (sizeof(T) == 2)
        piece[q] = (((c >> 1) ^ (r & (kUnits - 1))) << 1) | (c & 1);
      else
        piece[q] = c;
    }
  }
  // every piece of stage kt straight into LDS (wave-uniform base + 16 bytes a lane)
  __device__ __forceinline__ void to_lds(int kt, char* lds) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const char* at = base + (KM ? (int64_t)kt * 128 : (int64_t)kt * kBK * pitch);
    const __amdgpu_buffer_rsrc_t rs = rsrc_of(at);
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      const int kk = kt * kBK + (KM ? piece[q] * kPer : row[q]);
      const int nn = KM ? row[q] : piece[q] * kPer;
      const uint32_t off = (uint32_t)row[q] * (uint32_t)pitch + (uint32_t)piece[q] * 16u;
      buffer_to_lds(rs, lds + (q * THREADS + wave * 64) * 16, kk < k && nn < n ? off : kOutside);
    }
  }
  // the same through registers, V elements an access (V divides the pitch, the base and the contiguous extent)
  template <int V>
  __device__ __forceinline__ void fetch(int kt, u32x4 (&reg)[kP]) const {
    typedef T vec __attribute__((ext_vector_type(V)));
    union {
      u32x4 u;
      vec v[kPer / V];
    } x;
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      x.u = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < kPer / V; ++e) {
        const int kk = kt * kBK + (KM ? piece[q] * kPer + e * V : row[q]);
        const int nn = KM ? row[q] : piece[q] * kPer + e * V;
        if (kk < k && nn < n) {
          const int64_t r = KM ? row[q] : kk, c = KM ? kk : nn;
          x.v[e] = *reinterpret_cast<const vec*>(base + r * pitch + c * (int64_t)sizeof(T));
        }
      }
      reg[q] = x.u;
    }
  }
  __device__ __forceinline__ void fetch_any(int v, int kt, u32x4 (&reg)[kP]) const {
    if (v >= kPer)
      fetch<kPer>(kt, reg);
    else if (v >= kPer / 2)
      fetch<kPer / 2>(kt, reg);
    else if (v >= 2)
      fetch<2>(kt, reg);
    else
      fetch<1>(kt, reg);
  }
  __device__ __forceinline__ void put(char* lds, const u32x4 (&reg)[kP]) const {
#pragma unroll
    for (int q = 0; q < kP; ++q) *reinterpret_cast<u32x4*>(lds + (q * THREADS + (int)threadIdx.x) * 16) = reg[q];
  }
};

// ---- fragments of one k-step of 16-bit operands (16 k's) or fp32 operands (8 k's) ------------------------------------
template <typename T>
struct Frag;
template <>
struct Frag<float> {
  typedef f32x4 type;
  static __device__ __forceinline__ void mma(const f32x4& a, const f32x4& b, f32x16& c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
  }
};
template <>
struct Frag<bf16_t> {
  typedef bf16x8 type;
  static __device__ __forceinline__ void mma(const bf16x8& a, const bf16x8& b, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ bf16x8 transposed(const char* p0, const char* p1) {
    typedef __attribute__((address_space(3))) bf16x4* at;
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((at)(p0)), b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((at)(p1));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};
template <>
struct Frag<f16_t> {
  typedef f16x8v type;
  static __device__ __forceinline__ void mma(const f16x8v& a, const f16x8v& b, f32x16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f16x8v transposed(const char* p0, const char* p1) {
    typedef __attribute__((address_space(3))) f16x4s* at;
    union {
      f16x4s h[2];
      f16x8v v;
    } x;
    x.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4f16((at)(p0));
    x.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4f16((at)(p1));
    return x.v;
  }
};

// Fragment `f` (32 rows) of an operand stage for k-step s: lane (i = lane % 32, h = lane / 32) gets row 32 f + i, and
// k = (2 s + h) kPer + 0 .. kPer - 1 -- the same k's for both kinds of operand, which is all a product needs.
template <typename T, bool KM, int B>
struct Reader {
  int off[4];      // KM: byte offset of each k-step's piece; 16-bit MM: of each pair (first / second four k's)
  int lane;
  __device__ __forceinline__ void init(int row0) {
    lane = threadIdx.x & 63;
    const int i = lane & 31, h = lane >> 5;
    if (KM) {
#pragma unroll
      for (int s = 0; s < 4; ++s) off[s] = (row0 + i) * 128 + (((2 * s + h) ^ (i & 7)) << 4);
    } else if (sizeof(T) == 2) {
      off[0] = (h * 8 + ((lane & 15) >> 2)) * (B * 2) + (lane & 3) * 8;     // the unit is added per fragment
      off[1] = row0 / 16 + ((lane >> 4) & 1);
    } else {
      off[0] = h * 4 * (B * 4) + (row0 + i) * 4;
    }
  }
  __device__ __forceinline__ typename Frag<T>::type get(const char* lds, int f, int s) const {
    if constexpr (KM) {
      return *reinterpret_cast<const typename Frag<T>::type*>(lds + off[s] + f * 32 * 128);
    } else if constexpr (sizeof(T) == 2) {
      constexpr int U = B / 16;
      const int kk = (lane & 15) >> 2, u = off[1] + 2 * f;
      // k & (U - 1): s * 16 + h * 8 are multiples of 8 and U <= 8, or U = 16 where h * 8 counts too
      const int k0 = (s * 16 + (lane >> 5) * 8 + kk) & (U - 1), k1 = (s * 16 + (lane >> 5) * 8 + kk + 4) & (U - 1);
      const char* p = lds + off[0] + s * 16 * (B * 2);
      return Frag<T>::transposed(p + ((u ^ k0) << 5), p + 4 * (B * 2) + ((u ^ k1) << 5));
    } else {
      f32x4 v;
#pragma unroll
      for (int t = 0; t < 4; ++t) v[t] = *reinterpret_cast<const float*>(lds + off[0] + (8 * s + t) * (B * 4) + f * 128);
      return v;
    }
  }
};

// ---- the kernel ----------------------------------------------------------------------------------------------------
// Workgroup tile BR x BC, wave tile WR x WC.  Two LDS stages: while one is multiplied the other is filled; one barrier
// a stage.
template <int BR, int BC>
constexpr int gemm_lds_bytes() {
  return 2 * (BR + BC) * 128;
}

template <typename T, int KIND, int BR, int BC, int WR, int WC, bool DIRECT>
__global__ __launch_bounds__((BR / WR) * (BC / WC) * 64) void gemm_kernel(const GemmArgs a) {
  constexpr int THREADS = (BR / WR) * (BC / WC) * 64;
  constexpr bool RKM = KIND != kDw, SKM = KIND == kFwd;
  constexpr int FR = WR / 32, FC = WC / 32, BK = 128 / (int)sizeof(T);
  extern __shared__ __attribute__((aligned(16))) char lds[];

  // Workgroups go to the eight XCDs in turn; each XCD gets a contiguous run of tiles, columns first, so that the tiles
  // that share rows of R share an L2.
  const int64_t total = (int64_t)gridDim.x;
  const int64_t x = blockIdx.x & 7, q8 = total >> 3, rem = total & 7;
  const int64_t lin = x * q8 + (x < rem ? x : rem) + (blockIdx.x >> 3);
  const int ct = (int)(lin % a.col_tiles);
  const int64_t rt = (lin / a.col_tiles) % a.row_tiles;
  const int z = (int)(lin / a.col_tiles / a.row_tiles);
  const int split = z % a.splits;
  int g = z / a.splits;

  int64_t row0 = rt * BR, row_end = a.rows;
  const int64_t col0 = (int64_t)ct * BC;
  int64_t k_lo = 0, k_hi = a.K;
  if (KIND == kDw) {
    if (a.offsets != nullptr) {
      const int64_t M = a.K;
      int64_t lo = a.offsets[g], hi = a.offsets[g + 1];
      k_lo = lo < 0 ? 0 : lo > M ? M : lo;
      k_hi = hi < k_lo ? k_lo : hi > M ? M : hi;
    }
  } else if (a.map != nullptr) {
    const int4 m = a.map[rt];
    g = m.x;
    row0 = m.y;
    row_end = m.z;
    if (row0 >= row_end) return;
  }
  if (a.splits > 1) {
    const int64_t per = ((k_hi - k_lo + a.splits - 1) / a.splits + BK - 1) / BK * BK;
    k_lo = k_lo + split * per < k_hi ? k_lo + split * per : k_hi;
    k_hi = k_lo + per < k_hi ? k_lo + per : k_hi;
  }
  const int nr = (int)(row_end - row0 < BR ? row_end - row0 : BR);
  const int nc = (int)(a.cols - col0 < BC ? a.cols - col0 : BC);
  const int kext = g < 0 ? 0 : (int)(k_hi - k_lo);           // a tile of rows without a leaf has nothing to add up
  const int gs = g < 0 ? 0 : g;

  const T* Rp = reinterpret_cast<const T*>(a.R) + (RKM ? row0 * a.ldr + k_lo : k_lo * a.ldr + row0);
  const T* Sp = reinterpret_cast<const T*>(a.S) + (KIND == kDw ? 0 : gs * a.s_group) +
                (SKM ? col0 * a.lds + k_lo : k_lo * a.lds + col0);
  Source<T, RKM, BR, THREADS> sr;
  Source<T, SKM, BC, THREADS> ss;
  sr.init(Rp, a.ldr, nr, kext);
  ss.init(Sp, a.lds, nc, kext);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / (BC / WC) * WR, wc = wave % (BC / WC) * WC;
  Reader<T, RKM, BR> rr;
  Reader<T, SKM, BC> rs;
  rr.init(wr);
  rs.init(wc);

  f32x16 acc[FR][FC];
#pragma unroll
  for (int i = 0; i < FR; ++i)
#pragma unroll
    for (int j = 0; j < FC; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  constexpr int STAGE = (BR + BC) * 128;
  const int nk = (kext + BK - 1) / BK;
  auto multiply = [&](const char* stage) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      typename Frag<T>::type fr[FR], fc[FC];
#pragma unroll
      for (int i = 0; i < FR; ++i) fr[i] = rr.get(stage, i, s);
#pragma unroll
      for (int j = 0; j < FC; ++j) fc[j] = rs.get(stage + BR * 128, j, s);
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j) Frag<T>::mma(fc[j], fr[i], acc[i][j]);
    }
  };
  if constexpr (DIRECT) {
    if (nk > 0) {
      sr.to_lds(0, lds);
      ss.to_lds(0, lds + BR * 128);
    }
    for (int kt = 0; kt < nk; ++kt) {
      // this stage has arrived, and every wave is done reading the other one (its stage kt - 1)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (kt + 1 < nk) {
        char* next = lds + ((kt + 1) & 1) * STAGE;
        sr.to_lds(kt + 1, next);
        ss.to_lds(kt + 1, next + BR * 128);
      }
      multiply(lds + (kt & 1) * STAGE);
    }
  } else {
    u32x4 hr[decltype(sr)::kP], hs[decltype(ss)::kP];
    if (nk > 0) {
      sr.fetch_any(a.rv, 0, hr);
      ss.fetch_any(a.sv, 0, hs);
    }
    for (int kt = 0; kt < nk; ++kt) {
      char* stage = lds + (kt & 1) * STAGE;
      sr.put(stage, hr);
      ss.put(stage + BR * 128, hs);
      __syncthreads();                       // the stage written two turns ago is free: its readers passed this barrier
      if (kt + 1 < nk) {
        sr.fetch_any(a.rv, kt + 1, hr);
        ss.fetch_any(a.sv, kt + 1, hs);
      }
      multiply(stage);
    }
  }

  // ---- epilogue.  A lane has four consecutive columns (4 h + 0 .. 3 of every eight) of one row; exchanging the upper
  // half of one four with the lower half of the next between lanes 32 apart makes them eight consecutive ones.
  const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
  for (int j = 0; j < FC; ++j) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int cl = wc + 32 * j + 16 * p + 8 * h;
      const int64_t col = col0 + cl;
      const int left = nc - cl < 8 ? nc - cl : 8;
      const bool vec = a.cvec && left == 8;
      float b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = 0.f;
      if (KIND == kFwd && a.bias != nullptr && a.slab == nullptr && g >= 0) {
        const T* bp = reinterpret_cast<const T*>(a.bias) + g * a.bias_group + col;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) b[e] = (float)bp[e];
      }
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        float v[8];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][j][8 * p + t]), __float_as_uint(acc[i][j][8 * p + 4 + t]),
                                                          false, false);
          v[t] = __uint_as_float(x[0]);
          v[t + 4] = __uint_as_float(x[1]);
        }
        const int rl = wr + 32 * i + (lane & 31);
        if (rl >= nr || left <= 0) continue;
        const int64_t row = row0 + rl;
        if (a.slab != nullptr) {
          float* out = a.slab + ((int64_t)z * a.rows + row) * a.cols + col;
          if (left == 8 && a.cols % 4 == 0) {
            *reinterpret_cast<f32x4*>(out) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4*>(out + 4) = f32x4{v[4], v[5], v[6], v[7]};
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e < left) out[e] = v[e];
          }
          continue;
        }
        T* out = reinterpret_cast<T*>(a.C) + (KIND == kDw ? g * a.c_group : 0) + row * a.ldc + col;
        if (KIND == kFwd) {
          typedef typename Deriv<T>::type DT;
          constexpr bool FAST = sizeof(T) == 2;
          float d[8], r[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = d[e] = 0.f;
          if (g >= 0) {
            if (a.res != nullptr) {
              const T* rp = reinterpret_cast<const T*>(a.res) + row * a.ldres + col;
              if (vec) {
                load_vec<T, 8>(rp, r);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (e < left) r[e] = (float)rp[e];
              }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += b[e];
            activate<FAST, 8>(a.act, v, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
          }
          if (a.dact != nullptr) {
            DT* dp = reinterpret_cast<DT*>(a.dact) + row * a.lddact + col;
            if (vec) {
              store_vec<DT, 8>(dp, d);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (e < left) dp[e] = (DT)d[e];
            }
          }
        }
        if (vec) {
          store_vec<T, 8>(out, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < left) out[e] = (T)v[e];
        }
      }
    }
  }
}

int launch_gemm_f32(int kind, int tile, bool direct, const GemmArgs& a, int device, hipStream_t s);
int launch_gemm_bf16(int kind, int tile, bool direct, const GemmArgs& a, int device, hipStream_t s);
int launch_gemm_f16(int kind, int tile, bool direct, const GemmArgs& a, int device, hipStream_t s);

}  // namespace bnpvi
