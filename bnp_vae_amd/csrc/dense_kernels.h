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
// Operands whose rows do not start on 16 bytes come through registers into the same places.
//
// Products: v_mfma_f32_32x32x16 (bf16, f16) and v_mfma_f32_32x32x2_f32, fp32 accumulation.  S is the first operand of
// the instruction, so a lane ends with four consecutive columns of one row; the accumulators pass through LDS once
// more so that the epilogue reads and writes whole 16-byte pieces of rows, eight lanes and more a row.
//
// What bounds it.  A wave tile of 128 x 64 needs 6 KB of fragments for 8 instructions: of the LDS's 128 bytes a cycle the
// fragments take three quarters and the arriving stages the rest, so that matrix pipe and LDS are full at the same time,
// and 8192^3 in bf16 runs at 1190 / 1050 / 1100 TFLOP/s (forward, dx, dW; the library's forward 1640, on another card 1430).  Where
// the sum is short the epilogue counts: dx of 65536 x 256 -> 4096 takes 200 us, 95 of them its 537 MB of stores alone, 60
// the products, and a tile's stores and the next one's products share the time only as far as its loads reach ahead.
// 65536 x 4096 -> 256 forward reads 537 MB in 150 us (3.6 TB/s, a copy 4.7).  fp32 is bound by its matrix rate: 135 of 157
// TFLOP/s at K = 2048, and by stores where K is short (16384 x 64 -> 4096: 61 us of products, 68 of stores).
// Tried without gain: four waves of 128 x 128 (8192^3 1100 TFLOP/s; dx spills), stages of 64 bytes, a fourth stage in the
// ring, loads spread over the steps of a stage (dx 1035 -> 1125 us), the epilogue unrolled (it spills: 160 -> 300 us) or
// from registers (32 bytes a row and store: dx 200 -> 280 us), 128 x 256 tiles two a CU, co-resident workgroups out of phase.
#pragma once

#include <type_traits>

#include "layers_common.h"

namespace bnpvi {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8v __attribute__((ext_vector_type(8)));
typedef __fp16 f16x4s __attribute__((ext_vector_type(4)));

enum { kFwd = 0, kDx = 1, kDw = 2 };
enum { kTile128 = 0, kTile64 = 1, kTileFlat = 2, kTileTall = 3, kTile256 = 4 };      // 128x128, 64x64, 32x128, 128x32, 256x256

struct GemmArgs {
  const void* R;
  const void* S;
  int64_t ldr, lds;            // pitches in elements
  int64_t rows, cols, K;       // rows of C (all groups), columns, reduce extent (kDw with groups: unused)
  int64_t s_group, c_group;    // elements between the groups' S (kFwd, kDx) or C (kDw)
  const int4* map;             // with groups -- kFwd, kDx: row tiles {group, first row, end row}; kDw: pieces of the sum
                               // {group, first frame, end frame, part or -1}
  const int32_t* used;         // kDw with groups: entries of the map in use
  int entries;                 // at most
  int splits;
  int row_tiles, col_tiles;
  void* C;
  int64_t ldc;
  const void* bias;
  int64_t bias_group;
  const void* res;
  int64_t ldres;
  float* dact;                 // act'(z) in 32 bits beside every type: its far ends (softsign' 1e-8 at 1e4) pass fp16's range
  int64_t lddact;
  int act;
  float* slab;                 // [group x split][rows][cols] partial sums, or nullptr
  void* db;                    // kDw: [group][rows] sums of R over k, or nullptr
  float* db_slab;              // the same per group x split (with `slab`)
};

// act(z) and act'(z).  16-bit results (FAST) take the hardware's exp2 and reciprocal (1 ulp each) and the tail of the
// normal distribution function as exp(-z^2 / 2), which the derivative of gelu needs anyway, times a polynomial of degree 8 in
// t = 1 / (1 + 0.3182 |z|), fitted to it by weighted least squares: off by at most 2^-20 of itself however far out, so that
// a result of 1e-30 is as good as one of 1 (a polynomial made for absolute errors was off by 0.05 % at -4 and 1 % at -8).
// The accurate functions took as long as the product itself (gelu, 33.5M values: 90 of 195 us).
template <bool FAST>
__device__ __forceinline__ float exp_of(float v) {
  return FAST ? __builtin_amdgcn_exp2f(v * 1.4426950408889634f) : expf(v);
}
template <bool FAST>
__device__ __forceinline__ float inverse(float v) {
  return FAST ? __builtin_amdgcn_rcpf(v) : 1.f / v;
}

// v: z -> act(z), d: act'(z).  Limits at infinities come from clamped factors, not branches; NaN passes through.
__device__ __forceinline__ float clamped(float v, float at) { return __builtin_amdgcn_fmed3f(v, -at, at); }

template <bool FAST, int E>
__device__ __forceinline__ void activate(int act, float (&v)[E], float (&d)[E]) {
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
      const float z = v[i], m = fminf(fabsf(z), 1e30f), q = inverse<FAST>(1.f + m);
      v[i] = z != z ? z : copysignf(m * q, z);
      d[i] = z != z ? z : q * q;
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
      const float z = v[i], s = inverse<FAST>(1.f + exp_of<FAST>(-z));         // exp may be infinite: s = 0
      v[i] = s * fmaxf(z, -3e38f);
      d[i] = s * (1.f + clamped(z, 1e4f) * (1.f - s));
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float z = v[i], e = exp_of<FAST>(-0.5f * z * z);
      float c;
      if (FAST) {
        const float t = inverse<true>(1.f + 0.31819806f * fabsf(z));
        const float q = 0.19709866f + t * (0.025063414f + t * (0.22445743f + t * (-0.24875407f + t * 0.068758845f)));
        const float p = t * (0.25388074f + t * (0.25406945f + t * (0.22542551f + t * q)));
        const float h = 0.5f * p * e;                                          // of the tail beyond |z|
        c = z < 0.f ? h : 1.f - h;
      } else {
        c = 0.5f * erfcf(-0.70710678118654752f * z);
      }
      v[i] = c * fmaxf(z, -3e38f);
      d[i] = c + clamped(z, 1e4f) * (0.39894228040143268f * e);
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

// piece c of KM row r sits at c ^ swizzle(r): eight consecutive rows, read at the same k, fall on different 16 bytes of
// the 128 that one cycle of the LDS serves
template <int KB>
__device__ __forceinline__ int swizzle(int r) {
  static_assert(KB == 128, "eight pieces a row");
  return r & 7;
}

// Where the 16-byte pieces of one operand stage (KB bytes of k) come from.  B rows (KM) or columns (MM), P pieces a lane.
template <typename T, bool KM, int B, int THREADS, int KB>
struct Source {
  static constexpr int kP = B * (KB / 16) / THREADS;
  static constexpr int kPer = 16 / (int)sizeof(T);                 // elements of a piece
  static constexpr int kBK = KB / (int)sizeof(T);                  // k's of a stage
  static constexpr int kRow = KM ? KB / 16 : B * (int)sizeof(T) / 16;    // pieces of an LDS row
  static constexpr int kUnits = B / 16;                            // 32-byte units of a 16-bit MM row
  static_assert(kP > 0 && B * (KB / 16) % THREADS == 0, "whole pieces per lane");

  const char* base;      // first element of the tile's rows (KM) / columns (MM) at k = 0
  int64_t pitch;         // bytes
  int n, k;              // rows / columns left in the matrix, k's of this tile
  uint32_t off[kP];      // of a lane's pieces from the stage's first byte; kOutside behind the last row / column

  static __device__ __forceinline__ int row(int q) { return (q * THREADS + (int)threadIdx.x) / kRow; }
  static __device__ __forceinline__ int piece(int q) {
    const int r = row(q), c = (q * THREADS + (int)threadIdx.x) % kRow;
    if constexpr (KM) return c ^ swizzle<KB>(r);
    if (sizeof(T) == 2) return (((c >> 1) ^ (r & (kUnits - 1))) << 1) | (c & 1);
    return c;
  }
  __device__ __forceinline__ void init(const void* p, int64_t ld, int left, int kext) {
    base = reinterpret_cast<const char*>(p);
    pitch = ld * (int64_t)sizeof(T);
    n = left;
    k = kext;
#pragma unroll
    for (int q = 0; q < kP; ++q)
      off[q] = (KM ? row(q) : piece(q) * kPer) < n ? (uint32_t)row(q) * (uint32_t)pitch + (uint32_t)piece(q) * 16u : kOutside;
  }
  // every piece of stage kt straight into LDS (wave-uniform base + 16 bytes a lane)
  __device__ __forceinline__ void to_lds(int kt, char* lds) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const __amdgpu_buffer_rsrc_t rs = rsrc_of(base + (KM ? (int64_t)kt * KB : (int64_t)kt * kBK * pitch));
    if (kt * kBK + kBK <= k) {
#pragma unroll
      for (int q = 0; q < kP; ++q) buffer_to_lds(rs, lds + (q * THREADS + wave * 64) * 16, off[q]);
    } else {
#pragma unroll
      for (int q = 0; q < kP; ++q)
        buffer_to_lds(rs, lds + (q * THREADS + wave * 64) * 16, kt * kBK + (KM ? piece(q) * kPer : row(q)) < k ? off[q] : kOutside);
    }
  }
  // The same through registers, for rows that start anywhere: global loads take any address.  A piece that crosses the
  // end of its row (KM) or of the columns (MM) is put together element by element.
  __device__ __forceinline__ void fetch(int kt, u32x4 (&reg)[kP]) const {
#pragma unroll
    for (int q = 0; q < kP; ++q) {
      const int kk = kt * kBK + (KM ? piece(q) * kPer : row(q)), nn = KM ? row(q) : piece(q) * kPer;
      const int inside = nn < n && kk < k ? (KM ? k - kk : n - nn) : 0;           // elements of this piece
      const char* at = base + (KM ? (int64_t)nn * pitch + (int64_t)kk * sizeof(T) : (int64_t)kk * pitch + (int64_t)nn * sizeof(T));
      reg[q] = u32x4{0, 0, 0, 0};
      if (inside >= kPer) {
        const u32x4_anywhere v = *reinterpret_cast<const u32x4_anywhere*>(at);
        reg[q] = u32x4{v[0], v[1], v[2], v[3]};
      } else if (inside > 0) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t v = 0;
          if (sizeof(T) == 4) {
            if (w < inside) v = reinterpret_cast<const uint32_t*>(at)[w];
          } else {
            if (2 * w < inside) v = reinterpret_cast<const uint16_t*>(at)[2 * w];
            if (2 * w + 1 < inside) v |= (uint32_t)reinterpret_cast<const uint16_t*>(at)[2 * w + 1] << 16;
          }
          reg[q][w] = v;
        }
      }
    }
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
  static constexpr int kSteps = 4;
  static __device__ __forceinline__ void mma(const f32x4& a, const f32x4& b, f32x16& c, int t) {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum(const f32x4& a, float c) { return c + ((a[0] + a[1]) + (a[2] + a[3])); }
};
template <>
struct Frag<bf16_t> {
  typedef bf16x8 type;
  static constexpr int kSteps = 1;
  static __device__ __forceinline__ void mma(const bf16x8& a, const bf16x8& b, f32x16& c, int) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum(const bf16x8& a, float c) {
    typedef bf16_t two __attribute__((ext_vector_type(2)));
    const two one = {(bf16_t)1.f, (bf16_t)1.f};
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_fdot2_f32_bf16(two{a[2 * t], a[2 * t + 1]}, one, c, false);
    return c;
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
  static constexpr int kSteps = 1;
  static __device__ __forceinline__ void mma(const f16x8v& a, const f16x8v& b, f32x16& c, int) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum(const f16x8v& a, float c) {
    typedef f16_t two __attribute__((ext_vector_type(2)));
    const two one = {(f16_t)1.f, (f16_t)1.f};
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_fdot2(two{a[2 * t], a[2 * t + 1]}, one, c, false);
    return c;
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
template <typename T, bool KM, int B, int KB>
struct Reader {
  int off[4];      // KM: byte offset of each k-step's piece; 16-bit MM: of each pair (first / second four k's)
  int lane;
  int at;          // 16-bit MM: of the first pair of fragment 0 at k-step 0; the others differ in bits of the unit and in rows
  __device__ __forceinline__ void init(int row0) {
    lane = threadIdx.x & 63;
    const int i = lane & 31, h = lane >> 5;
    if constexpr (KM) {
#pragma unroll
      for (int s = 0; s < KB / 32; ++s) off[s] = (row0 + i) * KB + (((2 * s + h) ^ swizzle<KB>(i)) << 4);
    } else if (sizeof(T) == 2) {
      off[0] = (h * 8 + ((lane & 15) >> 2)) * (B * 2) + (lane & 3) * 8;     // the unit is added per fragment
      off[1] = row0 / 16 + ((lane >> 4) & 1);
      at = off[0] + ((off[1] ^ ((h * 8 + ((lane & 15) >> 2)) & (B / 16 - 1))) << 5);
    } else {
      off[0] = h * 4 * (B * 4) + (row0 + i) * 4;
    }
  }
  // The same fragment by one exclusive-or and one addition, made anew in every stage: kept in registers the addresses of all
  // fragments spill (dz in two parts, 256 x 256: 31 registers, dW of 65536 x 4096 -> 256 309 us,
  // so 300).
  __device__ __forceinline__ void anew() {
    if constexpr (!KM && sizeof(T) == 2) asm volatile("" : "+v"(at));
  }
  __device__ __forceinline__ typename Frag<T>::type get_anew(const char* lds, int f, int s) const {
    if constexpr (!KM && sizeof(T) == 2) {
      constexpr int U = B / 16, W = B * 2;
      const int u = (2 * f) ^ (16 * s & (U - 1));
      return Frag<T>::transposed(lds + ((at ^ (u << 5)) + s * 16 * W), lds + ((at ^ ((u ^ (4 & (U - 1))) << 5)) + (s * 16 + 4) * W));
    } else {
      return get(lds, f, s);
    }
  }
  __device__ __forceinline__ typename Frag<T>::type get(const char* lds, int f, int s) const {
    if constexpr (KM) {
      return *reinterpret_cast<const typename Frag<T>::type*>(lds + off[s] + f * 32 * KB);
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

// at most N vector memory operations of this wave still on their way (expcnt and lgkmcnt left alone)
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// ---- the kernel ----------------------------------------------------------------------------------------------------
// Workgroup tile BR x BC, wave tile WR x WC, stages of KB bytes of k.  The operand that comes from far (x or dz in the
// forward and dx products, x in the dW product) has a ring of three stages in LDS, the other one of two; through
// registers both have two.  One barrier a stage.
//
// PAIR: R is dz in two 16-bit parts, hi + lo, since dx and dW of one 16-bit part are 1.4 times as far from the exact ones as
// a single rounding of the results (0.0024 against 0.0017 relative in bf16).  A row of it holds 32 columns of hi, 32 of lo,
// and so on, so that a stage is as many bytes as ever, of half as many k's (dx) or of both parts of its columns (dW); S's
// stages are half as long, and each of its fragments is multiplied with both parts.  That is twice the
// instructions: 65536 x 4096 -> 256 in bf16 takes 287 / 303 us for dx / dW, from one part 203 / 175; 32768 x 1024 -> 1024 takes
// 136 / 151, from one part 84 / 92 (910 to 1010 TFLOP/s of the doubled products).
template <int KIND, bool PAIR, int BR, int BC, int KB>
struct Stages {
  static constexpr bool kRKM = KIND != kDw, kSKM = KIND == kFwd;
  static constexpr int kRRows = PAIR && !kRKM ? 2 * BR : BR, kRBytes = PAIR && !kRKM ? KB / 2 : KB;      // rows and k bytes of R's stage
  static constexpr int kSBytes = PAIR ? KB / 2 : KB;
};
template <int BR, int BC, int WR, int WC, int KB, int KIND, bool DIRECT, bool PAIR>
struct Rings {
  static constexpr int kR = DIRECT && KIND != kDw ? 3 : 2, kS = DIRECT && KIND == kDw ? 3 : 2;
  static constexpr int kRStage = BR * KB, kSStage = BC * Stages<KIND, PAIR, BR, BC, KB>::kSBytes;
  // the epilogue takes 32 rows of every wave at once: as many waves as fit in a stage of R, then of S, the others behind
  static constexpr int kEp = 32 * WC * 4, kWaves = (BR / WR) * (BC / WC);
  static constexpr int kRWaves = kRStage / kEp < kWaves ? kRStage / kEp : kWaves;
  static constexpr int kSWaves = kSStage / kEp < kWaves - kRWaves ? kSStage / kEp : kWaves - kRWaves;
  static constexpr int kBehind = kR * kRStage + kS * kSStage;
  static constexpr int kBytes = kBehind + (kWaves - kRWaves - kSWaves) * kEp;
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// the dW kernel can add up the rows of R for the bias, but not where its accumulators already fill the registers; with an
// activation in 16 bits the pass that makes dz's two parts does that
template <int KIND, int BR, bool PAIR>
constexpr bool kRowSums = KIND == kDw && BR < 256 && !PAIR;

// One output tile: its place in C, its group, its part of the sum.
struct Tile {
  int64_t row0, col0, k_lo;
  int nr, nc, kext, g, z;
  // stages of the sum; an empty one is one stage of zeros
  __device__ __forceinline__ int stages(int bk) const { return kext > bk ? (kext + bk - 1) / bk : 1; }
};

// One XCD's share of a grouped dW, a like mixture of the pieces for all eight: every eighth piece with all its tiles, which
// then share an L2, or where there are few pieces of many tiles an eighth of every piece's.
struct Share {
  uint32_t per, tile0, entry0, every;
};

template <int KIND, int BR, int BC, int BK>
__device__ __forceinline__ bool find_tile(const GemmArgs& a, uint32_t lin, const Share& sh, Tile& t) {
  // divisions are done by the vector unit: their results are told to be the same in every lane
  if (KIND == kDw && a.map != nullptr) {
    const uint32_t e = uniform(lin / sh.per), rest = sh.tile0 + lin - e * sh.per;
    const uint32_t rt = uniform(rest / (uint32_t)a.col_tiles), ct = rest - rt * (uint32_t)a.col_tiles;
    const int4 m = a.map[sh.entry0 + sh.every * e];
    t.g = m.x;
    t.z = m.w;
    t.row0 = (int64_t)rt * BR;
    t.col0 = (int64_t)ct * BC;
    t.k_lo = m.y;
    t.kext = m.z - m.y;
    t.nr = (int)(a.rows - t.row0 < BR ? a.rows - t.row0 : BR);
    t.nc = (int)(a.cols - t.col0 < BC ? a.cols - t.col0 : BC);
    return true;
  }
  const uint32_t row = uniform(lin / (uint32_t)a.col_tiles), ct = lin - row * (uint32_t)a.col_tiles;
  const uint32_t zz = uniform(row / (uint32_t)a.row_tiles), rt = row - zz * (uint32_t)a.row_tiles;
  const int split = (int)zz;
  t.z = split;
  t.g = 0;
  t.row0 = (int64_t)rt * BR;
  t.col0 = (int64_t)ct * BC;
  int64_t row_end = a.rows, k_lo = 0, k_hi = a.K;
  if (KIND != kDw && a.map != nullptr) {
    const int4 m = a.map[rt];
    t.g = m.x;
    t.row0 = m.y;
    row_end = m.z;
    if (t.row0 >= row_end) return false;
  }
  if (a.splits > 1) {
    const uint32_t each = uniform((uint32_t)(k_hi - k_lo + a.splits - 1) / (uint32_t)a.splits);      // k's: below 2^31
    const int64_t per = ((int64_t)each + BK - 1) / BK * BK;
    k_lo = k_lo + split * per < k_hi ? k_lo + split * per : k_hi;
    k_hi = k_lo + per < k_hi ? k_lo + per : k_hi;
  }
  t.nr = (int)(row_end - t.row0 < BR ? row_end - t.row0 : BR);
  t.nc = (int)(a.cols - t.col0 < BC ? a.cols - t.col0 : BC);
  t.k_lo = k_lo;
  t.kext = t.g < 0 ? 0 : (int)(k_hi - k_lo);           // a tile of rows without a leaf has nothing to add up
  return true;
}

// The stages of one operand, tile after tile of this workgroup, in the order in which they are multiplied.
template <typename T, int KIND, bool PAIR, int BR, int BC, int KB, int THREADS, bool ROWS>
struct Stream {
  typedef Stages<KIND, PAIR, BR, BC, KB> St;
  static constexpr bool kKM = ROWS ? St::kRKM : St::kSKM;
  static constexpr int kBK = St::kSBytes / (int)sizeof(T);
  typedef Source<T, kKM, ROWS ? St::kRRows : BC, THREADS, ROWS ? St::kRBytes : St::kSBytes> Src;
  Src src;
  uint32_t lin, last, inc, twice;
  Share sh;
  int kt, nk;

  __device__ __forceinline__ void begin(const GemmArgs& a, uint32_t first, uint32_t end, uint32_t ahead, uint32_t two_turns, const Share& of) {
    lin = first;
    sh = of;
    last = end;
    inc = ahead;
    twice = two_turns;
    enter(a);
  }
  __device__ __forceinline__ void enter(const GemmArgs& a) {
    Tile t;
    kt = 0;
    while (lin < last) {
      const bool found = find_tile<KIND, BR, BC, kBK>(a, lin, sh, t);
      lin += inc;
      inc = twice - inc;
      if (found) {
        const int g = t.g < 0 ? 0 : t.g;
        if (ROWS && PAIR)          // both parts of whole 32s of columns
          src.init(reinterpret_cast<const T*>(a.R) + (kKM ? t.row0 * a.ldr + 2 * t.k_lo : t.k_lo * a.ldr + 2 * t.row0), a.ldr,
                   kKM ? t.nr : 2 * ((t.nr + 31) & ~31), kKM ? 2 * ((t.kext + 31) & ~31) : t.kext);
        else if (ROWS)
          src.init(reinterpret_cast<const T*>(a.R) + (kKM ? t.row0 * a.ldr + t.k_lo : t.k_lo * a.ldr + t.row0), a.ldr, t.nr, t.kext);
        else
          src.init(reinterpret_cast<const T*>(a.S) + (KIND == kDw ? 0 : g * a.s_group) +
                       (kKM ? t.col0 * a.lds + t.k_lo : t.k_lo * a.lds + t.col0),
                   a.lds, t.nc, t.kext);
        nk = t.stages(kBK);
        return;
      }
    }
    src.k = 0;                 // behind the last tile: zeros, so that the count of loads on their way stays the same
    nk = 0x7fffffff;
  }
  __device__ __forceinline__ void step_on(const GemmArgs& a) {
    if (++kt == nk) enter(a);
  }
};

// The grid is as many workgroups as the chip holds at once; each takes tile after tile.  Workgroups go to the eight
// XCDs in turn; every XCD owns a contiguous run of tiles, columns first, which its workgroups walk side by side, so that
// the tiles that share rows of R share an L2.  The operands' stages follow each other across tiles, so the next tile
// arrives while the last stages of this one are multiplied and while its epilogue runs.
template <typename T, int KIND, int BR, int BC, int WR, int WC, int KB, bool DIRECT, bool PAIR>
__global__ __launch_bounds__((BR / WR) * (BC / WC) * 64) __attribute__((amdgpu_waves_per_eu(BR * BC >= 128 * 128 ? 2 : 4)))
void gemm_kernel(const GemmArgs a, uint32_t tiles) {
  constexpr int THREADS = (BR / WR) * (BC / WC) * 64;
  static_assert(!PAIR || (sizeof(T) == 2 && KIND != kFwd), "dz of 16 bits in two parts");
  typedef Stages<KIND, PAIR, BR, BC, KB> St;
  constexpr int FR = WR / 32, FC = WC / 32, BK = St::kSBytes / (int)sizeof(T);
  typedef Rings<BR, BC, WR, WC, KB, KIND, DIRECT, PAIR> Ring;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* const ring_s = lds + Ring::kR * Ring::kRStage;

  const uint32_t xcd = blockIdx.x & 7, q8 = tiles >> 3, rem = tiles & 7;
  const uint32_t step = (gridDim.x + 7 - xcd) >> 3;
  uint32_t first = xcd * q8 + (xcd < rem ? xcd : rem), last = first + q8 + (xcd < rem ? 1 : 0);
  Share sh = {1, 0, 0, 1};
  if (KIND == kDw && a.map != nullptr) {
    const int32_t u = *a.used;
    const uint32_t used = u < 0 ? 0 : u < a.entries ? u : a.entries, per = (uint32_t)a.row_tiles * (uint32_t)a.col_tiles;
    first = 0;
    if (per >= 64 && used < 64) {
      sh = Share{(per >> 3) + (xcd < (per & 7) ? 1 : 0), xcd * (per >> 3) + (xcd < (per & 7) ? xcd : per & 7), 0, 1};
      last = used * sh.per;
    } else {
      sh = Share{per, 0, xcd, 8};
      last = used > xcd ? (used - xcd + 7) / 8 * per : 0;
    }
  }
  // a grouped dW's tiles come longest first: odd turns go through the workgroups backwards, so that long meets short
  const uint32_t wg = blockIdx.x >> 3, twice = 2 * step;
  uint32_t lin = first + wg, inc = KIND == kDw && a.map != nullptr ? twice - 2 * wg - 1 : step;
  if (lin >= last) return;
  Stream<T, KIND, PAIR, BR, BC, KB, THREADS, true> sr;
  Stream<T, KIND, PAIR, BR, BC, KB, THREADS, false> ss;
  sr.begin(a, lin, last, inc, twice, sh);
  ss.begin(a, lin, last, inc, twice, sh);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wr = wave / (BC / WC) * WR, wc = wave % (BC / WC) * WC;
  Reader<T, St::kRKM, St::kRRows, St::kRBytes> rr;
  Reader<T, St::kSKM, BC, St::kSBytes> rs;
  rr.init(PAIR && !St::kRKM ? 2 * wr : wr);
  rs.init(wc);
  // step s of a stage: a k-step, or with two parts hi and then lo of k-step s / 2
  auto get_r = [&](const char* at, int i, int s) {
    return !PAIR ? rr.get(at, i, s) : St::kRKM ? rr.get(at, i, s / 2 + 2 * (s & 1)) : rr.get_anew(at, 2 * i + (s & 1), s / 2);
  };
  auto get_s = [&](const char* at, int j, int s) { return PAIR ? rs.get_anew(at, j, s / 2) : rs.get(at, j, s); };
  auto slot_s = [](int s) { return PAIR ? (s / 2) & 1 : s & 1; };

  u32x4 hr[DIRECT ? 1 : decltype(sr.src)::kP], hs[DIRECT ? 1 : decltype(ss.src)::kP];
  int fill_r = 0, fill_s = 0, use_r = 0, use_s = 0;          // ring positions
  auto load_r = [&] {
    if constexpr (DIRECT) {
      sr.src.to_lds(sr.kt, lds + fill_r * Ring::kRStage);
      fill_r = fill_r == Ring::kR - 1 ? 0 : fill_r + 1;
    } else {
      sr.src.fetch(sr.kt, hr);
    }
    sr.step_on(a);
  };
  auto load_s = [&] {
    if constexpr (DIRECT) {
      ss.src.to_lds(ss.kt, ring_s + fill_s * Ring::kSStage);
      fill_s = fill_s == Ring::kS - 1 ? 0 : fill_s + 1;
    } else {
      ss.src.fetch(ss.kt, hs);
    }
    ss.step_on(a);
  };
  // the operand with the longer ring is loaded last: its newest stage is what may still be on its way at a barrier
  constexpr bool DEEP_R = Ring::kR == 3, DEEP_S = Ring::kS == 3;
  constexpr int AHEAD = DEEP_R ? decltype(sr.src)::kP : DEEP_S ? decltype(ss.src)::kP : 0;
  load_r();
  load_s();
  if (DEEP_R) load_r();
  if (DEEP_S) load_s();

  // vector stores of a full tile's epilogue that a wave issues behind its loads (0: unknown, wait for all of them)
  constexpr int LPR = WC / 8, RPI = 64 / LPR, SLOTS = WC / 4;
  constexpr int Y_OPS = FR * (32 / RPI) * (int)sizeof(T) / 2;
  constexpr int D_OPS = FR * (32 / RPI) * 2;
  int behind = 0;

  Tile t;
  for (; lin < last; lin += inc, inc = twice - inc) {
    if (!find_tile<KIND, BR, BC, BK>(a, lin, sh, t)) continue;
    f32x16 acc[FR][FC];
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int j = 0; j < FC; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // the bias gradient where dz is dy: row sums of R, by the waves that hold the first columns
    const bool row_sums = kRowSums<KIND, BR, PAIR> && (a.db != nullptr || a.db_slab != nullptr) && t.col0 == 0 && wc == 0;
    float rsum[FR];
#pragma unroll
    for (int i = 0; i < FR; ++i) rsum[i] = 0.f;
    const int nk = t.stages(BK);
    auto add_up = [&](auto with_sums) {
    for (int kt = 0; kt < nk; ++kt) {
      char* const at_r = lds + use_r * Ring::kRStage;
      char* const at_s = ring_s + use_s * Ring::kSStage;
      if constexpr (!DIRECT) {
        sr.src.put(at_r, hr);
        ss.src.put(at_s, hs);
      } else {
        // this stage of both operands has arrived (vector memory operations end in the order of their issue)
        if (behind == 0)
          wait_loads<AHEAD>();
        else if (behind == 1)
          wait_loads<AHEAD + Y_OPS>();
        else
          wait_loads<AHEAD + Y_OPS + D_OPS>();
        behind = 0;
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // ... and all waves are done with the one before
      if constexpr (PAIR) {
        rr.anew();
        rs.anew();
      }
      typename Frag<T>::type fr[2][FR], fc[2][FC];
#pragma unroll
      for (int i = 0; i < FR; ++i) fr[0][i] = get_r(at_r, i, 0);
#pragma unroll
      for (int j = 0; j < FC; ++j) fc[0][j] = get_s(at_s, j, 0);
      if (DEEP_S) {
        load_r();
        load_s();
      } else {
        load_s();
        load_r();
      }
#pragma unroll
      for (int s = 0; s < KB / 32; ++s) {       // the next k-step's fragments are read while this one's are multiplied
        if (s + 1 < KB / 32) {
#pragma unroll
          for (int i = 0; i < FR; ++i) fr[(s + 1) & 1][i] = get_r(at_r, i, s + 1);
          if (!PAIR || (s & 1)) {
#pragma unroll
            for (int j = 0; j < FC; ++j) fc[slot_s(s + 1)][j] = get_s(at_s, j, s + 1);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < Frag<T>::kSteps; ++u)
#pragma unroll
          for (int i = 0; i < FR; ++i)
#pragma unroll
            for (int j = 0; j < FC; ++j) Frag<T>::mma(fc[slot_s(s)][j], fr[s & 1][i], acc[i][j], u);
        if constexpr (decltype(with_sums)::value) {
#pragma unroll
          for (int i = 0; i < FR; ++i) rsum[i] = Frag<T>::sum(fr[s & 1][i], rsum[i]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      use_r = use_r == Ring::kR - 1 ? 0 : use_r + 1;
      use_s = use_s == Ring::kS - 1 ? 0 : use_s + 1;
    }
    };
    if constexpr (kRowSums<KIND, BR, PAIR>) {
      if (row_sums)
        add_up(std::true_type());
      else
        add_up(std::false_type());
    } else {
      add_up(std::false_type());
    }
    if (kRowSums<KIND, BR, PAIR> && row_sums) {
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        const float sum = rsum[i] + __shfl_xor(rsum[i], 32);
        const int rl = wr + 32 * i + lane;
        if (lane < 32 && rl < t.nr) {
          if (a.db_slab != nullptr && t.z >= 0)
            a.db_slab[(int64_t)t.z * a.rows + t.row0 + rl] = sum;
          else
            reinterpret_cast<T*>(a.db)[(int64_t)t.g * a.rows + t.row0 + rl] = (T)sum;
        }
      }
    }

    // ---- epilogue, 32 rows of the wave's tile at a time through the stages just multiplied, which nothing fills before
    // the next barrier (and the LDS behind the rings, where those are short).  A lane holds four consecutive columns of one row; 16-byte slot s of row r lies at
    // s ^ (r mod slots), so that eight rows written at the same column fall on different banks.
    char* const mine = wave < Ring::kRWaves ? lds + (use_r == 0 ? Ring::kR - 1 : use_r - 1) * Ring::kRStage + wave * Ring::kEp
                       : wave < Ring::kRWaves + Ring::kSWaves
                           ? ring_s + (use_s == 0 ? Ring::kS - 1 : use_s - 1) * Ring::kSStage + (wave - Ring::kRWaves) * Ring::kEp
                           : lds + Ring::kBehind + (wave - Ring::kRWaves - Ring::kSWaves) * Ring::kEp;
    const int c = lane % LPR, cl = wc + 8 * c;
    const int64_t col = t.col0 + cl;
    const int left = t.nc - cl < 8 ? t.nc - cl : 8;
    float b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = 0.f;
    if (KIND == kFwd && a.bias != nullptr && a.slab == nullptr && t.g >= 0) {
      const T* bp = reinterpret_cast<const T*>(a.bias) + t.g * a.bias_group + col;
      load_any<T, 8>(bp, left, b);
    }
    // This lane's first row; the others are uniform distances away.  The residual's pieces of 32 rows are under way together
    // and used in order without an index (one after the other the residual block of 32768 x 1024 takes 328 us, so 317; the
    // registers that this costs make 65536 x 4096 -> 256 without a residual 1 % slower).
    const int64_t row0 = t.row0 + wr + lane / LPR;
    T* const out0 = reinterpret_cast<T*>(a.C) + (KIND == kDw ? t.g * a.c_group : 0) + row0 * a.ldc + col;
    constexpr int IT = 32 / RPI, RP = 8 * (int)sizeof(T) / 16;
    const bool with_res = KIND == kFwd && a.res != nullptr && a.slab == nullptr && t.g >= 0;
    u32x4 ahead[KIND == kFwd ? IT * RP : 1];
    const T* const res0 = reinterpret_cast<const T*>(a.res) + row0 * a.ldres + col;
    auto fetch = [&](int i) {
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        if (wr + 32 * i + it * RPI + lane / LPR >= t.nr || left <= 0) continue;
        const T* rp = res0 + (int64_t)(32 * i + it * RPI) * a.ldres;
        if (left == 8) {
#pragma unroll
          for (int q = 0; q < RP; ++q) ahead[it * RP + q] = reinterpret_cast<const u32x4_anywhere*>(rp)[q];
        } else {
          union {
            u32x4 u[RP];
            T t[8];
          } x;
#pragma unroll
          for (int e = 0; e < 8; ++e) x.t[e] = e < left ? rp[e] : (T)0.f;
#pragma unroll
          for (int q = 0; q < RP; ++q) ahead[it * RP + q] = x.u[q];
        }
      }
    };
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // every wave is done reading the stages
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      if (wr + 32 * i >= t.nr) break;          // uniform over the wave
      if constexpr (KIND != kFwd && sizeof(T) == 2) {
        // nothing is added to dx and dW any more: rounded first, half as much passes through LDS
        if (a.slab == nullptr || t.z < 0) {
          typedef T four __attribute__((ext_vector_type(4)));
#pragma unroll
          for (int j = 0; j < FC; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = lane & 31, s = 4 * j + e;
              const f32x16& v = acc[i][j];
              *reinterpret_cast<four*>(mine + r * (WC * 2) + ((s ^ (r & (WC / 8 - 1))) << 4) + 8 * (lane >> 5)) =
                  four{(T)v[4 * e], (T)v[4 * e + 1], (T)v[4 * e + 2], (T)v[4 * e + 3]};
            }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
          for (int it = 0; it < IT; ++it) {
            const int r = it * RPI + lane / LPR, rl = wr + 32 * i + r;
            if (rl >= t.nr || left <= 0) continue;
            const u32x4 v = *reinterpret_cast<const u32x4*>(mine + r * (WC * 2) + ((c ^ (r & (WC / 8 - 1))) << 4));
            T* out = out0 + (int64_t)(32 * i + it * RPI) * a.ldc;
            if (left == 8) {
              __builtin_nontemporal_store((u32x4_anywhere)v, reinterpret_cast<u32x4_anywhere*>(out));
            } else {
              union {
                u32x4 u;
                T t[8];
              } x;
              x.u = v;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (e < left) out[e] = x.t[e];
            }
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // read before the next 32 rows are written
          continue;
        }
      }
#pragma unroll
      for (int j = 0; j < FC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = lane & 31, s = 8 * j + 2 * e + (lane >> 5);
          *reinterpret_cast<f32x4*>(mine + r * (WC * 4) + ((s ^ (r & (SLOTS - 1))) << 4)) =
              f32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // the wave reads only what it wrote itself
      if (with_res) fetch(i);
#pragma unroll 1
      for (int it = 0; it < IT; ++it) {
        const int r = it * RPI + lane / LPR, rl = wr + 32 * i + r;
        if (rl >= t.nr || left <= 0) continue;
        const f32x4 v0 = *reinterpret_cast<const f32x4*>(mine + r * (WC * 4) + (((2 * c) ^ (r & (SLOTS - 1))) << 4));
        const f32x4 v1 = *reinterpret_cast<const f32x4*>(mine + r * (WC * 4) + (((2 * c + 1) ^ (r & (SLOTS - 1))) << 4));
        if (a.slab != nullptr && t.z >= 0) {
          float* out = a.slab + ((int64_t)t.z * a.rows + row0 + 32 * i + it * RPI) * a.cols + col;
          if (left == 8 && a.cols % 4 == 0) {
            *reinterpret_cast<f32x4*>(out) = v0;
            *reinterpret_cast<f32x4*>(out + 4) = v1;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e < left) out[e] = e < 4 ? v0[e] : v1[e - 4];
          }
          continue;
        }
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = v0[e];
          v[e + 4] = v1[e];
        }
        T* out = out0 + (int64_t)(32 * i + it * RPI) * a.ldc;
        if (KIND == kFwd) {
          float d[8], q[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = d[e] = 0.f;
          if (t.g >= 0) {
            if (with_res) {
              union {
                u32x4 u[RP];
                T t[8];
              } x;
#pragma unroll
              for (int p = 0; p < RP; ++p) x.u[p] = ahead[p];
#pragma unroll
              for (int e = 0; e < 8; ++e) q[e] = (float)x.t[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += b[e];
            activate<sizeof(T) == 2, 8>(a.act, v, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += q[e];
          }
          if (a.dact != nullptr) {
            float* dp = a.dact + row0 * a.lddact + col + (int64_t)(32 * i + it * RPI) * a.lddact;
            store_any<true, float, 8>(dp, left, d);
          }
        }
        store_any<true, T, 8>(out, left, v);
        if constexpr (KIND == kFwd) {
#pragma unroll
          for (int p = 0; p + RP < IT * RP; ++p) ahead[p] = ahead[p + RP];
        }
      }
    }
    // a full tile in 16-byte pieces: the number of its stores is known
    behind = a.slab == nullptr && t.nr == BR && t.nc == BC ? (KIND == kFwd && a.dact != nullptr ? 2 : 1) : 0;
  }
  if constexpr (DIRECT) wait_loads<0>();         // the zeros behind the last tile: nothing may write into the next workgroup's LDS
}

int launch_gemm_f32(int kind, int tile, bool direct, bool pair, const GemmArgs& a, const bnpvi_ctx* ctx, hipStream_t s);
int launch_gemm_bf16(int kind, int tile, bool direct, bool pair, const GemmArgs& a, const bnpvi_ctx* ctx, hipStream_t s);
int launch_gemm_f16(int kind, int tile, bool direct, bool pair, const GemmArgs& a, const bnpvi_ctx* ctx, hipStream_t s);

}  // namespace bnpvi
