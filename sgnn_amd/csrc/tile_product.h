// Matrix products of fp32 or bf16 operands on the bf16 matrix instructions: element types, the
// exact splitting of fp32 and the inner loop of a 128 x 128 tile.
//
// bf16 operands go in as they are: their products are exact and summed in 32 bits.  An fp32 number
// is the sum of three bf16 numbers (8 bits of its mantissa cut off, the next 8 rounded to nearest, the
// rest exactly), taken apart in registers on the way from LDS to the matrix instruction.  The second
// is at most 2^-7, the third 2^-16 of the number's power of two, so of the nine products of two numbers
// the three smallest, at most 2^-22 of the whole and of either sign, are left out.  (With the first
// rounded, too, that would be 2^-24, for 4 % of the time and no visible difference in the results: the
// sums' roundings are larger.)
#pragma once
#include "common.h"

namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Bf16 { uint16_t bits; };

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(Bf16 v) { return __uint_as_float(unsigned(v.bits) << 16); }
__device__ __forceinline__ uint16_t to_bf16(float v) {                       // nearest even
  const __bf16 h = static_cast<__bf16>(v);
  uint16_t bits;
  __builtin_memcpy(&bits, &h, 2);
  return bits;
}
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ Bf16 narrow<Bf16>(float v) { return Bf16{to_bf16(v)}; }

// v = a + b + c exactly, each a bf16 number, 8 + 8 + 8 bits of its mantissa cut off: for products that
// take all three.  An infinity or NaN leaves a NaN behind.
__device__ __forceinline__ void split3(float v, float& a, float& b, float& c) {
  a = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  const float r = v - a;
  b = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  c = r - b;
}
// the high halves of two floats as a bf16 pair
__device__ __forceinline__ unsigned high_halves(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// two numbers as pairs of bf16 numbers, v = a + b + c exactly: a cut off, b rounded to nearest (cut off,
// too, it would leave c twice as large and always of v's sign).  An infinity or NaN leaves a NaN behind.
__device__ __forceinline__ void split_pair(float lo, float hi, unsigned& a, unsigned& b, unsigned& c) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  a = high_halves(lo, hi);
  const float rl = lo - __uint_as_float(__float_as_uint(lo) & 0xffff0000u);
  const float rh = hi - __uint_as_float(__float_as_uint(hi) & 0xffff0000u);
  const bf16x2 rounded = __builtin_convertvector((f32x2{rl, rh}), bf16x2);
  __builtin_memcpy(&b, &rounded, 4);
  c = high_halves(rl - __uint_as_float(b << 16), rh - __uint_as_float(b & 0xffff0000u));
}

// bf16 numbers an element of type T is made of
template <typename T> struct Planes { static constexpr int kCount = sizeof(T) == 4 ? 3 : 1; };

__device__ __forceinline__ void planes_of(const float (&v)[8], bf16x8 (&out)[3]) {
  u32x4 pl[3];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    unsigned a, b, c;
    split_pair(v[e], v[e + 1], a, b, c);
    pl[0][e / 2] = a;
    pl[1][e / 2] = b;
    pl[2][e / 2] = c;
  }
#pragma unroll
  for (int q = 0; q < 3; ++q) __builtin_memcpy(&out[q], &pl[q], 16);
}
__device__ __forceinline__ void planes_of(const Bf16 (&v)[8], bf16x8 (&out)[1]) { __builtin_memcpy(&out[0], &v, 16); }

// acc += a . b over the planes' products that count
template <int P>
__device__ __forceinline__ void multiply_planes(const bf16x8 (&a)[P], const bf16x8 (&b)[P], f32x16& acc) {
#pragma unroll
  for (int pa = 0; pa < P; ++pa)
#pragma unroll
    for (int pb = 0; pa + pb < P; ++pb) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[pa], b[pb], acc, 0, 0, 0);
}

// row of element e of a 32 x 32 block of results (its column is lane & 31)
__device__ __forceinline__ int block_row(int e, int lane) { return 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }

// ------------------------------------------------------------------ the 128 x 128 tile
// Four wavefronts form a 128 x 128 tile, 64 x 64 each, in steps of 128 bytes of the reduction.
// Operands travel from memory to LDS without passing registers, one step ahead.  An operand is
// "deep" when its memory is contiguous along the reduction (LDS holds [128 rows][128 bytes], read
// directly) and "flat" when it is contiguous along the tile ([reduction][128 columns]; bf16 is read
// through the transposing LDS load, fp32 element by element).  16-byte chunks are permuted on the
// way in so that no read meets bank conflicts.
constexpr int kTile = 128;
constexpr int kThreads = 256;
constexpr int kStageBytes = kTile * 128;         // of one operand
constexpr int kProductLds = 4 * kStageBytes;     // two operands, two stages

template <typename T>
struct Operand {
  const T* base;           // 16-byte aligned, as every row is
  int64_t ld;              // row stride in elements
  int64_t rows;            // rows that exist: reads beyond repeat the last one
  int64_t cols;            // columns that exist (flat operands; a multiple of 16 bytes): likewise
};

template <typename T> struct Step { static constexpr int kDepth = 128 / sizeof(T); };

// 16 bytes a lane from `src` to LDS byte `dst` + 16 * lane (`dst` the same for the wavefront).
// Written as an instruction, since behind the builtin the compiler makes every later transposing
// LDS read wait for all loads in flight, which undoes the prefetch.  It has no result to wait for
// in a register: `landed` and a barrier come before anybody reads the LDS.  m0 is reserved (the
// compiler sets it right before the few instructions that take it, none of which is in these
// kernels), so it is set here each time and needs no mention as a clobber.
__device__ __forceinline__ void load_to_lds(const void* src, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory");
}
// the same from a uniform base and a 32-bit offset of the lane's own
__device__ __forceinline__ void load_to_lds(const char* base, unsigned offset, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(offset), "s"(base)
               : "memory");
}
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ unsigned lds_offset(const char* p) {
  return unsigned(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p));
}

// A 16-byte LDS read is served sixteen lanes at a time, not all of them neighbours (0-3, 12-15,
// 20-23, 24-27, and so on); its chunks have to lie in sixteen different places of 256 bytes.
// Rows of 128 bytes alternate between the halves; this moves the chunks of the others apart, and
// the four rows that a transposing read touches together to different 64-byte blocks.
__device__ __forceinline__ int spread_128(int row) { return ((row & 2) << 1) | ((row >> 2) & 3); }
// the same for rows of 256 bytes (or a multiple): sixteen chunks
__device__ __forceinline__ int spread_256(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }

// deep: rows r0 .. r0 + 127 at reduction offset k0;  flat: reduction rows k0 .. at columns r0 ..
template <typename T, bool DEEP>
__device__ __forceinline__ void stage_operand(const Operand<T>& op, int64_t r0, int64_t k0, unsigned lds, int wave,
                                              int lane) {
  constexpr int V = 16 / sizeof(T);              // elements of a chunk
#pragma unroll
  for (int l = 0; l < kStageBytes / 16 / kThreads; ++l) {
    const int first = (l * 4 + wave) * 64, q = first + lane;
    const T* src;
    if constexpr (DEEP) {
      const int row = q >> 3, c = (q & 7) ^ spread_128(row);
      int64_t r = r0 + row;
      r = r < op.rows ? r : op.rows - 1;
      src = op.base + r * op.ld + k0 + c * V;
    } else {
      constexpr int cpr = kTile / V;
      const int row = q / cpr;
      const int c = (q % cpr) ^ (sizeof(T) == 2 ? (row & 3) << 2 : ((row >> 3) & 1) << 3);
      int64_t r = k0 + row, col = r0 + c * V;
      r = r < op.rows ? r : op.rows - 1;
      col = col < op.cols ? col : op.cols - V;
      src = op.base + r * op.ld + col;
    }
    load_to_lds(src, lds + first * 16);
  }
}

// byte of element (reduction row k, column m) of a staged flat operand of bf16
__device__ __forceinline__ int flat_at(int k, int m) { return k * 256 + ((m >> 3) ^ ((k & 3) << 2)) * 16 + (m & 7) * 2; }

// the operand of one 32 x 32 x 16 instruction: element `lane & 31` of the block at m0, eight
// reduction indexes from k0 + 8 * (lane / 32)
template <bool DEEP>
__device__ __forceinline__ void read_fragment(const char* lds, int m0, int k0, int lane, bf16x8& out) {
  if constexpr (DEEP) {
    const int row = m0 + (lane & 31), c = (k0 >> 3) + (lane >> 5);
    out = *reinterpret_cast<const bf16x8*>(lds + row * 128 + ((c ^ spread_128(row)) << 4));
  } else {
    const int k = k0 + 8 * (lane >> 5) + ((lane & 15) >> 2);
    const int m = m0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const char* at = lds + flat_at(k, m);                                // k and k + 4 share k & 3
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * 256));
    __builtin_memcpy(&out, &lo, 8);
    __builtin_memcpy(reinterpret_cast<char*>(&out) + 8, &hi, 8);
  }
}
template <bool DEEP>
__device__ __forceinline__ void read_fragment(const char* lds, int m0, int k0, int lane, float (&out)[8]) {
  if constexpr (DEEP) {
    const int row = m0 + (lane & 31), c = (k0 >> 2) + 2 * (lane >> 5);
    const char* at = lds + row * 128;
    *reinterpret_cast<f32x4*>(&out[0]) = *reinterpret_cast<const f32x4*>(at + ((c ^ spread_128(row)) << 4));
    *reinterpret_cast<f32x4*>(&out[4]) = *reinterpret_cast<const f32x4*>(at + (((c + 1) ^ spread_128(row)) << 4));
  } else {
    const int k = k0 + 8 * (lane >> 5), m = m0 + (lane & 31);
    const char* at = lds + k * 512 + (((m >> 5) ^ ((k >> 3) & 1)) << 7) + (m & 31) * 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = *reinterpret_cast<const float*>(at + j * 512);
  }
}

typedef f32x16 Tile[2][2];

__device__ __forceinline__ void clear(Tile& acc) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
}

// What a wavefront's 64 x 64 needs for sixteen of the reduction: A's two blocks, then B's
typedef float Sixteen[4][8];
typedef u32x4 SixteenPlanes[4][3];

template <bool ADEEP, bool BDEEP>
__device__ __forceinline__ void read_sixteen(const char* stage, int kk, int wm, int wn, int lane, Sixteen& v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    read_fragment<ADEEP>(stage, wm + 32 * i, kk, lane, v[i]);
    read_fragment<BDEEP>(stage + kStageBytes, wn + 32 * i, kk, lane, v[2 + i]);
  }
}
// two neighbours of the 32 numbers a lane holds, to their planes
__device__ __forceinline__ void take_apart(const Sixteen& v, int pair, SixteenPlanes& out) {
  const int x = pair >> 2, e = 2 * (pair & 3);
  unsigned a, b, c;
  split_pair(v[x][e], v[x][e + 1], a, b, c);
  asm volatile("" : "+v"(a), "+v"(b), "+v"(c));  // now, not where it is used
  out[x][0][e / 2] = a;
  out[x][1][e / 2] = b;
  out[x][2][e / 2] = c;
}
// the products of `now`, and between them `next` taken apart: a wavefront's arithmetic fills the 32
// cycles of each matrix instruction (with all of a step's numbers taken apart before its products
// 2048 x 602 against 10007 classes in fp32 takes 190 + 173 us for statistics and dz, so 177 + 166 us)
__device__ __forceinline__ void multiply_sixteen(const SixteenPlanes& now, Tile& acc, const Sixteen& next,
                                                 SixteenPlanes& then) {
  constexpr int kPa[6] = {0, 0, 0, 1, 1, 2}, kPb[6] = {0, 1, 2, 0, 1, 0};
  int pair = 0;
#pragma unroll
  for (int s = 0; s < 24; ++s) {
    const int i = s / 12, j = s / 6 % 2, q = s % 6;
    bf16x8 a, b;
    __builtin_memcpy(&a, &now[i][kPa[q]], 16);
    __builtin_memcpy(&b, &now[2 + j][kPb[q]], 16);
    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc[i][j], 0, 0, 0);
    if (s >= 4 && s % 5 != 3) take_apart(next, pair++, then);
  }
}

// acc += A[m0 .., k0 .. k1] . B[n0 .., k0 .. k1]; k1 - k0 a multiple of the step.  `lds` holds two
// stages of both operands; every wavefront has left them when this returns.  bf16: `each` has its say
// in every step: `landed` before the next step's loads, `ahead`(k of the next) among them, `behind`(B's
// stage, acc) behind the products.
struct Nothing {
  __device__ __forceinline__ void landed() const {}
  __device__ __forceinline__ void ahead(int64_t) const {}
  __device__ __forceinline__ void behind(const char*, Tile&) const {}
};
template <typename T, bool ADEEP, bool BDEEP, typename Each = Nothing>
__device__ __forceinline__ void multiply(const Operand<T>& A, int64_t m0, const Operand<T>& B, int64_t n0, int64_t k0,
                                         int64_t k1, char* lds, Tile& acc, Each&& each = Each{}) {
  constexpr int kDepth = Step<T>::kDepth;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  const unsigned stages = lds_offset(lds);
  const auto stage = [&](int64_t k, int at) {
    stage_operand<T, ADEEP>(A, m0, k, stages + at * 2 * kStageBytes, wave, lane);
    stage_operand<T, BDEEP>(B, n0, k, stages + (at * 2 + 1) * kStageBytes, wave, lane);
  };
  stage(k0, 0);
  int cur = 0;
  if constexpr (sizeof(T) == 4) {
    static_assert(kDepth == 32, "two sixteens a step");
    Sixteen raw;
    SixteenPlanes first, second;
    landed();
    __syncthreads();
    if (k0 + kDepth < k1) stage(k0 + kDepth, 1);
    read_sixteen<ADEEP, BDEEP>(lds, 0, wm, wn, lane, raw);
#pragma unroll
    for (int pair = 0; pair < 16; ++pair) take_apart(raw, pair, first);
    for (int64_t k = k0; k < k1; k += kDepth) {
      read_sixteen<ADEEP, BDEEP>(lds + cur * 2 * kStageBytes, 16, wm, wn, lane, raw);
      multiply_sixteen(first, acc, raw, second);
      landed();                                  // this wavefront's part of the next stage
      __syncthreads();                           // everybody's, and this one has been read
      cur ^= 1;
      if (k + 2 * kDepth < k1) stage(k + 2 * kDepth, cur ^ 1);
      read_sixteen<ADEEP, BDEEP>(lds + cur * 2 * kStageBytes, 0, wm, wn, lane, raw);    // behind the last: not used
      multiply_sixteen(second, acc, raw, first);
    }
    __syncthreads();
    return;
  }
  for (int64_t k = k0; k < k1; k += kDepth) {
    landed();                                    // this wavefront's part of the stage
    each.landed();
    __syncthreads();                             // everybody's, and the other stage is free
    if (k + kDepth < k1) {
      stage(k + kDepth, cur ^ 1);
      each.ahead(k + kDepth);
    }
    const char* a = lds + cur * 2 * kStageBytes;
#pragma unroll
    for (int kk = 0; kk < kDepth; kk += 16) {
      bf16x8 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        read_fragment<ADEEP>(a, wm + 32 * i, kk, lane, fa[i]);
        read_fragment<BDEEP>(a + kStageBytes, wn + 32 * i, kk, lane, fb[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
    each.behind(a + kStageBytes, acc);
    cur ^= 1;
  }
  __syncthreads();
}

}  // namespace
