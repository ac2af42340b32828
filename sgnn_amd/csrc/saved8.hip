// A layer's input kept in 8 bits between its forward and its backward pass.
//
// a = x > 0 ? x : slope * x (the inner activation of a layer) is held as one byte per element
// plus one byte per group of 32 consecutive features of a row, the group's power-of-two step
// 2^s (biased by 127; 255 marks a group that holds a NaN or an infinity and decodes to NaN):
//   slope == 1 : code = rint(a / 2^s),     value = code * 2^s,         s = smallest with |code| <= 127
//                (s <= 121: the last numbers before infinity are held as +-127 * 2^121)
//   otherwise  : code = ceil(a / 2^s) - 1, value = (code + 1/2) 2^s,   s = smallest with |a| <= 128 * 2^s
// In the second form a code is negative exactly where "x > 0" is false, so the same byte also
// answers for the activation's derivative; with slope 0 the negative codes stand for 0 and the
// group's range is that of its positive elements.  Either form is off by at most half a step.
//
// Steps are powers of two so that every value (at most 8 significant bits) is a bf16 number
// without any rounding: the weight gradient dW = grad^T . value runs on the bf16 matrix
// instructions with an exact left operand, and coding is exact in 32 bits, too (a multiplication
// by a power of two, one rounding to a whole number).
#include "tile_product.h"

namespace {

constexpr int kGroup = 32;
constexpr int kMinBiased = 2;                     // s >= -125: half a step is still a normal number
constexpr int kMaxBiased = 248;                   // s <= 121: 127.5 steps are still finite
constexpr int kBadGroup = 255;

// slope 0 is a selection, not a product: -inf becomes 0 there, NaN stays NaN
template <int N>
__device__ __forceinline__ void activate(float (&x)[N], float slope) {
  if (slope == 1.f) return;
  if (slope == 0.f) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = x[e] <= 0.f ? 0.f : x[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = x[e] > 0.f ? x[e] : slope * x[e];
  }
}
// the largest magnitude, as bits: a NaN is larger than any number there
template <int N>
__device__ __forceinline__ unsigned peak_of(const float (&a)[N], unsigned peak = 0) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const unsigned m = __float_as_uint(a[e]) & 0x7fffffffu;
    peak = m > peak ? m : peak;
  }
  return peak;
}

__device__ __forceinline__ int step_of(unsigned peak_bits, bool plain) {      // peak = max |a|, as bits
  const int e = int(peak_bits >> 23);
  const unsigned frac = peak_bits & 0x7fffffu;
  if (e == 255) return kBadGroup;
  // plain: 127.5 of 128 would round to 128; else a power of two is still held by its own exponent
  const int b = plain ? e - 6 + (frac >= 0x7f0000u ? 1 : 0) : e - 6 - (frac == 0u ? 1 : 0);
  return b < kMinBiased ? kMinBiased : b > kMaxBiased ? kMaxBiased : b;
}
__device__ __forceinline__ float step_value(int biased) {      // NaN for a bad group
  return biased == kBadGroup ? __uint_as_float(0x7fc00000u) : __uint_as_float(unsigned(biased) << 23);
}

// four codes at 1 / step = inv (0 in a bad group), as a word.  They are formed as code + 128, which
// the conversion to a byte holds within 0 .. 255 by itself: -129 becomes -128 and 128 becomes 127.
// A positive element whose quotient fell to 0 keeps its sign by the maximum with `floor`, which also
// drops the NaN of a bad group.
template <bool PLAIN>
__device__ __forceinline__ unsigned pack_four(const float* a, float inv) {
  unsigned word = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float s = a[e] * inv;
    const float u = PLAIN ? fmaxf(rintf(s) + 128.f, 1.f) : fmaxf(ceilf(s) + 127.f, a[e] > 0.f ? 128.f : 0.f);
    word = __builtin_amdgcn_cvt_pk_u8_f32(u, e, word);
  }
  return word ^ 0x80808080u;
}
// 4 * W elements: the choice is made once, not for every element
template <int W>
__device__ __forceinline__ void pack_codes(const float (&a)[4 * W], float inv, bool plain, unsigned (&word)[W]) {
  if (plain) {
#pragma unroll
    for (int w = 0; w < W; ++w) word[w] = pack_four<true>(a + 4 * w, inv);
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w) word[w] = pack_four<false>(a + 4 * w, inv);
  }
}
__device__ __forceinline__ float inverse_step(int biased) {
  return biased == kBadGroup ? 0.f : __uint_as_float(unsigned(254 - biased) << 23);
}

// `u` = code + 128 as a number: value = (u - (plain ? 128 : 127.5)) * step, exact.  With slope 0
// the clamp at 127.5 makes the negative codes exactly 0 and leaves a NaN step NaN.
__device__ __forceinline__ float decode(float u, float step, float offset, float floor_u) {
  return (fmaxf(u, floor_u) + offset) * step;
}

// Elements per thread of the element-wise passes: 16 bytes of the wide operand.
template <typename T> struct Lane { static constexpr int kElems = 16 / sizeof(T); };

// A lane's piece of a row: one access of 16 bytes wherever the row begins (memory takes any alignment;
// element by element 19717 x 500 in bf16 takes 14 us to save and 17 to restore, so 10 and 8), single
// elements at its end.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, int left, T (&out)[V]) {
  if (left >= V) {
    __builtin_memcpy(&out, p, sizeof(out));
  } else {
    asm("" : "+v"(p));                           // or the last of these is merged with the last of those
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = i < left ? p[i] : narrow<T>(0.f);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, int left, const T (&v)[V]) {
  if (left >= V) {
    __builtin_memcpy(p, &v, sizeof(v));
  } else {
    asm("" : "+v"(p));
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < left) p[i] = v[i];
  }
}

// A workgroup owns `rows` whole rows; `per_row` = lanes a row takes (a multiple of a group's
// lanes, so that a group never leaves its wavefront's aligned block of lanes).
// Bound by memory: 232965 x 256 fp32 saved in 70 us (301 MB, 4.3 TB/s) and restored in 59 us (5.1; a
// copy reaches 5.1).
constexpr int kEltThreads = 256;

template <typename T>
__global__ __launch_bounds__(kEltThreads) void k_save8(int64_t n, int F, const T* __restrict__ x, int64_t ldx,
                                                       float slope, int rows, int per_row, uint8_t* __restrict__ codes, uint8_t* __restrict__ steps) {
  constexpr int V = Lane<T>::kElems, kPer = kGroup / V;
  const bool plain = slope == 1.f;
  const int groups = (F + kGroup - 1) / kGroup;
  const int64_t row0 = int64_t(blockIdx.x) * rows;
  const int count = int(n - row0 < rows ? n - row0 : rows) * per_row;
  for (int i = threadIdx.x; i < count; i += kEltThreads) {
    const int lr = i / per_row, at = i - lr * per_row;
    const int64_t r = row0 + lr;
    const int f = at * V, left = F - f;
    T raw[V];
    load_row<T, V>(x + r * ldx + f, left, raw);
    float a[V];
#pragma unroll
    for (int e = 0; e < V; ++e) a[e] = widen(raw[e]);
    activate(a, slope);
    unsigned peak = peak_of(a);
#pragma unroll
    for (int off = 1; off < kPer; off <<= 1) {
      const unsigned o = unsigned(__shfl_xor(int(peak), off));
      peak = o > peak ? o : peak;
    }
    const int biased = step_of(peak, plain);
    const float inv = inverse_step(biased);
    unsigned packed[V / 4];
    pack_codes(a, inv, plain, packed);
    unsigned* dst = reinterpret_cast<unsigned*>(codes + r * (int64_t(groups) * kGroup) + f);
    if constexpr (V == 4) dst[0] = packed[0];
    else *reinterpret_cast<u32x2*>(dst) = u32x2{packed[0], packed[1]};
    if (at % kPer == 0) steps[r * groups + at / kPer] = uint8_t(biased);
  }
}

template <typename T>
__global__ __launch_bounds__(kEltThreads) void k_restore8(int64_t n, int F, const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ steps, float slope, int rows,
                                                          int per_row, T* __restrict__ out, int64_t ldo) {
  constexpr int V = Lane<T>::kElems, kPer = kGroup / V;
  const float offset = slope == 1.f ? -128.f : -127.5f, floor_u = slope == 0.f ? 127.5f : 0.f;
  const int groups = (F + kGroup - 1) / kGroup;
  const int64_t row0 = int64_t(blockIdx.x) * rows;
  const int count = int(n - row0 < rows ? n - row0 : rows) * per_row;
  for (int i = threadIdx.x; i < count; i += kEltThreads) {
    const int lr = i / per_row, at = i - lr * per_row;
    const int64_t r = row0 + lr;
    const int f = at * V;
    const unsigned* src = reinterpret_cast<const unsigned*>(codes + r * (int64_t(groups) * kGroup) + f);
    const float step = step_value(steps[r * groups + at / kPer]);
    T v[V];
#pragma unroll
    for (int w = 0; w < V / 4; ++w) {
      const unsigned u = src[w] ^ 0x80808080u;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        v[4 * w + b] = narrow<T>(decode(float((u >> (8 * b)) & 0xffu), step, offset, floor_u));
    }
    store_row<T, V>(out + r * ldo + f, F - f, v);
  }
}

// dx = grad where the code says x > 0, slope * grad elsewhere; dx may be grad itself.
template <typename T>
__global__ __launch_bounds__(kEltThreads) void k_input_grad8(int64_t n, int F, const uint8_t* __restrict__ codes,
                                                             float slope, int rows, int per_row, const T* g,
                                                             int64_t ldg, T* dx, int64_t lddx) {
  constexpr int V = Lane<T>::kElems;
  const int groups = (F + kGroup - 1) / kGroup;
  const int64_t row0 = int64_t(blockIdx.x) * rows;
  const int count = int(n - row0 < rows ? n - row0 : rows) * per_row;
  for (int i = threadIdx.x; i < count; i += kEltThreads) {
    const int lr = i / per_row, at = i - lr * per_row;
    const int64_t r = row0 + lr;
    const int f = at * V, left = F - f;
    if (left <= 0) continue;
    const unsigned* src = reinterpret_cast<const unsigned*>(codes + r * (int64_t(groups) * kGroup) + f);
    T v[V];
    load_row<T, V>(g + r * ldg + f, left, v);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const bool negative = (src[e / 4] >> (8 * (e % 4) + 7)) & 1u;
      if (negative) v[e] = slope == 0.f ? narrow<T>(0.f) : narrow<T>(slope * widen(v[e]));
    }
    store_row<T, V>(dx + r * lddx + f, left, v);
  }
}

// ---------------------------------------------------------------------------------
// dW[h][f] = sum_r grad[r][h] * value[r][f]: a product whose reduction runs over the rows, both
// operands row-major over it.  A workgroup forms a BH x BF tile of dW over a chunk of rows, 32
// rows at a time: codes are decoded and grad split into bf16 planes on the way from registers to
// LDS, both kept row-major there, and the matrix instructions' operands (8 consecutive rows of
// one column per lane) come out of the transposing LDS read.  grad in 32 bits is the sum of three
// bf16 numbers (8 + 8 + 8 bits of its mantissa, cut off, not rounded, so the sum is exact), which
// makes every product exact and the sums those of 32-bit arithmetic; bf16 grad takes one plane.
// Chunks go to the workspace and are added in chunk order by a second launch.
// Measured with its sum on 232965 x 602 fp32, 128 units: 143 us (codes and grad are 260 MB, 51 us; the
// matrix instructions of three planes 65 us, decoding and splitting as much again).  Two workgroups
// of eight wavefronts on a compute unit take turns at these; at one, 227 us.  Staging one step
// ahead into a second buffer saves a barrier a step and gains nothing (140 us instead of 137 without
// the sum).  169343 x 256 bf16, 256 units after a ReLU: 53 us, for 130 MB and as much of partial sums.
constexpr int kRowsStep = 32;

template <int COLS>                               // byte offset of (row, col) in a row-major bf16 slab of COLS columns
__device__ __forceinline__ int slab_at(int k, int col) {
  // 64-byte blocks of a row are permuted by the row so that the 4 rows x 64 bytes which a
  // transposing read touches at once fall into different banks
  constexpr int nb = COLS / 32;
  const int swz = nb >= 4 ? (k & 3) : nb == 2 ? ((k >> 1) & 1) : 0;
  return k * (COLS * 2) + (((col >> 5) ^ swz) << 6) + (col & 31) * 2;
}

template <int COLS>
__device__ __forceinline__ bf16x8 slab_frag(const char* slab, int k0, int c0, int lane) {
  const int k = k0 + 8 * (lane >> 5) + ((lane & 15) >> 2);
  const int c = c0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(slab + slab_at<COLS>(k, c)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(slab + slab_at<COLS>(k + 4, c)));
  bf16x8 r;
  __builtin_memcpy(&r, &lo, 8);
  __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &hi, 8);
  return r;
}

template <typename T, int BH, int BF, int WH, int WF>
__global__ __launch_bounds__(64 * WH * WF, BH >= 128 ? 4 : 2) void k_weight_grad8(
    int64_t n, int F, int H, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ steps, float slope,
    const T* __restrict__ g, int64_t ldg, int64_t chunk_rows, int chunks, int tiles_f, int tiles_h,
    T* __restrict__ dW, int64_t lddw, float* __restrict__ partial) {
  constexpr int kThreads = 64 * WH * WF;
  constexpr int P = sizeof(T) == 4 ? 3 : 1;
  constexpr int MH = BH / (32 * WH), MF = BF / (32 * WF);       // 32 x 32 blocks of a wavefront
  constexpr int kCodeLoads = kRowsStep * BF / 16 / kThreads;    // 16 codes each
  constexpr int GV = 8;                                         // grad elements a thread loads at once
  constexpr int kGradSlots = kRowsStep * BH / GV;
  constexpr int kGradLoads = (kGradSlots + kThreads - 1) / kThreads;
  __shared__ __align__(128) char sB[kRowsStep * BF * 2];
  __shared__ __align__(128) char sA[P * kRowsStep * BH * 2];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int wh = wave / WF, wf = wave % WF;
  // the tiles of one chunk of rows go to one XCD, one after the other: they share grad and codes through its L2
  const int tiles = tiles_f * tiles_h;
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  const bool spread = chunks < 8;                 // too few chunks for that: over all of them
  const int tile = (spread ? int(blockIdx.x) : slot) % tiles;
  const int chunk = spread ? int(blockIdx.x) / tiles : (slot / tiles) * 8 + xcd;
  if (chunk >= chunks) return;                    // the whole workgroup
  const int f0 = (tile % tiles_f) * BF, h0 = (tile / tiles_f) * BH;
  const int groups = (F + kGroup - 1) / kGroup, ldq = groups * kGroup;
  const int64_t first = int64_t(chunk) * chunk_rows;
  const int64_t last = first + chunk_rows < n ? first + chunk_rows : n;
  const float offset = slope == 1.f ? -128.f : -127.5f, floor_u = slope == 0.f ? 127.5f : 0.f;

  u32x4 rc[kCodeLoads];
  int rs[kCodeLoads];
  T rg[kGradLoads][GV];
  const auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int l = 0; l < kCodeLoads; ++l) {
      const int s = t + l * kThreads, k = s / (BF / 16), f = f0 + (s % (BF / 16)) * 16;
      const int64_t r = r0 + k;
      rc[l] = u32x4{0, 0, 0, 0};
      rs[l] = kMinBiased;
      if (r < last && f < ldq) {
        rc[l] = *reinterpret_cast<const u32x4*>(codes + r * ldq + f);
        rs[l] = steps[r * groups + (f >> 5)];
      }
    }
#pragma unroll
    for (int l = 0; l < kGradLoads; ++l) {
      const int s = t + l * kThreads, k = s / (BH / GV), h = h0 + (s % (BH / GV)) * GV;
      const int64_t r = r0 + k;
#pragma unroll
      for (int e = 0; e < GV; ++e) rg[l][e] = narrow<T>(0.f);
      if (s < kGradSlots && r < last && h < H) {
        const T* p = g + r * ldg + h;
        if (h + GV <= H) {
          __builtin_memcpy(&rg[l], p, sizeof(rg[l]));
        } else {
          asm("" : "+v"(p));
#pragma unroll
          for (int e = 0; e < GV; ++e)
            if (h + e < H) rg[l][e] = p[e];
        }
      }
    }
  };
  const auto stage = [&]() {
#pragma unroll
    for (int l = 0; l < kCodeLoads; ++l) {
      const int s = t + l * kThreads, k = s / (BF / 16), c = (s % (BF / 16)) * 16;
      const float step = step_value(rs[l]);
      unsigned out[8];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const unsigned u = rc[l][w] ^ 0x80808080u;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float lo = decode(float((u >> (16 * b)) & 0xffu), step, offset, floor_u);
          const float hi = decode(float((u >> (16 * b + 8)) & 0xffu), step, offset, floor_u);
          out[2 * w + b] = high_halves(lo, hi);
        }
      }
      u32x4* dst = reinterpret_cast<u32x4*>(sB + slab_at<BF>(k, c));
      dst[0] = u32x4{out[0], out[1], out[2], out[3]};
      dst[1] = u32x4{out[4], out[5], out[6], out[7]};
    }
#pragma unroll
    for (int l = 0; l < kGradLoads; ++l) {
      const int s = t + l * kThreads, k = s / (BH / GV), c = (s % (BH / GV)) * GV;
      if (s < kGradSlots) {
        if constexpr (P == 1) {
          u32x4 w;
          __builtin_memcpy(&w, &rg[l][0], 16);
          *reinterpret_cast<u32x4*>(sA + slab_at<BH>(k, c)) = w;
        } else {
          u32x4 pl[3];
#pragma unroll
          for (int e = 0; e < GV; e += 2) {
            float a0, b0, c0, a1, b1, c1;
            split3(widen(rg[l][e]), a0, b0, c0);
            split3(widen(rg[l][e + 1]), a1, b1, c1);
            pl[0][e / 2] = high_halves(a0, a1);
            pl[1][e / 2] = high_halves(b0, b1);
            pl[2][e / 2] = high_halves(c0, c1);
          }
#pragma unroll
          for (int p = 0; p < 3; ++p)
            *reinterpret_cast<u32x4*>(sA + p * (kRowsStep * BH * 2) + slab_at<BH>(k, c)) = pl[p];
        }
      }
    }
  };

  f32x16 acc[MH][MF];
#pragma unroll
  for (int i = 0; i < MH; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  fetch(first);
  for (int64_t r0 = first; r0 < last; r0 += kRowsStep) {
    __syncthreads();                              // the previous step's reads are done
    stage();
    if (r0 + kRowsStep < last) fetch(r0 + kRowsStep);
    __syncthreads();
#pragma unroll
    for (int k0 = 0; k0 < kRowsStep; k0 += 16) {
      bf16x8 b[MF];
#pragma unroll
      for (int j = 0; j < MF; ++j) b[j] = slab_frag<BF>(sB, k0, (wf * MF + j) * 32, lane);
#pragma unroll
      for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < MH; ++i) {
          const bf16x8 a = slab_frag<BH>(sA + p * (kRowsStep * BH * 2), k0, (wh * MH + i) * 32, lane);
#pragma unroll
          for (int j = 0; j < MF; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], acc[i][j], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MH; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j) {
      const int f = f0 + (wf * MF + j) * 32 + (lane & 31);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int h = h0 + (wh * MH + i) * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        if (h < H && f < F) {
          if (chunks > 1) partial[(int64_t(chunk) * H + h) * F + f] = acc[i][j][e];
          else dW[int64_t(h) * lddw + f] = narrow<T>(acc[i][j][e]);
        }
      }
    }
}

// dW = sum of the chunks' tiles: four quarters of the chunks in order, then the quarters in order.
template <typename T>
__global__ __launch_bounds__(256) void k_weight_grad_sum8(int F, int64_t total, int chunks,
                                                          const float* __restrict__ partial, T* __restrict__ dW,
                                                          int64_t lddw) {
  __shared__ float part[4][64];
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int64_t e = int64_t(blockIdx.x) * 64 + c;
  const int lo = int(int64_t(chunks) * q / 4), hi = int(int64_t(chunks) * (q + 1) / 4);
  float s = 0.f;
  if (e < total) {
#pragma unroll 8
    for (int z = lo; z < hi; ++z) s += partial[int64_t(z) * total + e];
  }
  part[q][c] = s;
  __syncthreads();
  if (q == 0 && e < total)
    dW[(e / F) * lddw + e % F] = narrow<T>((part[0][c] + part[1][c]) + (part[2][c] + part[3][c]));
}

// ---------------------------------------------------------------------------------
// The layer around the codes: y = a . weight^T from x itself, its codes written on the way, and
// dx = (grad . weight) * act'(x) with the activation's derivative read off the codes.  Both are
// bound by the rows they stream (x and y, grad and dx): a wavefront takes 32 of them straight from
// memory into the matrix instructions' operand, a lane holding eight features of one row; features
// 0-3 and 8-11 of sixteen in the first half of the wavefront, the others in the second, so that a
// load takes whole 32-byte pieces of a row.  The weight is split into bf16 planes on its way to LDS,
// 64 features (of x, or units of grad) at a time, and serves the workgroup's rows.  Measured on
// 232965 x 256 fp32 with 64 units: y and the codes 104 us (3.5 TB/s of the 360 MB it moves), dx 111 us
// (in pieces of 32 bytes, without the way through LDS, 118 us);
// with 64 rows a wavefront, so that a piece of the weight read from LDS serves two products, 114 and
// 129 us: half the wavefronts wait for the same loads.
constexpr int kLinStep = 64;

// eight elements of a row from `k`: k .. k + 3 and k + 8 .. k + 11; unless `whole`, which is the same
// for the wavefront, zeros from `left` on
template <typename T>
__device__ __forceinline__ void load_eight(const T* src, bool whole, int left, T (&v)[8]) {
  if (whole) {
    __builtin_memcpy(&v[0], src, 4 * sizeof(T));
    __builtin_memcpy(&v[4], src + 8, 4 * sizeof(T));
  } else {
    asm("" : "+v"(src));                         // or the last of these is merged with the last of those
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (e & 3) + (e >> 2) * 8 < left ? src[(e & 3) + (e >> 2) * 8] : T{};
  }
}

// one group's codes from a lane's sixteen of its 32 elements; lanes l and l + 32 share a row
__device__ __forceinline__ void save_group(const float (&a)[2][8], bool plain, bool store, int half, uint8_t* code_row,
                                           uint8_t* step_at) {
  const unsigned peak = peak_of(a[1], peak_of(a[0])), other = unsigned(__shfl_xor(int(peak), 32));
  const int biased = step_of(other > peak ? other : peak, plain);
  const float inv = inverse_step(biased);
  unsigned word[2][2];                           // features 16 s + 8 w + 4 half ..
  pack_codes(a[0], inv, plain, word[0]);
  pack_codes(a[1], inv, plain, word[1]);
  // the first half keeps features 0 .. 15, the second 16 .. 31
  const unsigned g0 = unsigned(__shfl_xor(int(half ? word[0][0] : word[1][0]), 32));
  const unsigned g1 = unsigned(__shfl_xor(int(half ? word[0][1] : word[1][1]), 32));
  const u32x4 out = half ? u32x4{g0, word[1][0], g1, word[1][1]} : u32x4{word[0][0], g0, word[0][1], g1};
  if (store) {
    *reinterpret_cast<u32x4*>(code_row + 16 * half) = out;
    if (half == 0) *step_at = uint8_t(biased);
  }
}

__device__ __forceinline__ void lin_planes(const float (&v)[8], bf16x8 (&out)[3]) { planes_of(v, out); }
__device__ __forceinline__ void lin_planes(const float (&v)[8], bf16x8 (&out)[1]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) out[0][e] = static_cast<__bf16>(v[e]);
}

// y[r][h] for 128 rows and 32 * NB units a workgroup; `codes` NULL: nothing is kept.  SPLIT, for few
// rows: 32 rows a workgroup, whose wavefronts take turns at the steps of the features, each with a
// piece of the weight of its own, and add their sums up in the end, in order.  MOVED, for bf16 whose slope
// is neither 0 nor 1: activations are two bf16 numbers each in the product (169343 x 128, 256 units, forward
// and backward 172 us; with one 170, and at slope 0.2 the output moves by 1.0e-3 of its norm).
template <typename T, int NB, bool SPLIT, bool MOVED>
__global__ __launch_bounds__(256) void k_linear8(int64_t n, int F, int H, const T* __restrict__ x, int64_t ldx,
                                                 const T* __restrict__ w, int64_t ldw, float slope,
                                                 uint8_t* __restrict__ codes, uint8_t* __restrict__ steps,
                                                 T* __restrict__ y, int64_t ldy) {
  constexpr int P = Planes<T>::kCount, kUnits = 32 * NB;
  constexpr int kLoaders = SPLIT ? 64 : 256;
  constexpr int kChunks = kUnits * (kLinStep / 8) / kLoaders;   // of 8 features, a thread's share of a weight step
  constexpr int kPiece = P * kUnits * kLinStep * 2, kStride = SPLIT ? 4 * kLinStep : kLinStep;
  static_assert(!SPLIT || NB <= 2, "LDS");
  __shared__ __align__(128) char all[SPLIT ? 4 * (kPiece > 128 * kUnits ? kPiece : 128 * kUnits) : kPiece];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int t = SPLIT ? lane : threadIdx.x;
  char* const lds = all + (SPLIT ? wave * kPiece : 0);
  const auto sync = [&] {
    if constexpr (SPLIT) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else __syncthreads();
  };
  const int h0 = int(blockIdx.y) * kUnits, groups = (F + kGroup - 1) / kGroup;
  const int64_t first = (SPLIT ? int64_t(blockIdx.x) : int64_t(blockIdx.x) * 4 + wave) * 32, r = first + (lane & 31);
  const bool plain = slope == 1.f, save = codes != nullptr && blockIdx.y == 0;
  const T* row_at = x + (r < n ? r : n - 1) * ldx + 4 * half;
  T wreg[kChunks][8];
  const auto fetch_weight = [&](int f0) {
#pragma unroll
    for (int l = 0; l < kChunks; ++l) {
      const int c = t + kLoaders * l, h = h0 + (c >> 3), f = f0 + 16 * ((c & 7) >> 1) + 4 * (c & 1);
#pragma unroll
      for (int e = 0; e < 8; ++e) wreg[l][e] = T{};
      if (h < H) load_eight(w + int64_t(h) * ldw + f, F - f0 >= kLinStep, F - f, wreg[l]);
    }
  };
  T xreg[2][8];
  const auto fetch_rows = [&](int f0) {
#pragma unroll
    for (int s = 0; s < 2; ++s) load_eight(row_at + f0 + 16 * s, F - f0 >= kGroup, F - f0 - 16 * s - 4 * half, xreg[s]);
  };
  f32x16 acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
  const int begin = SPLIT ? wave * kLinStep : 0;
  fetch_weight(begin);
  fetch_rows(begin);
  for (int f0 = begin; f0 < F; f0 += kStride) {
    sync();
#pragma unroll
    for (int l = 0; l < kChunks; ++l) {
      const int c = t + kLoaders * l, row = c >> 3;
      bf16x8 pl[P];
      planes_of(wreg[l], pl);
#pragma unroll
      for (int q = 0; q < P; ++q)
        *reinterpret_cast<bf16x8*>(lds + (q * kUnits + row) * (kLinStep * 2) + (((c & 7) ^ spread_128(row)) << 4)) = pl[q];
    }
    sync();
    if (f0 + kStride < F) fetch_weight(f0 + kStride);
#pragma unroll
    for (int g = 0; g < 2; ++g) {                // groups of 32 features
      const int f = f0 + 32 * g;
      if (f >= F) break;
      float a[2][8];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[s][e] = widen(xreg[s][e]);
        activate(a[s], slope);
      }
      const int next = g == 0 ? f + 32 : f0 + kStride;
      if (next < F) fetch_rows(next);
      if (save)
        save_group(a, plain, r < n, half, codes + r * (int64_t(groups) * kGroup) + f, steps + r * groups + (f >> 5));
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf16x8 fa[P], off;
        lin_planes(a[s], fa);
        if constexpr (MOVED) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float d = a[s][e] - static_cast<float>(fa[0][e]);
            off[e] = static_cast<__bf16>(fabsf(d) < INFINITY ? d : 0.f);       // infinities have said it all
          }
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const int row = 32 * j + (lane & 31), c = 4 * g + 2 * s + half;
          bf16x8 fb[P];
#pragma unroll
          for (int q = 0; q < P; ++q)
            fb[q] = *reinterpret_cast<const bf16x8*>(lds + (q * kUnits + row) * (kLinStep * 2) +
                                                     ((c ^ spread_128(row)) << 4));
          multiply_planes<P>(fa, fb, acc[j]);
          if constexpr (MOVED) acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(off, fb[0], acc[j], 0, 0, 0);
        }
      }
    }
  }
  if constexpr (SPLIT) {
    __syncthreads();
    float* const shares = reinterpret_cast<float*>(all);         // [wave][row][unit]
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        shares[(wave * 32 + block_row(e, lane)) * kUnits + 32 * j + (lane & 31)] = acc[j][e];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * kUnits; c += 256) {
      const int64_t out = first + c / kUnits;
      const int h = h0 + c % kUnits;
      const float sum = (shares[c] + shares[c + 32 * kUnits]) + (shares[c + 64 * kUnits] + shares[c + 96 * kUnits]);
      if (out < n && h < H) y[out * ldy + h] = narrow<T>(sum);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int h = h0 + 32 * j + (lane & 31);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t out = first + block_row(e, lane);
      if (out < n && h < H) y[out * ldy + h] = narrow<T>(acc[j][e]);
    }
  }
}

// dx[r][f] for 128 rows and the features of blockIdx.y, 64 at a time, a workgroup.  The product
// comes out features x rows, so that a lane holds four neighbouring features of one row: their codes
// are one word and their results one store.
template <typename T>
__global__ __launch_bounds__(256) void k_linear_grad8(int64_t n, int F, int H, const T* __restrict__ g, int64_t ldg,
                                                      const T* __restrict__ w, int64_t ldw, float slope,
                                                      const uint8_t* __restrict__ codes, T* __restrict__ dx,
                                                      int64_t lddx) {
  constexpr int P = Planes<T>::kCount;
  constexpr int kChunks = kLinStep * 8 / 256;    // of 8 features, a thread's share of a weight step (64 x 64)
  constexpr int kKept = 4;                       // sixteens of units whose grad stays in registers
  constexpr int kJoined = sizeof(T) == 4 ? 1 : 2;        // blocks of 32 features in 128 bytes of a row
  __shared__ __align__(128) char lds[P * kLinStep * 128], turned[4][32 * 128];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), half = lane >> 5;
  const int64_t first = (int64_t(blockIdx.x) * 4 + wave) * 32, r = first + (lane & 31);
  const int ldq = (F + kGroup - 1) / kGroup * kGroup;
  const T* row_at = g + (r < n ? r : n - 1) * ldg + 4 * half;
  bf16x8 fb[kKept][P];
  const auto fetch_grad = [&](int k0) {
#pragma unroll
    for (int s = 0; s < kKept; ++s) {
      T v[8];
      load_eight(row_at + k0 + 16 * s, H - k0 >= 16 * (s + 1), H - k0 - 16 * s - 4 * half, v);
      planes_of(v, fb[s]);
    }
  };
  T wreg[kChunks][8];
  const auto fetch_weight = [&](int k0, int f0) {
#pragma unroll
    for (int l = 0; l < kChunks; ++l) {
      const int c = t + 256 * l, h = k0 + (c >> 3), f = f0 + 8 * (c & 7);
#pragma unroll
      for (int e = 0; e < 8; ++e) wreg[l][e] = T{};
      if (h < H) {
        const T* src = w + int64_t(h) * ldw + f;
        if (f + 8 <= F) {
          __builtin_memcpy(&wreg[l], src, sizeof(wreg[l]));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (f + e < F) wreg[l][e] = src[e];
        }
      }
    }
  };
  const int tiles = (F + kLinStep - 1) / kLinStep;
  const int tile0 = int(int64_t(tiles) * blockIdx.y / gridDim.y), tile1 = int(int64_t(tiles) * (blockIdx.y + 1) / gridDim.y);
  if (tile0 >= tile1) return;                    // the whole workgroup
  fetch_grad(0);
  fetch_weight(0, tile0 * kLinStep);
  for (int tile = tile0; tile < tile1; ++tile) {
    const int f0 = tile * kLinStep;
    unsigned signs[2][4];                        // four features each, under way while the product forms
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int f = f0 + 32 * j + block_row(4 * e, lane);
        signs[j][e] = slope != 1.f && r < n && f < F ? *reinterpret_cast<const unsigned*>(codes + r * ldq + f) : 0u;
      }
    f32x16 acc[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
    for (int k0 = 0; k0 < H; k0 += kLinStep) {
      if (H > kLinStep) fetch_grad(k0);
      __syncthreads();
#pragma unroll
      for (int l = 0; l < kChunks; ++l) {
        const int c = t + 256 * l, row = c >> 3;
        bf16x8 pl[P];
        planes_of(wreg[l], pl);
#pragma unroll
        for (int q = 0; q < P; ++q)
          *reinterpret_cast<bf16x8*>(lds + (q * kLinStep + row) * 128 + (((c & 7) ^ spread_128(row)) << 4)) = pl[q];
      }
      __syncthreads();
      if (k0 + kLinStep < H) fetch_weight(k0 + kLinStep, f0);
      else if (tile + 1 < tile1) fetch_weight(0, f0 + kLinStep);
#pragma unroll
      for (int s = 0; s < kKept; ++s) {
        if (k0 + 16 * s >= H) break;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // units 16 s + 4 half .. and eight further on, features 32 j ..
          const int row = 16 * s + 4 * half + ((lane & 15) >> 2);
          const int c = 4 * j + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), inner = (lane & 1) * 8;
          typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
          bf16x8 fa[P];
#pragma unroll
          for (int q = 0; q < P; ++q) {
            const char* at = lds + (q * kLinStep + row) * 128;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + ((c ^ spread_128(row)) << 4) + inner));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(at + 8 * 128 + ((c ^ spread_128(row + 8)) << 4) + inner));
            __builtin_memcpy(&fa[q], &lo, 8);
            __builtin_memcpy(reinterpret_cast<char*>(&fa[q]) + 8, &hi, 8);
          }
          multiply_planes<P>(fa, fb[s], acc[j]);
        }
      }
    }
    // x > 0 is false where the code's sign bit is set
    const auto result = [&](int j, int e) {
      const float d = acc[j][e];
      return narrow<T>((signs[j][e >> 2] >> (8 * (e & 3) + 7)) & 1u ? (slope == 0.f ? 0.f : slope * d) : d);
    };
    // whole 128-byte pieces of a row at a time, by way of LDS: as the lanes hold them, four features of
    // a row each, dx would leave in pieces of 32 bytes, or 2 where rows are not aligned
    char* const mine = turned[wave];
#pragma unroll
    for (int jj = 0; jj < 2; jj += kJoined) {
#pragma unroll
      for (int j = jj; j < jj + kJoined; ++j)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const T v[4] = {result(j, e), result(j, e + 1), result(j, e + 2), result(j, e + 3)};
          typedef unsigned Word __attribute__((ext_vector_type(sizeof(T))));
          Word word;
          __builtin_memcpy(&word, &v, sizeof(word));
          const int row = lane & 31, byte = (32 * (j - jj) + block_row(e, lane)) * int(sizeof(T));
          *reinterpret_cast<Word*>(mine + row * 128 + (((byte >> 4) ^ ((row >> 1) & 7)) << 4) + (byte & 15)) = word;
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      T* const out = dx + first * lddx + f0 + 32 * jj;
      if (f0 + kLinStep <= F) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 8 * i + (lane >> 3), c = lane & 7;
          const u32x4 word = *reinterpret_cast<const u32x4*>(mine + row * 128 + ((c ^ ((row >> 1) & 7)) << 4));
          if (first + row < n) __builtin_memcpy(reinterpret_cast<char*>(out + row * lddx) + 16 * c, &word, 16);
        }
      } else {
        constexpr int kAcross = 128 / sizeof(T);               // lanes along a row
#pragma unroll 8
        for (int i = 0; i < 32 * kAcross / 64; ++i) {
          const int row = i * (64 / kAcross) + lane / kAcross, f = lane % kAcross, byte = f * int(sizeof(T));
          const T v = *reinterpret_cast<const T*>(mine + row * 128 + (((byte >> 4) ^ ((row >> 1) & 7)) << 4) + (byte & 15));
          if (first + row < n && f0 + 32 * jj + f < F) out[row * lddx + f] = v;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

struct GradPlan {
  int bh, bf, tiles_h, tiles_f, chunks;
  int64_t chunk_rows;
};

// Workgroups that run at once on an XCD: two on each of its 32 compute units.  A workgroup more than
// that starts when the others end: 232965 x 602 x 128 units (3 tiles) with 66 on two of the XCDs 180 us,
// with 63 on each 137 us; with 32 165 us, with 96 147 us.
constexpr int kSlots = 64;

GradPlan grad_plan(int64_t n, int64_t F, int64_t H) {
  GradPlan p;
  p.bh = H <= 32 ? 32 : H <= 64 ? 64 : 128;
  p.bf = 256;
  p.tiles_h = int((H + p.bh - 1) / p.bh);
  p.tiles_f = int((F + p.bf - 1) / p.bf);
  const int64_t steps = (n + kRowsStep - 1) / kRowsStep;
  const int64_t tiles = int64_t(p.tiles_h) * p.tiles_f;
  int64_t want = tiles < 512 ? 512 / tiles : 1;
  if (tiles <= kSlots) {                         // whole chunks for every XCD, filling its slots 1 to 4 times over
    int per_xcd = 1;
    double best = 0.;
    for (int rounds = 1; rounds <= 4; ++rounds) {
      const int c = int(rounds * kSlots / tiles);
      const double used = double(c * tiles) / (rounds * kSlots);
      if (used > best + 0.02) best = used, per_xcd = c;
    }
    want = 8 * int64_t(per_xcd);
  }
  if (want > steps) want = steps;
  int64_t per = (steps + want - 1) / want;
  if (per < 1) per = 1;
  p.chunk_rows = per * kRowsStep;
  p.chunks = int((n + p.chunk_rows - 1) / p.chunk_rows);
  if (p.chunks < 1) p.chunks = 1;
  return p;
}

int check_saved(int dtype, int64_t n, int64_t F, float slope) {
  using sgnn::fail;
  if (dtype != SGNN_F32 && dtype != SGNN_BF16) return fail(SGNN_ERR_INVALID, "unknown element type");
  if (n < 0 || F <= 0) return fail(SGNN_ERR_INVALID, "need n >= 0 and F > 0");
  if (F > (int64_t(1) << 24)) return fail(SGNN_ERR_UNSUPPORTED, "more than 2^24 features");
  if (n > (int64_t(1) << 31) * 64) return fail(SGNN_ERR_UNSUPPORTED, "too many rows");
  if (!(slope >= 0.f) || !(slope <= 3.4e38f)) return fail(SGNN_ERR_INVALID, "the activation's slope must be finite and not negative");
  return SGNN_OK;
}

struct EltGrid { int rows, per_row; unsigned blocks; };
int elt_grid(int64_t n, int64_t F, int elems, EltGrid* g) {
  const int64_t per_row = (F + kGroup - 1) / kGroup * (kGroup / elems);
  // about four trips of the workgroup: enough loads in flight, and n * F / 4096 workgroups to spread
  int64_t rows = (4 * kEltThreads) / per_row;
  if (rows < 1) rows = 1;
  const int64_t blocks = (n + rows - 1) / rows;
  if (blocks > 0xffffff) return sgnn::fail(SGNN_ERR_UNSUPPORTED, "too many rows for one launch");
  *g = {int(rows), int(per_row), unsigned(blocks)};
  return SGNN_OK;
}

template <typename T>
int launch_weight_grad(const GradPlan& p, int64_t n, int64_t F, int64_t H, const uint8_t* codes, const uint8_t* steps,
                       float slope, const void* grad, int64_t ldg, void* dW, int64_t lddw, float* partial,
                       hipStream_t st) {
  const T* g = static_cast<const T*>(grad);
  T* out = static_cast<T*>(dW);
  const unsigned blocks = unsigned((p.chunks < 8 ? p.chunks : (p.chunks + 7) / 8 * 8) * p.tiles_f * p.tiles_h);
#define SGNN_WG8(BH, BF, WH, WF)                                                                                  \
  hipLaunchKernelGGL((k_weight_grad8<T, BH, BF, WH, WF>), dim3(blocks), dim3(64 * WH * WF), 0, st, n, int(F),     \
                     int(H), codes, steps, slope, g, ldg, p.chunk_rows, p.chunks, p.tiles_f, p.tiles_h, out,       \
                     lddw, partial)
  if (p.bh == 32) SGNN_WG8(32, 256, 1, 4);
  else if (p.bh == 64) SGNN_WG8(64, 256, 1, 4);
  else SGNN_WG8(128, 256, 2, 4);
#undef SGNN_WG8
  HIP_TRY(hipGetLastError());
  if (p.chunks > 1) {
    const int64_t total = F * H;
    hipLaunchKernelGGL((k_weight_grad_sum8<T>), dim3(unsigned((total + 63) / 64)), dim3(256), 0, st, int(F), total,
                       p.chunks, partial, out, lddw);
    HIP_TRY(hipGetLastError());
  }
  return SGNN_OK;
}

}  // namespace

extern "C" int sgnn_save8(int dtype, int64_t n, int64_t F, const void* x, int64_t ldx, float slope, void* codes,
                          void* steps, void* stream) {
  using sgnn::fail;
  if (int rc = check_saved(dtype, n, F, slope)) return rc;
  if (ldx < F) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (n == 0) return SGNN_OK;
  if (!x || !codes || !steps) return fail(SGNN_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16) return fail(SGNN_ERR_INVALID, "codes must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  EltGrid g;
  uint8_t* q = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(steps);
  if (dtype == SGNN_F32) {
    if (int rc = elt_grid(n, F, Lane<float>::kElems, &g)) return rc;
    hipLaunchKernelGGL((k_save8<float>), dim3(g.blocks), dim3(kEltThreads), 0, st, n, int(F),
                       static_cast<const float*>(x), ldx, slope, g.rows, g.per_row, q, s);
  } else {
    if (int rc = elt_grid(n, F, Lane<Bf16>::kElems, &g)) return rc;
    hipLaunchKernelGGL((k_save8<Bf16>), dim3(g.blocks), dim3(kEltThreads), 0, st, n, int(F),
                       static_cast<const Bf16*>(x), ldx, slope, g.rows, g.per_row, q, s);
  }
  HIP_TRY(hipGetLastError());
  return SGNN_OK;
}

namespace {
int check_linear(int dtype, int64_t n, int64_t F, int64_t H, float slope, const void* weight, int64_t ldw) {
  using sgnn::fail;
  if (int rc = check_saved(dtype, n, F, slope)) return rc;
  if (H <= 0) return fail(SGNN_ERR_INVALID, "need H > 0");
  if (H > (int64_t(1) << 20)) return fail(SGNN_ERR_UNSUPPORTED, "more than 2^20 units");
  if ((n + 127) / 128 > 0xffffff) return fail(SGNN_ERR_UNSUPPORTED, "too many rows for one launch");
  if (ldw < F) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (n > 0 && !weight) return fail(SGNN_ERR_INVALID, "null pointer");
  return SGNN_OK;
}

template <typename T>
int launch_linear(int64_t n, int64_t F, int64_t H, const void* x, int64_t ldx, const void* w, int64_t ldw, float slope,
                  uint8_t* codes, uint8_t* steps, void* y, int64_t ldy, hipStream_t st) {
#define SGNN_LIN8_AS(NB, SPLIT, MOVED)                                                                               \
  hipLaunchKernelGGL((k_linear8<T, NB, SPLIT, MOVED>), dim3(unsigned((n + (SPLIT ? 31 : 127)) / (SPLIT ? 32 : 128)),        \
                                                     unsigned((H + 32 * NB - 1) / (32 * NB))),                       \
                     dim3(256), 0, st, n, int(F), int(H), static_cast<const T*>(x), ldx, static_cast<const T*>(w),   \
                     ldw, slope, codes, steps, static_cast<T*>(y), ldy)
#define SGNN_LIN8(NB, SPLIT)                                                                                         \
  if (sizeof(T) == 2 && slope != 0.f && slope != 1.f) SGNN_LIN8_AS(NB, SPLIT, (sizeof(T) == 2));                     \
  else SGNN_LIN8_AS(NB, SPLIT, false)
  // Few rows are bound by the wait for one load after the other along the features, which four
  // wavefronts share; more rows than fill the card gain nothing by it.  fp32, together / split, at 8192,
  // 16384 and 32768 rows: 1433 features, 16 units 64 / 24, 64 / 32, 67 / 62 us; 500, 64: 33 / 15, 35 / 27,
  // 37 / 51 us; 602, 128 (two workgroups for the same rows): 51 / 30, 53 / 57, 55 / 108 us.  A single step
  // has nothing to share.
  const bool split = F > kLinStep && (n + 31) / 32 * ((H + 63) / 64) <= 512;
  if (H <= 32 && split) { SGNN_LIN8(1, true); }
  else if (H <= 32) { SGNN_LIN8(1, false); }
  else if (split) { SGNN_LIN8(2, true); }
  else if (H <= 64) { SGNN_LIN8(2, false); }
  else { SGNN_LIN8(4, false); }
#undef SGNN_LIN8_AS
#undef SGNN_LIN8
  HIP_TRY(hipGetLastError());
  return SGNN_OK;
}

template <typename T>
int launch_linear_grad(int64_t n, int64_t F, int64_t H, const void* g, int64_t ldg, const void* w, int64_t ldw,
                       float slope, const uint8_t* codes, void* dx, int64_t lddx, hipStream_t st) {
  const int64_t blocks = (n + 127) / 128, tiles = (F + kLinStep - 1) / kLinStep;
  // Few rows: features over several workgroups, each of which reads its rows of grad again.  Aimed at
  // 1024 workgroups; at 2048 the 232965 rows (1821 workgroups by themselves) take 10 us longer.
  int64_t across = (1024 + blocks - 1) / blocks;
  if (across > tiles) across = tiles;
  hipLaunchKernelGGL((k_linear_grad8<T>), dim3(unsigned(blocks), unsigned(across)), dim3(256), 0, st, n, int(F), int(H),
                     static_cast<const T*>(g), ldg, static_cast<const T*>(w), ldw, slope, codes, static_cast<T*>(dx),
                     lddx);
  HIP_TRY(hipGetLastError());
  return SGNN_OK;
}
}  // namespace

extern "C" int sgnn_saved8_linear(int dtype, int64_t n, int64_t F, int64_t H, const void* x, int64_t ldx,
                                  const void* weight, int64_t ldw, float slope, void* codes, void* steps, void* y,
                                  int64_t ldy, void* stream) {
  using sgnn::fail;
  if (int rc = check_linear(dtype, n, F, H, slope, weight, ldw)) return rc;
  if (ldx < F || ldy < H) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (n == 0) return SGNN_OK;
  if (!x || !y || (codes == nullptr) != (steps == nullptr)) return fail(SGNN_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16) return fail(SGNN_ERR_INVALID, "codes must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint8_t* q = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(steps);
  if (dtype == SGNN_F32) return launch_linear<float>(n, F, H, x, ldx, weight, ldw, slope, q, s, y, ldy, st);
  return launch_linear<Bf16>(n, F, H, x, ldx, weight, ldw, slope, q, s, y, ldy, st);
}

extern "C" int sgnn_saved8_linear_grad(int dtype, int64_t n, int64_t F, int64_t H, const void* codes, float slope,
                                       const void* grad, int64_t ldg, const void* weight, int64_t ldw, void* dx,
                                       int64_t lddx, void* stream) {
  using sgnn::fail;
  if (int rc = check_linear(dtype, n, F, H, slope, weight, ldw)) return rc;
  if (ldg < H || lddx < F) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (n == 0) return SGNN_OK;
  if (!grad || !dx || (!codes && slope != 1.f)) return fail(SGNN_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16) return fail(SGNN_ERR_INVALID, "codes must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint8_t* q = static_cast<const uint8_t*>(codes);
  if (dtype == SGNN_F32) return launch_linear_grad<float>(n, F, H, grad, ldg, weight, ldw, slope, q, dx, lddx, st);
  return launch_linear_grad<Bf16>(n, F, H, grad, ldg, weight, ldw, slope, q, dx, lddx, st);
}

extern "C" int sgnn_restore8(int dtype, int64_t n, int64_t F, const void* codes, const void* steps, float slope,
                             void* out, int64_t ldo, void* stream) {
  using sgnn::fail;
  if (int rc = check_saved(dtype, n, F, slope)) return rc;
  if (ldo < F) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (n == 0) return SGNN_OK;
  if (!codes || !steps || !out) return fail(SGNN_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16) return fail(SGNN_ERR_INVALID, "codes must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  EltGrid g;
  const uint8_t* q = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(steps);
  if (dtype == SGNN_F32) {
    if (int rc = elt_grid(n, F, Lane<float>::kElems, &g)) return rc;
    hipLaunchKernelGGL((k_restore8<float>), dim3(g.blocks), dim3(kEltThreads), 0, st, n, int(F), q, s, slope, g.rows,
                       g.per_row, static_cast<float*>(out), ldo);
  } else {
    if (int rc = elt_grid(n, F, Lane<Bf16>::kElems, &g)) return rc;
    hipLaunchKernelGGL((k_restore8<Bf16>), dim3(g.blocks), dim3(kEltThreads), 0, st, n, int(F), q, s, slope, g.rows,
                       g.per_row, static_cast<Bf16*>(out), ldo);
  }
  HIP_TRY(hipGetLastError());
  return SGNN_OK;
}

extern "C" int sgnn_saved8_input_grad(int dtype, int64_t n, int64_t F, const void* codes, float slope,
                                      const void* grad, int64_t ldg, void* dx, int64_t lddx, void* stream) {
  using sgnn::fail;
  if (int rc = check_saved(dtype, n, F, slope)) return rc;
  if (slope == 1.f) return fail(SGNN_ERR_INVALID, "codes of slope 1 hold no sign of the input");
  if (ldg < F || lddx < F) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (n == 0) return SGNN_OK;
  if (!codes || !grad || !dx) return fail(SGNN_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16) return fail(SGNN_ERR_INVALID, "codes must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  EltGrid g;
  const uint8_t* q = static_cast<const uint8_t*>(codes);
  if (dtype == SGNN_F32) {
    if (int rc = elt_grid(n, F, Lane<float>::kElems, &g)) return rc;
    hipLaunchKernelGGL((k_input_grad8<float>), dim3(g.blocks), dim3(kEltThreads), 0, st, n, int(F), q, slope, g.rows,
                       g.per_row, static_cast<const float*>(grad), ldg,
                       static_cast<float*>(dx), lddx);
  } else {
    if (int rc = elt_grid(n, F, Lane<Bf16>::kElems, &g)) return rc;
    hipLaunchKernelGGL((k_input_grad8<Bf16>), dim3(g.blocks), dim3(kEltThreads), 0, st, n, int(F), q, slope, g.rows,
                       g.per_row, static_cast<const Bf16*>(grad), ldg,
                       static_cast<Bf16*>(dx), lddx);
  }
  HIP_TRY(hipGetLastError());
  return SGNN_OK;
}

extern "C" size_t sgnn_saved8_weight_grad_workspace_bytes(int64_t n, int64_t F, int64_t H) {
  if (n <= 0 || F <= 0 || H <= 0) return 0;
  const GradPlan p = grad_plan(n, F, H);
  return p.chunks > 1 ? size_t(p.chunks) * size_t(F) * size_t(H) * sizeof(float) : 0;
}

extern "C" int sgnn_saved8_weight_grad(int dtype, int64_t n, int64_t F, int64_t H, const void* codes,
                                       const void* steps, float slope, const void* grad, int64_t ldg, void* dW,
                                       int64_t lddw, void* workspace, size_t workspace_bytes, void* stream) {
  using sgnn::fail;
  if (int rc = check_saved(dtype, n, F, slope)) return rc;
  if (n == 0 || H <= 0) return fail(SGNN_ERR_INVALID, "need n > 0 and H > 0");
  if (H > (int64_t(1) << 24) || F * H > (int64_t(1) << 31)) return fail(SGNN_ERR_UNSUPPORTED, "weight too large");
  if (ldg < H || lddw < F) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (!codes || !steps || !grad || !dW) return fail(SGNN_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 16) return fail(SGNN_ERR_INVALID, "codes must be 16-byte aligned");
  if (workspace_bytes < sgnn_saved8_weight_grad_workspace_bytes(n, F, H))
    return fail(SGNN_ERR_WORKSPACE, "weight-gradient workspace too small");
  const GradPlan p = grad_plan(n, F, H);
  if (p.chunks > 1 && !workspace) return fail(SGNN_ERR_INVALID, "null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint8_t* q = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(steps);
  float* part = static_cast<float*>(workspace);
  if (dtype == SGNN_F32) return launch_weight_grad<float>(p, n, F, H, q, s, slope, grad, ldg, dW, lddw, part, st);
  return launch_weight_grad<Bf16>(p, n, F, H, q, s, slope, grad, ldg, dW, lddw, part, st);
}
