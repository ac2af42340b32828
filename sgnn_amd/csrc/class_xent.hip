// Softmax cross-entropy of x . weight^T over many classes, and its gradients, without the logits.
//
//   z = x . weight^T (B x V),  loss_b = log sum_v exp(z_bv) - z_b,y(b),
//   dz_bv = g_b (exp(z_bv) / sum_v exp(z_bv) - [v = y(b)]),  dx = dz . weight,  dweight = dz^T . x
//
// The forward pass runs over the classes once and keeps a running maximum and sum per row; the
// backward pass forms the logits again, a piece of the classes at a time, writes that piece of dz
// and multiplies it from either side.
//
// All four products run on the bf16 matrix instructions (tile_product.h): bf16 operands as they
// are, fp32 ones as three bf16 numbers each.  dz of bf16 operands is rounded to bf16 there
// (relative 2^-8 per element at most, the half step that each result is rounded by, too), but for the
// label's element, the largest of its row and of nearly every class: that keeps 16 bits or more in both
// gradients.  4096 x 256 against 50000 classes: dweight is off by 2.3e-5 of its norm before its own
// rounding, with that element rounded like the others by 2.1e-4.
//
// Bound by the matrix unit.  2048 x 602 against 10007 classes in fp32 (24.7 GFLOP a product, six bf16
// products each): statistics 156 us, dz 148, the gradients' products 322 together, that is 0.92 to 1.00
// PFLOP/s of the 1.04 (8192^3) to 1.34 (16384^3) that a library product of bf16 matrices reaches.
#include "tile_product.h"

namespace {

__device__ __forceinline__ float exp2_raw(float v) { return __builtin_amdgcn_exp2f(v); }   // 0 below 2^-126

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ int64_t label_of(int64_t b, const int64_t* labels, const int64_t* idx, int64_t n_labels,
                                            int64_t V) {
  const int64_t at = idx ? idx[b] : b;
  const int64_t y = (at >= 0 && at < n_labels) ? labels[at] : -1;
  return (y >= 0 && y < V) ? y : -1;
}

// ------------------------------------------------------------------ operands
struct Labels {
  const int64_t *labels, *idx;
  int64_t n_labels, V;
  bool all;                                      // rows without a class are rows like the others (fp32)
};
// does row b (of B or more) add to the gradients?
__device__ __forceinline__ bool counts(int64_t b, int64_t B, const Labels& of) {
  return b < B && (of.all || label_of(b, of.labels, of.idx, of.n_labels, of.V) >= 0);
}

struct RowStat { float m, s, picked; };          // what the backward pass needs of a row; picked = the label's logit

// What the gradients of the kernels with rows in registers need of a row: p = 2^((z - top) log2 e - shift)
// with top = 0 but for rows whose logits are so large that the rounding of shift would be felt (2^12: by
// 2^-12, a bf16 half step being 2^-8); shift = infinity without a class; its factor, its label, and what
// the label's element of dz adds in dx beyond its rounded probability.
constexpr float kLargeLogit = 4096.f;
struct RowConst {
  float *shift, *top, *factor, *rest;
  int* label;
};
struct Rows {
  int64_t B;
  const RowStat* stats;                          // NULL: no more than the label is wanted, or nothing
  const float *grad, *share;
  RowConst out;
};

__device__ __forceinline__ void prepare_row(const Rows& rows, int64_t b, const Labels& of) {
  const int64_t y = b < rows.B ? label_of(b, of.labels, of.idx, of.n_labels, of.V) : -1;
  const RowStat st = y >= 0 ? rows.stats[b] : RowStat{INFINITY, 1.f, 0.f};
  const bool large = y >= 0 && !(fabsf(st.m) <= kLargeLogit);
  const float top = large ? st.m : 0.f, shift = large ? log2f(st.s) : fmaf(st.m, kLog2e, log2f(st.s));
  const float p = exp2_raw(fmaf(st.picked - top, kLog2e, -shift));
  rows.out.shift[b] = shift;
  rows.out.top[b] = top;
  rows.out.factor[b] = y < 0 ? 0.f : rows.share ? rows.grad[0] * rows.share[0] : rows.grad[b];
  rows.out.rest[b] = (p - widen(Bf16{to_bf16(p)})) - 1.f;
  rows.out.label[b] = int(y);
}

// in[r][d] at r * sr + d * sd  ->  out[r][Dp], columns D .. Dp zero.  Rows of x without a class
// become zeros, so that whatever a padded row holds (NaN too) reaches no gradient.
struct Source {
  const void* in;
  int64_t rows, sr, sd;
  void* out;
  int64_t blocks;          // workgroups it takes: one for 64 x 64 elements
};

// x and the weight in one launch, and with `rows` what the gradients need of each row, up to a whole
// number of 64.  Rows that are contiguous go straight through registers, eight
// elements a lane; a weight stored by feature goes through a tile in LDS.
template <typename T>
__global__ __launch_bounds__(256) void k_class_operands(int D, int Dp, Source first, Source second, Labels of, Rows rows) {
  __shared__ T tile[64][sizeof(T) == 4 ? 65 : 66];
  const bool is_x = int64_t(blockIdx.x) < first.blocks;
  const Source src = is_x ? first : second;
  const int64_t block = is_x ? blockIdx.x : blockIdx.x - first.blocks;
  const int across = Dp / 64;
  const int64_t r0 = block / across * 64;
  const int d0 = int(block % across) * 64, t = threadIdx.x;
  const T* in = static_cast<const T*>(src.in);
  if (is_x && d0 == 0 && t < 64) {
    if (rows.stats) prepare_row(rows, r0 + t, of);
    else if (rows.out.label && r0 + t < rows.B) rows.out.label[r0 + t] = int(label_of(r0 + t, of.labels, of.idx, of.n_labels, of.V));
  }
  const auto live = [&](int64_t r) {
    return is_x ? counts(r, src.rows, of) : r < src.rows;
  };
  if (src.sd != 1) {
    for (int i = t; i < 64 * 64; i += 256) {
      const int lr = i & 63, ld = i >> 6;
      const int64_t r = r0 + lr;
      const int d = d0 + ld;
      tile[lr][ld] = (d < D && live(r)) ? in[r * src.sr + d * src.sd] : T{};
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = t; i < 64 * 8; i += 256) {
    const int lr = i >> 3, c = (i & 7) * 8, d = d0 + c;
    const int64_t r = r0 + lr;
    if (r >= src.rows) continue;
    T v[8];
    if (src.sd != 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile[lr][c + e];
    } else if (!live(r)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = T{};
    } else if (d + 8 <= D) {
      __builtin_memcpy(&v, in + r * src.sr + d, sizeof(v));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = d + e < D ? in[r * src.sr + d + e] : T{};
    }
    u32x4 w[sizeof(v) / 16];
    __builtin_memcpy(&w, &v, sizeof(v));
    u32x4* dst = reinterpret_cast<u32x4*>(static_cast<T*>(src.out) + r * Dp + d);
#pragma unroll
    for (int q = 0; q < int(sizeof(v) / 16); ++q) dst[q] = w[q];
  }
}

// ------------------------------------------------------------------ forward
// (m, s): m = the largest logit, s = sum of 2^((z - m) log2 e).  While everything is -inf the sum
// stays 0; a NaN never becomes the maximum but makes the sum NaN.
__device__ __forceinline__ void join_stats(float& m, float& s, float om, float os) {
  const float top = fmaxf(m, om), ref = top == -INFINITY ? 0.f : top;
  s = s * exp2_raw((m - ref) * kLog2e) + os * exp2_raw((om - ref) * kLog2e);
  m = top;
}

// One multiply-add per logit: 2^(z log2 e - c) with c = ref * log2 e rounded, and what the rounding
// took put right in the sum.  Where that could leave the exponent's range (logits of millions) the
// reference is taken off the logits first.
struct Reference { float c, fix; };
constexpr float kFarLogit = 1048576.f;
template <int N>
__device__ __forceinline__ Reference reference_of(f32x16 (&z)[N], float ref) {
  const bool far = !(fabsf(ref) < kFarLogit);
  if (__any(far)) {
    const float off = far ? ref : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) z[i][e] -= off;
  }
  const float c = far ? 0.f : ref * kLog2e;
  return {c, far ? 1.f : exp2_raw(-fmaf(ref, kLog2e, -c))};
}
template <int N>
__device__ __forceinline__ float largest(const f32x16 (&z)[N]) {
  float top = z[0][0];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 2) top = fmaxf(fmaxf(z[i][e], z[i][e + 1]), top);
  return top;
}
template <int N>
__device__ __forceinline__ void accumulate(f32x16 (&z)[N], float& m, float& s) {
  const float top = fmaxf(largest(z), m), ref = top == -INFINITY ? 0.f : top;
  const Reference at = reference_of(z, ref);
  float sum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e)
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += exp2_raw(fmaf(z[i][e], kLog2e, -at.c));
#pragma unroll
  for (int i = 1; i < N; ++i) sum[0] += sum[i];
  s = s * exp2_raw((m - ref) * kLog2e) + sum[0] * at.fix;
  m = top;
}

// A workgroup takes 128 rows of x and a range of the classes, 128 at a time.  The tile is formed
// as classes x rows, so that a lane holds 32 classes of each of two rows and its running maximum
// and sum need no other lane until the end.  part[row][split][half] = (m, s).
template <typename T>
__global__ __launch_bounds__(kThreads) void k_class_stats(int64_t B, int64_t V, int Dp, Operand<T> x, Operand<T> w,
                                                          const int64_t* __restrict__ labels,
                                                          const int64_t* __restrict__ idx, int64_t n_labels,
                                                          int64_t tiles_v, int splits, float2* __restrict__ part,
                                                          float* __restrict__ picked) {
  __shared__ __align__(128) char lds[kProductLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wv = (wave >> 1) * 64, wb = (wave & 1) * 64;
  const int split = blockIdx.x % splits;
  const int64_t b0 = int64_t(blockIdx.x / splits) * kTile;
  const int64_t t0 = tiles_v * split / splits, t1 = tiles_v * (split + 1) / splits;
  float top[2], sum[2];
  int64_t y[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t b = b0 + wb + 32 * j + (lane & 31);
    top[j] = -INFINITY;
    sum[j] = 0.f;
    y[j] = b < B ? label_of(b, labels, idx, n_labels, V) : -1;
  }
  for (int64_t t = t0; t < t1; ++t) {
    Tile acc;
    clear(acc);
    multiply<T, true, true>(w, t * kTile, x, b0, 0, Dp, lds, acc);
    const int64_t vw = t * kTile + wv;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (__any(y[j] >= vw && y[j] < vw + 64)) {       // one tile in V / 64 holds a row's label
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (vw + 32 * i + block_row(e, lane) == y[j]) picked[b0 + wb + 32 * j + (lane & 31)] = acc[i][j][e];
      }
      if (vw + 64 > V) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (vw + 32 * i + block_row(e, lane) >= V) acc[i][j][e] = -INFINITY;
      }
      f32x16 z[2] = {acc[0][j], acc[1][j]};
      accumulate(z, top[j], sum[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float om = __shfl_xor(top[j], 32), os = __shfl_xor(sum[j], 32);
    join_stats(top[j], sum[j], om, os);
    const int64_t b = b0 + wb + 32 * j + (lane & 31);
    if (lane < 32 && b < B) part[b * (2 * splits) + split * 2 + (wave >> 1)] = make_float2(top[j], sum[j]);
  }
}

// A row's pieces joined by one wavefront: stats[b], row_loss[b] (0 where the row has no class).
__global__ __launch_bounds__(256) void k_class_rows(int64_t B, int64_t V, int parts, const float2* __restrict__ part,
                                                    const float* __restrict__ picked,
                                                    const int64_t* __restrict__ labels,
                                                    const int64_t* __restrict__ idx, int64_t n_labels,
                                                    RowStat* __restrict__ stats, float* __restrict__ row_loss) {
  const int lane = threadIdx.x & 63;
  const int64_t b = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (b >= B) return;
  float m = -INFINITY, s = 0.f;
  for (int q = lane; q < parts; q += 64) {
    const float2 o = part[b * parts + q];
    join_stats(m, s, o.x, o.y);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const float om = __shfl_xor(m, off), os = __shfl_xor(s, off);
    join_stats(m, s, om, os);
  }
  if (lane == 0) {
    const bool live = label_of(b, labels, idx, n_labels, V) >= 0;
    const float zy = live ? picked[b] : 0.f;
    stats[b] = RowStat{m, s, zy};
    row_loss[b] = live ? (m - zy) + log2f(s) * kLn2 : 0.f;
  }
}

// loss[0] = mean loss of the counted rows (0 if there are none), share[0] = 1 / their number.
__global__ __launch_bounds__(1024) void k_class_mean(int64_t B, Labels of, const float* __restrict__ row_loss,
                                                     float* __restrict__ loss, float* __restrict__ share) {
  __shared__ double s_sum[16];
  __shared__ int64_t s_count[16];
  double sum = 0.0;
  int64_t count = 0;
  for (int64_t b = threadIdx.x; b < B; b += 1024)
    if (counts(b, B, of)) {                      // a row without a class has loss 0
      sum += double(row_loss[b]);
      ++count;
    }
  for (int off = 32; off >= 1; off >>= 1) {
    sum += __shfl_xor(sum, off);
    count += __shfl_xor(count, off);
  }
  if ((threadIdx.x & 63) == 0) {
    s_sum[threadIdx.x >> 6] = sum;
    s_count[threadIdx.x >> 6] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int q = 1; q < 16; ++q) {
      sum += s_sum[q];
      count += s_count[q];
    }
    loss[0] = count ? float(sum / double(count)) : 0.f;
    share[0] = count ? float(1.0 / double(count)) : 0.f;
  }
}

// ------------------------------------------------------------------ backward
// dz of the classes v0 .. v0 + 128 * tiles and all rows, [Bp][ldz]; rows and
// classes beyond the last are 0.  `grad` NULL leaves the mean's factor to the gradients' last step.
// The label's element dominates a row, and often its class, and is the one whose rounding to bf16 would be
// felt: what it loses is kept in rest[b] and joins both gradients in 32 bits.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_class_dz(int64_t B, int Dp, Operand<T> x, Operand<T> w, Labels of,
                                                       const RowStat* __restrict__ stats,
                                                       const float* __restrict__ grad, float* __restrict__ rest,
                                                       int64_t v0, int tiles, T* __restrict__ dz, int64_t ldz) {
  __shared__ __align__(128) char lds[kProductLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wv = (wave >> 1) * 64, wb = (wave & 1) * 64;
  const int64_t V = of.V, vt = v0 + int64_t(blockIdx.x % tiles) * kTile;
  const int64_t b0 = int64_t(blockIdx.x / tiles) * kTile;
  Tile acc;
  clear(acc);
  multiply<T, true, true>(w, vt, x, b0, 0, Dp, lds, acc);
  const int64_t vw = vt + wv;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t b = b0 + wb + 32 * j + (lane & 31);
    const int64_t y = b < B ? label_of(b, of.labels, of.idx, of.n_labels, V) : -1;
    const bool live = y >= 0 || (of.all && b < B);
    const float g = live ? (grad ? grad[b] : 1.f) : 0.f;
    const RowStat st = b < B ? stats[b] : RowStat{0.f, 1.f, 0.f};
    const float scale = g / st.s;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = exp2_raw((acc[i][j][e] - st.m) * kLog2e) * scale;
    if (__any(y >= vw && y < vw + 64)) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (vw + 32 * i + block_row(e, lane) == y) {
            const float d = acc[i][j][e] - g;
            acc[i][j][e] = d;
            if constexpr (sizeof(T) == 2) rest[b] = d - widen(Bf16{to_bf16(d)});
          }
    }
    if (vw + 64 > V || __any(!live)) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!live || vw + 32 * i + block_row(e, lane) >= V) acc[i][j][e] = 0.f;
    }
  }
  T* out = dz + b0 * ldz + (vt - v0);
  if constexpr (sizeof(T) == 4) {                  // four classes a lane: whole 16 bytes
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<f32x4*>(out + (wb + 32 * j + (lane & 31)) * ldz + wv + 32 * i + block_row(e, lane)) =
              f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
  } else {
    constexpr int kRow = kTile * 2 + 16;           // bytes of a staged row of dz
    static_assert(kTile * kRow <= kProductLds, "a tile of dz fits the product's stages");
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          uint16_t four[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) four[q] = to_bf16(acc[i][j][e + q]);
          u32x2 u;
          __builtin_memcpy(&u, &four, 8);
          *reinterpret_cast<u32x2*>(lds + (wb + 32 * j + (lane & 31)) * kRow + (wv + 32 * i + block_row(e, lane)) * 2) = u;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < kTile * kTile / 8; c += kThreads) {
      const int row = c >> 4, col = (c & 15) * 8;
      *reinterpret_cast<u32x4*>(out + row * ldz + col) = *reinterpret_cast<const u32x4*>(lds + row * kRow + col * 2);
    }
  }
}

// Where a product that is one share goes at once: row m of the result to out + m * stride, times the
// mean's factor if there is one.
template <typename T>
struct Direct {
  T* out;                                        // NULL: to the shares
  int64_t stride, rows;
  int cols;
  const float *grad, *share;
};

// C[m][n] += or = A . B over a workgroup's share of the reduction, 32 bits, one buffer per share:
// out[split][Mp][Np]; or, where there is one share, the result itself.
template <typename T>
struct Product {
  Operand<T> a, b;
  int64_t K;
  int tiles_n, splits, add;
  float* out;
  int64_t plane, ldo;
  Direct<T> direct;
  unsigned blocks;                               // workgroups it takes: tiles_m * splits * tiles_n
  // dweight in bf16: what the labels' elements lost by their rounding, `rest` of each of `rows` rows, at
  // row label - first of the result
  const float* rest;
  const int* label;
  int64_t rows, first;
};

// acc[m][n] += rest[b] * x[b][n] for the rows b whose label is class m, the element of dz that is nearly
// all of a class's gradient, so that it keeps 16 bits: step by step of the reduction, whose rows of x are
// in LDS.  A step's labels and rests are under way while the step before is multiplied.  Costs 4096 x 512
// against 50000 classes 20 us of 270, 16384 x 512 against 500 (a label in every sixteen rows) 15 of 145 in all.
struct RestOfLabels {
  const Product<Bf16>& p;
  int64_t m, end;                                // the wavefront's first class; the reduction's end
  int n, lane;                                   // its first column in the tile
  int label = -1, next_label = -1;
  float rest = 0.f, next_rest = 0.f;
  __device__ __forceinline__ void ahead(int64_t k) {
    const int64_t b = k + lane;
    const bool real = b < end && b < p.rows;
    next_label = real ? p.label[b] : -1;
    next_rest = real ? p.rest[b] : 0.f;
  }
  // waited for here, before the next stage's loads are on their way, which would be waited for, too
  __device__ __forceinline__ void landed() {
    asm volatile("" : "+v"(next_label), "+v"(next_rest));
    label = next_label;
    rest = next_rest;
  }
  __device__ __forceinline__ void behind(const char* x, Tile& acc) {
    const int64_t at = label - (p.first + m);
    const int in = label >= 0 && at >= 0 && at < 64 ? int(at) : -1;
    const unsigned mine = to_bf16(rest);
    const uint64_t hits = __ballot(in >= 0);
    if (hits == 0) return;
    for (int kk = 0; kk < Step<Bf16>::kDepth; kk += 16) {
      unsigned h = unsigned(hits >> kk) & 0xffffu;
      if (h == 0) continue;
      // the operand classes x rows of sixteen rows, nearly all of it zeros
      u32x4 rows[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
      for (; h != 0; h &= h - 1) {
        const int r = __builtin_ctz(h);
        const int to = __builtin_amdgcn_readlane(in, kk + r);
        const unsigned value = unsigned(__builtin_amdgcn_readlane(int(mine), kk + r)) << (16 * (r & 1));
        const unsigned here = (to & 31) == (lane & 31) && r >> 3 == lane >> 5 ? value : 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) rows[i][w] |= i == to >> 5 && w == (r & 7) >> 1 ? here : 0u;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        bf16x8 columns;
        read_fragment<false>(x, n + 32 * j, kk, lane, columns);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          bf16x8 a;
          __builtin_memcpy(&a, &rows[i], 16);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, columns, acc[i][j], 0, 0, 0);
        }
      }
    }
  }
};

template <typename T, bool ADEEP>
__device__ __forceinline__ void form_product(const Product<T>& p, unsigned block, char* lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  const int tn = block % unsigned(p.tiles_n), rest = block / unsigned(p.tiles_n);
  const int split = rest % p.splits, tm = rest / p.splits;
  const int64_t m0 = int64_t(tm) * kTile, n0 = int64_t(tn) * kTile;
  const int64_t steps = p.K / Step<T>::kDepth;
  const int64_t k0 = steps * split / p.splits * Step<T>::kDepth, k1 = steps * (split + 1) / p.splits * Step<T>::kDepth;
  Tile acc;
  clear(acc);
  if constexpr (!ADEEP && sizeof(T) == 2) {
    RestOfLabels rest{p, m0 + wm, k1, wn, lane};
    if (k0 < k1) {
      rest.ahead(k0);
      multiply<T, ADEEP, false>(p.a, m0, p.b, n0, k0, k1, lds, acc, rest);
    }
  } else {
    if (k0 < k1) multiply<T, ADEEP, false>(p.a, m0, p.b, n0, k0, k1, lds, acc);
  }
  if (!ADEEP && p.direct.out) {
    const Direct<T>& direct = p.direct;
    const float factor = direct.share ? direct.grad[0] * direct.share[0] : 1.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + wn + 32 * j + (lane & 31);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int64_t m = m0 + wm + 32 * i + block_row(e, lane);
          if (m < direct.rows && n < direct.cols) direct.out[m * direct.stride + n] = narrow<T>(factor * acc[i][j][e]);
        }
      }
    return;
  }
  float* dst = p.out + split * p.plane + (m0 + wm) * p.ldo + n0 + wn + (lane & 31);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (p.add) {                               // all loads before the first sum waits
        float old[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) old[e] = dst[(32 * i + block_row(e, lane)) * p.ldo + 32 * j];
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] += old[e];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) dst[(32 * i + block_row(e, lane)) * p.ldo + 32 * j] = acc[i][j][e];
    }
}

// Both gradients' products in one launch: 512 x 128 against 1000 classes in fp32 11 us, one after the
// other 17 and a launch more; 4096 x 128 against 50000, all of it, 1491 us and 1510.  Not so in bf16 where
// neither leaves half the slots empty: there kernels of their own, in which dx does without dweight's steps
// for the labels (in one kernel they cost it 60 us): 4096 x 512 against 50000 1193 us, in one launch 1229;
// 1777 x 700 against 10007 211 and 215.
template <typename T, bool DX, bool DW>
__global__ __launch_bounds__(kThreads) void k_class_products(Product<T> dx, Product<T> dw) {
  __shared__ __align__(128) char lds[kProductLds];
  if (!DW || (DX && blockIdx.x < dx.blocks)) form_product<T, true>(dx, blockIdx.x, lds);
  else form_product<T, false>(dw, blockIdx.x - dx.blocks, lds);
}

// out[r][d] = factor * (sum over the shares, in order, + rest[r] * weight[y(r)][d]), out at r * sr +
// d * sd; factor = grad[0] * share[0] with `share`, grad[r] with `grad` alone, else 1; `rest` (dx in
// bf16) may be NULL.  With `of` rows that do not count are 0 whatever the weight holds.
template <typename T>
struct Join {
  int64_t R;
  int D, splits;
  const float* in;
  int64_t plane, ldi;
  const float *grad, *share, *rest;
  Labels of;
  const T* weight;
  int64_t sv, sdw;
  T* out;
  int64_t sr, sd;
  unsigned blocks() const { return out ? unsigned((R + 31) / 32 * ((D + 31) / 32)) : 0u; }
};

template <typename T>
__global__ __launch_bounds__(256) void k_class_join(Join<T> first, Join<T> second, unsigned of_first) {
  const bool one = blockIdx.x < of_first;
  const Join<T> j = one ? first : second;
  const unsigned block = one ? blockIdx.x : blockIdx.x - of_first, across = unsigned(j.D + 31) / 32;
  __shared__ float tile[32][33];
  const int64_t r0 = int64_t(block / across) * 32;
  const int t = threadIdx.x, lr = t >> 3, ld = (t & 7) * 4, db = int(block % across) * 32, d = db + ld;
  const int64_t r = r0 + lr;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (r < j.R && d < j.D) {
    const float factor = j.share ? j.grad[0] * j.share[0] : j.grad ? j.grad[r] : 1.f;
    const float* src = j.in + r * j.ldi + d;         // j.ldi is a multiple of 4 and covers d .. d + 3
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int q = 0; q < j.splits; ++q) sum += *reinterpret_cast<const f32x4*>(src + q * j.plane);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = sum[e];
    if (j.of.V) {
      const int64_t y = label_of(r, j.of.labels, j.of.idx, j.of.n_labels, j.of.V);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (y < 0) v[e] = j.of.all ? v[e] : 0.f;
        else if (j.rest && d + e < j.D) v[e] += j.rest[r] * widen(j.weight[y * j.sv + (d + e) * j.sdw]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= factor;
    if (j.sd == 1) {
      T* dst = j.out + r * j.sr + d;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < j.D) dst[e] = narrow<T>(v[e]);
    }
  }
  if (j.sd == 1) return;                         // the whole workgroup
#pragma unroll
  for (int e = 0; e < 4; ++e) tile[lr][ld + e] = v[e];
  __syncthreads();
  for (int i = t; i < 32 * 32; i += 256) {
    const int fr = i & 31, fd = i >> 5, at = db + fd;
    if (r0 + fr < j.R && at < j.D) j.out[(r0 + fr) * j.sr + at * j.sd] = narrow<T>(tile[fr][fd]);
  }
}

// ------------------------------------------------------------------ few rows
// With up to 32 rows the weight is what counts: it is read once forward and twice backward (the
// second time mostly from the last-level cache), as it lies, and its gradient written once.  x
// waits in LDS as bf16 planes; a wavefront takes 32 classes at a time straight from memory into the
// matrix instructions' operand, splitting them in registers.  Both gradients are plain 32-bit
// multiply-adds: 2 * rows of them per element of the weight.  Losses of one row against 100003 classes of
// 256 features in fp32: 26 us, 3.9 TB/s; with 512 or 1024 workgroups or 128 features loaded together 27 to 30.
constexpr int kFewRows = 32;
constexpr int kFewBlocks = 768;                  // workgroups: three per CU
constexpr int kFewSteps = 4;                     // 16-feature steps loaded together

template <int P>
__device__ __forceinline__ int few_at(int p, int row, int chunk, int Dk) {       // byte offset of 8 features in LDS
  return ((p * kFewRows + row) * Dk) * 2 + ((chunk ^ (row & 7)) << 4);
}

// x's rows to LDS, features D .. Dk and rows without a class zero
template <typename T>
__device__ __forceinline__ void few_stage(const Labels& of, int B, int D, int Dk, const T* __restrict__ x, int64_t ldx,
                                          char* lds) {
  constexpr int P = Planes<T>::kCount;
  for (int i = threadIdx.x; i < kFewRows * (Dk / 8); i += kThreads) {
    const int row = i / (Dk / 8), chunk = i - row * (Dk / 8), d = chunk * 8;
    const bool live = counts(row, B, of);
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = live && d + e < D ? x[row * ldx + d + e] : T{};
    bf16x8 pl[P];
    planes_of(v, pl);
#pragma unroll
    for (int q = 0; q < P; ++q) *reinterpret_cast<bf16x8*>(lds + few_at<P>(q, row, chunk, Dk)) = pl[q];
  }
  __syncthreads();
}

// logits of classes v0 .. v0 + 31 (rows of the block) and all 32 rows of x (columns)
template <typename T>
__device__ __forceinline__ f32x16 few_logits(int D, int Dk, int64_t v0, int64_t V, const T* __restrict__ w, int64_t sv,
                                             const char* lds, int lane) {
  const int64_t v = v0 + (lane & 31) < V ? v0 + (lane & 31) : V - 1;
  const int half = lane >> 5;
  constexpr int P = Planes<T>::kCount;
  const T* src = w + v * sv + 8 * half;
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  for (int k = 0; k < Dk; k += 16 * kFewSteps) {
    T raw[kFewSteps][8];
    if (k + 16 * kFewSteps <= D) {
#pragma unroll
      for (int u = 0; u < kFewSteps; ++u) __builtin_memcpy(&raw[u], src + k + 16 * u, sizeof(raw[u]));
    } else {
#pragma unroll
      for (int u = 0; u < kFewSteps; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          raw[u][e] = k + 16 * u + 8 * half + e < D ? src[k + 16 * u + e] : T{};
    }
#pragma unroll
    for (int u = 0; u < kFewSteps; ++u) {
      if (k + 16 * u >= Dk) break;
      bf16x8 a[P], b[P];
      planes_of(raw[u], a);
#pragma unroll
      for (int q = 0; q < P; ++q)
        b[q] = *reinterpret_cast<const bf16x8*>(lds + few_at<P>(q, lane & 31, (k + 16 * u) / 8 + half, Dk));
      multiply_planes(a, b, acc);
    }
  }
  return acc;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_few_stats(int B, int D, int Dk, int64_t V, const T* __restrict__ x,
                                                        int64_t ldx, const T* __restrict__ w, int64_t sv, Labels of,
                                                        float2* __restrict__ part, float* __restrict__ picked) {
  extern __shared__ __align__(128) char few_lds[];
  __shared__ float2 joined[4][kFewRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  few_stage<T>(of, B, D, Dk, x, ldx, few_lds);
  const int b = lane & 31;
  const int64_t y = b < B ? label_of(b, of.labels, of.idx, of.n_labels, of.V) : -1;
  float m = -INFINITY, s = 0.f;
  for (int64_t v0 = (int64_t(blockIdx.x) * 4 + wave) * 32; v0 < V; v0 += int64_t(gridDim.x) * 128) {
    f32x16 z = few_logits<T>(D, Dk, v0, V, w, sv, few_lds, lane);
    if (__any(y >= v0 && y < v0 + 32)) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (v0 + block_row(e, lane) == y) picked[b] = z[e];
    }
    if (v0 + 32 > V) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (v0 + block_row(e, lane) >= V) z[e] = -INFINITY;
    }
    f32x16 one[1] = {z};
    accumulate(one, m, s);
  }
  const float om = __shfl_xor(m, 32), os = __shfl_xor(s, 32);
  join_stats(m, s, om, os);
  if (lane < kFewRows) joined[wave][lane] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x < unsigned(B)) {
    m = -INFINITY;
    s = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) join_stats(m, s, joined[q][threadIdx.x].x, joined[q][threadIdx.x].y);
    part[int64_t(threadIdx.x) * gridDim.x + blockIdx.x] = make_float2(m, s);
  }
}

// dz[v][ROWS] in 32 bits, the rows' factors included
template <typename T>
__global__ __launch_bounds__(kThreads) void k_few_dz(int B, int rows, int D, int Dk, int64_t V,
                                                     const T* __restrict__ x, int64_t ldx, const T* __restrict__ w,
                                                     int64_t sv, Labels of, const RowStat* __restrict__ stats,
                                                     const float* __restrict__ grad, const float* __restrict__ share,
                                                     float* __restrict__ dz) {
  extern __shared__ __align__(128) char few_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  few_stage<T>(of, B, D, Dk, x, ldx, few_lds);
  const int b = lane & 31;
  const int64_t y = b < B ? label_of(b, of.labels, of.idx, of.n_labels, of.V) : -1;
  const bool live = counts(b, B, of);
  const RowStat st = live ? stats[b] : RowStat{0.f, 1.f, 0.f};
  const float g = live ? (share ? grad[0] * share[0] : grad[b]) : 0.f;
  const float scale = g / st.s;
  for (int64_t v0 = (int64_t(blockIdx.x) * 4 + wave) * 32; v0 < V; v0 += int64_t(gridDim.x) * 128) {
    const f32x16 z = few_logits<T>(D, Dk, v0, V, w, sv, few_lds, lane);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t v = v0 + block_row(e, lane);
      const float d = exp2_raw((z[e] - st.m) * kLog2e) * scale - (v == y ? g : 0.f);
      if (b < rows && v < V) dz[v * rows + b] = live ? d : 0.f;
    }
  }
}

// A wavefront owns 64 * VEC features and four classes in every gridDim.y * 16; dz's rows are the
// same for all its lanes.  dweight leaves at once, dx's share of the workgroup goes to
// part[blockIdx.y][ROWS][D].
template <typename T, int ROWS, int VEC>
__global__ __launch_bounds__(kThreads) void k_few_grads(int B, int D, int64_t V, const T* __restrict__ x, int64_t ldx,
                                                        const T* __restrict__ w, int64_t sv, Labels of,
                                                        const float* __restrict__ dz, T* __restrict__ dw, int64_t dsv,
                                                        int64_t dsd, float* __restrict__ part) {
  __shared__ float joined[4][64 * VEC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int d0 = (int(blockIdx.x) * 64 + lane) * VEC;
  const int left = D - d0;
  float xr[ROWS][VEC], dx[ROWS][VEC];
  // bit b: row b counts; the loads below do not wait for each other
  const uint64_t live = __ballot(counts(lane, B, of));
#pragma unroll
  for (int b = 0; b < ROWS; ++b)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int64_t at = int64_t(b < B ? b : B - 1) * ldx + (e < left ? d0 + e : D - 1);
      const float v = widen(x[at]);
      xr[b][e] = (live >> b & 1) && e < left ? v : 0.f;
      dx[b][e] = 0.f;
    }
  const int64_t stride = int64_t(gridDim.y) * 16;
  for (int64_t v0 = (int64_t(blockIdx.y) * 4 + wave) * 4; v0 < V; v0 += stride) {
    T raw[4][VEC];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t v = v0 + u < V ? v0 + u : V - 1;
      if (left >= VEC) {
        __builtin_memcpy(&raw[u], w + v * sv + d0, sizeof(raw[u]));
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) raw[u][e] = e < left ? w[v * sv + d0 + e] : T{};
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (v0 + u >= V) break;
      const float* row = dz + (v0 + u) * ROWS;
      float out[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) out[e] = 0.f;
#pragma unroll
      for (int b = 0; b < ROWS; ++b) {
        const float z = row[b];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          dx[b][e] = fmaf(z, widen(raw[u][e]), dx[b][e]);
          out[e] = fmaf(z, xr[b][e], out[e]);
        }
      }
      if (dw != nullptr) {
        T res[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) res[e] = narrow<T>(out[e]);
        T* dst = dw + (v0 + u) * dsv + d0 * dsd;
        if (dsd == 1 && left >= VEC) {
          __builtin_memcpy(dst, &res, sizeof(res));
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (e < left) dst[e * dsd] = res[e];
        }
      }
    }
  }
  if (part == nullptr) return;                   // the whole launch
#pragma unroll
  for (int b = 0; b < ROWS; ++b) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) joined[wave][lane * VEC + e] = dx[b][e];
    __syncthreads();
    for (int c = threadIdx.x; c < 64 * VEC; c += kThreads) {
      const int d = int(blockIdx.x) * 64 * VEC + c;
      if (d < D)
        part[(int64_t(blockIdx.y) * ROWS + b) * D + d] = (joined[0][c] + joined[1][c]) + (joined[2][c] + joined[3][c]);
    }
  }
}

// dx[b][d] = sum over the shares: eight of them apart, each in order, then joined in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_few_join(int D, int rows, int splits, const float* __restrict__ part,
                                                       Labels of, T* __restrict__ dx, int64_t lddx) {
  __shared__ float joined[8][32];
  const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int b = blockIdx.x, d = int(blockIdx.y) * 32 + c;
  float s = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int z = q; z < splits; z += 8) s += part[(int64_t(z) * rows + b) * D + d];
  }
  joined[q][c] = s;
  __syncthreads();
  if (q == 0 && d < D) {
#pragma unroll
    for (int z = 1; z < 8; ++z) s += joined[z][c];
    dx[b * lddx + d] = counts(b, b + 1, of) ? narrow<T>(s) : T{};
  }
}

// ------------------------------------------------------------------ bf16, up to 256 features
// Both operands of the logits are rows of up to 16 x 16 features, so one of them can stay in
// registers: a wavefront owns 64 rows of it (or 32; the matrix instruction's columns) and the other
// operand streams through LDS, 64 rows at a time, one step ahead.  The logits of a step come out
// with a lane per owned row; turned into probabilities they already are the right operand of the
// second product, streamed^T . p, which reads the same LDS tile through the transposing load.  So
// logits and probabilities never leave the registers:
//   owner x, stream weight:  statistics;  dx^T = weight^T . p
//   owner weight, stream x:  dweight^T = x^T . dz
// The step's rows are permuted within LDS so that neither way of reading meets bank conflicts.
// 4096 x 256 against 50000 classes: statistics 105 us (1.00 PFLOP/s), dx 174 and dweight 225 us with their
// own logits (1.21 and 0.93), 507 in all; 257 features, by the tiles with dz in memory, 983.
constexpr int kOwnRows = 256;                    // of a workgroup: NB blocks of 32 a wavefront
constexpr int kStreamRows = 64;                  // of a step

template <int KD> constexpr int stream_bytes() { return kStreamRows * KD * 32; }

// position of a row's 16-byte chunk; only the low bits of its number change, and how depends on
// the row alone
template <int KD>
__device__ __forceinline__ int stream_spread(int row) {
  return KD % 8 == 0 ? spread_256(row) : spread_128(row);
}
template <int KD> constexpr int stream_window() { return KD % 8 == 0 ? 256 : 128; }        // bytes it permutes

template <int KD, int WAVES>
__device__ __forceinline__ void stage_stream(const Operand<Bf16>& op, int64_t r0, unsigned lds, int wave, int lane) {
  constexpr int cpr = KD * 2;                    // chunks of a row
  const char* base = reinterpret_cast<const char*>(op.base + r0 * op.ld);              // uniform
  const int left = op.rows - r0 < kStreamRows ? int(op.rows - r0) : kStreamRows;       // at least 1
  const unsigned pitch = unsigned(op.ld) * 2;    // 64 of them below 2^32 (weight_as_is)
#pragma unroll
  for (int l = 0; l < stream_bytes<KD>() / 16 / (64 * WAVES); ++l) {
    const int first = (l * WAVES + wave) * 64, q = first + lane;
    const int row = q / cpr, c = (q % cpr) ^ stream_spread<KD>(row);
    load_to_lds(base, unsigned(row < left ? row : left - 1) * pitch + c * 16, lds + first * 16);
  }
}

template <int KD, int NB>
__device__ __forceinline__ void load_owned(const Operand<Bf16>& op, int64_t r0, int lane, bf16x8 (&own)[NB][KD]) {
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    int64_t r = r0 + 32 * j + (lane & 31);
    r = r < op.rows ? r : op.rows - 1;
    const Bf16* src = op.base + r * op.ld + 8 * (lane >> 5);
#pragma unroll
    for (int k = 0; k < KD; ++k) own[j][k] = *reinterpret_cast<const bf16x8*>(src + 16 * k);
  }
}

// Where a lane reads.  Rows are aligned to the permuted windows, so another chunk of the same window
// is an exclusive-or away and everything else a constant offset of the read.
struct StreamLane {
  int direct;              // logits: row lane & 31, chunk lane / 32
  int across;              // second product: its row of the first four (second half: of the next), first 64 features
};
template <int KD>
__device__ __forceinline__ StreamLane stream_lane(int lane) {
  const int row = lane & 31, half = lane >> 5;
  const int r = 4 * half + ((lane & 15) >> 2), c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  return {row * (KD * 32) + ((half ^ stream_spread<KD>(row)) << 4),
          r * (KD * 32) + ((c ^ stream_spread<KD>(r)) << 4) + (lane & 1) * 8};
}
template <int KD>
__device__ __forceinline__ bf16x8 stream_row(const char* tile, int sub, int k, const StreamLane& at) {
  constexpr int kWindow = stream_window<KD>();
  const int place = (at.direct ^ ((32 * k) % kWindow)) + (32 * sub * KD * 32 + 32 * k / kWindow * kWindow);
  return *reinterpret_cast<const bf16x8*>(tile + place);
}

// streamed^T as an operand: features 32 * block .. + 31, and of rows 32 * sub .. the sixteen that
// elements 8 * q .. of a logits block hold (in that order)
template <int KD>
__device__ __forceinline__ bf16x8 stream_across(const char* tile, int sub, int q, int block, const StreamLane& at) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  constexpr int kWindow = stream_window<KD>();
  const int place = at.across ^ ((64 * block) % kWindow);
  const char* src = tile + ((32 * sub + 16 * q) * KD * 32 + 64 * block / kWindow * kWindow);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src + place));
  // eight rows on the permutation differs by two chunks
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src + (place ^ 32) + 8 * KD * 32));
  bf16x8 r;
  __builtin_memcpy(&r, &lo, 8);
  __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &hi, 8);
  return r;
}

// Logits of the step's rows 32 * sub .. + 31 (rows of a block) and the owned rows (columns), with
// other work between the matrix instructions: between(i) is called for i = 0 .. 16 * NB - 1, a few
// after each of them, and stays there.  The matrix unit works on while the
// vector unit does; left to itself the compiler puts one after the other.
template <int KD, int NB, typename Between>
__device__ __forceinline__ void stream_logits_between(const char* tile, int sub, const StreamLane& at,
                                                      const bf16x8 (&own)[NB][KD], f32x16 (&z)[NB],
                                                      Between&& between) {
  const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  constexpr int kAhead = KD < 16 ? 3 : 2;        // reads under way
  bf16x8 a[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) a[k] = stream_row<KD>(tile, sub, k, at);
#pragma unroll
  for (int k = 0; k < KD; ++k) {
    const bf16x8 cur = a[k % kAhead];
    if (k + kAhead < KD) a[k % kAhead] = stream_row<KD>(tile, sub, k + kAhead, at);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      z[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cur, own[j][k], k ? z[j] : zero, 0, 0, 0);
      const int step = NB * k + j;
#pragma unroll
      for (int i = 16 * step / KD; i < 16 * (step + 1) / KD; ++i) between(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <int KD>
__global__ __launch_bounds__(kThreads) void k_wide_stats(int64_t B, int64_t V, Operand<Bf16> x, Operand<Bf16> w,
                                                         Labels of, int64_t steps, int splits,
                                                         float2* __restrict__ part, float* __restrict__ picked) {
  __shared__ __align__(128) char lds[2 * stream_bytes<KD>()];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.x % splits;
  const int64_t b0 = int64_t(blockIdx.x / splits) * kOwnRows + 64 * wave;
  const int64_t t0 = steps * split / splits, t1 = steps * (split + 1) / splits;
  const StreamLane at = stream_lane<KD>(lane);
  bf16x8 own[2][KD];
  load_owned(x, b0, lane, own);
  // The sums are relative to a reference logit that follows the largest one only when that gets
  // kSlack ahead (2^60), so that most half steps are a multiply-add, an exponential and an addition
  // per logit: 2^(z log2 e - c), c = ref * log2 e rounded, `back` = what the rounding has to be put
  // right by.  Where the rounding alone could leave the exponent's range (logits of millions) c is 0
  // and the reference is taken off the logits first.
  constexpr float kSlack = 41.f;
  float top[2], sum[2], ref[2], limit[2], c[2], back[2];
  bool any_far = false;
  int y[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t b = b0 + 32 * j + (lane & 31);
    top[j] = -INFINITY;
    ref[j] = limit[j] = -INFINITY;
    c[j] = 0.f;
    back[j] = 1.f;
    sum[j] = 0.f;
    y[j] = b < B ? int(label_of(b, of.labels, of.idx, of.n_labels, of.V)) : -1;
  }
  // the label's logit and the classes beyond the last, both rare
  const auto settle = [&](f32x16 (&z)[2], int64_t v0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int at = y[j] - int(v0);
      int mine = at - 4 * (lane >> 5);           // compared with constants
      asm("" : "+v"(mine));                      // and not taken apart into sixteen registers
      if (__any(at >= 0 && at < 32)) {
        float hit = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) hit = block_row(e, 0) == mine ? z[j][e] : hit;
        if (at >= 0 && at < 32 && ((at >> 2) & 1) == lane >> 5) picked[b0 + 32 * j + (lane & 31)] = hit;
      }
    }
    if (v0 + 32 > V) {
      int left = int(V - v0) - 4 * (lane >> 5);
      asm("" : "+v"(left));
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) z[j][e] = block_row(e, 0) < left ? z[j][e] : -INFINITY;
    }
  };
  // the logits of one half step while the other's are summed
  const auto turn = [&](const char* tile, int sub, f32x16 (&next)[2], f32x16 (&z)[2]) {
    float m[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x16 one[1] = {z[j]};
      m[j] = largest(one);
      top[j] = fmaxf(top[j], m[j]);
    }
    if (__any(m[0] > limit[0] || m[1] > limit[1])) {                       // rare after the first few
      any_far = false;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (m[j] > limit[j]) {
          sum[j] *= exp2_raw((ref[j] - m[j]) * kLog2e) * back[j];
          ref[j] = m[j];
          limit[j] = m[j] + kSlack;
          const bool far = !(fabsf(m[j]) < kFarLogit);
          c[j] = far ? 0.f : m[j] * kLog2e;
          back[j] = far ? 1.f : exp2_raw(-fmaf(m[j], kLog2e, -c[j]));
          sum[j] *= far ? 1.f : exp2_raw(fmaf(m[j], kLog2e, -c[j]));
        }
        any_far = any_far || __any(!(fabsf(ref[j]) < kFarLogit) && ref[j] != -INFINITY);
      }
    }
    if (any_far) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float off = !(fabsf(ref[j]) < kFarLogit) && ref[j] != -INFINITY ? ref[j] : 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) z[j][e] -= off;
      }
    }
    StreamLane here = at;                        // its variants are made where they are used, not kept
    asm volatile("" : "+v"(here.direct));
    stream_logits_between(tile, sub, here, own, next, [&](int i) {
      sum[i >> 4] += exp2_raw(fmaf(z[i >> 4][i & 15], kLog2e, -c[i >> 4]));
      asm volatile("" : "+v"(sum[i >> 4]));      // now, not where the sum is used
    });
  };
  const unsigned stages = lds_offset(lds);
  if (t0 < t1) {
    stage_stream<KD, 4>(w, t0 * kStreamRows, stages, wave, lane);
    f32x16 first[2], second[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) second[j][e] = -INFINITY;               // adds nothing
    for (int64_t t = t0; t < t1; ++t) {
      landed();
      __syncthreads();
      const int cur = int(t - t0) & 1;
      if (t + 1 < t1) stage_stream<KD, 4>(w, (t + 1) * kStreamRows, stages + (cur ^ 1) * stream_bytes<KD>(), wave, lane);
      const char* tile = lds + cur * stream_bytes<KD>();
      turn(tile, 0, first, second);
      settle(first, t * kStreamRows);
      turn(tile, 1, second, first);
        settle(second, t * kStreamRows + 32);
    }
    // to the largest logit, and the last half step's share
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m = ref[j];
      sum[j] *= back[j];
      join_stats(m, sum[j], top[j], 0.f);
      f32x16 one[1] = {second[j]};
      top[j] = m;
      accumulate(one, top[j], sum[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float om = __shfl_xor(top[j], 32), os = __shfl_xor(sum[j], 32);
    join_stats(top[j], sum[j], om, os);
    const int64_t b = b0 + 32 * j + (lane & 31);
    if (lane < 32 && b < B) part[b * splits + split] = make_float2(top[j], sum[j]);
  }
}

// acc += streamed^T . p over a half step, with other work between as above
template <int KD, int NB, typename Between>
__device__ __forceinline__ void stream_gather_between(const char* tile, int sub, const StreamLane& at,
                                                      const bf16x8 (&p)[NB][2], f32x16 (&acc)[KD / 2][NB],
                                                      Between&& between) {
  constexpr int kAhead = 2;                      // reads under way
  bf16x8 a[kAhead];
#pragma unroll
  for (int n = 0; n < kAhead; ++n) a[n] = stream_across<KD>(tile, sub, n & 1, n >> 1, at);
#pragma unroll
  for (int n = 0; n < KD; ++n) {                 // features 32 * (n / 2), rows 16 * (n & 1)
    const bf16x8 cur = a[n % kAhead];
    if (n + kAhead < KD) a[n % kAhead] = stream_across<KD>(tile, sub, (n + kAhead) & 1, (n + kAhead) >> 1, at);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      acc[n >> 1][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cur, p[j][n & 1], acc[n >> 1][j], 0, 0, 0);
      const int step = NB * n + j;
#pragma unroll
      for (int i = 16 * step / KD; i < 16 * (step + 1) / KD; ++i) between(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// BY_CLASS: owner weight, stream x, dz^T with the label's -1; else owner x, stream weight, p alone
// (what the label takes off joins dx in its last step).  PER_ROW: every row has a factor of its own
// (in dweight here; dx takes it in its last step).  The sums go to part[split][owned row][KD * 16] in
// 32 bits or, with `out` (dweight from one split), times the mean's factor to where they belong.
// A wavefront owns 32 rows: 64 (half the LDS reads, but one wavefront a SIMD instead of two) took
// 58 + 58 us instead of 56 + 52 us at 1777 x 100 x 30011, and spilled at 256 features, where dweight's
// kernel keeps 6 registers in scratch as it is (21 and 292 us with a factor for every row).
constexpr int kGradThreads = 512;

template <int KD, bool BY_CLASS, bool PER_ROW>
__global__ __launch_bounds__(kGradThreads, 2) void k_wide_grads(int64_t owners, int64_t streams, Operand<Bf16> owned,
                                                            Operand<Bf16> streamed, RowConst rows, int64_t steps,
                                                            int splits, float* __restrict__ part, int64_t plane,
                                                            int D, Bf16* __restrict__ out, int64_t sr, int64_t sd,
                                                            const float* __restrict__ grad,
                                                            const float* __restrict__ share) {
  __shared__ __align__(128) char lds[2 * stream_bytes<KD>()];
  constexpr int NB = 1, kWaves = kGradThreads / 64;
  // Taking turns keeps p across half steps; at 256 features that no longer fits the registers
  // (4096 x 256 x 50000: dweight 306 us with turns, 253 us without; dx 218 and 193 us).
  constexpr bool kTurns = KD < 16;
  __shared__ __align__(16) float row_shift[kWaves][kStreamRows], row_top[kWaves][kStreamRows],
      row_factor[kWaves][kStreamRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.x % splits;
  const int64_t o0 = int64_t(blockIdx.x / splits) * kOwnRows + 32 * NB * wave;
  const int64_t t0 = steps * split / splits, t1 = steps * (split + 1) / splits;
  const StreamLane at = stream_lane<KD>(lane);
  bf16x8 own[NB][KD];
  load_owned(owned, o0, lane, own);
  f32x16 acc[KD / 2][NB];
#pragma unroll
  for (int d = 0; d < KD / 2; ++d)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[d][j][e] = 0.f;
  float shift[NB] = {};
  bool any_large = false, wild = false;          // wild: an owned class holds an infinity or NaN
  if constexpr (BY_CLASS) {
    unsigned lo = 0, hi = 0;                     // the largest magnitudes of either half of the words
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        u32x4 w;
        __builtin_memcpy(&w, &own[j][k], 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          lo = max(lo, w[q] & 0x7fffu);
          hi = max(hi, w[q] & 0x7fff0000u);
        }
      }
    wild = __any(lo >= 0x7f80u || hi >= 0x7f800000u);
  }
  if constexpr (!BY_CLASS) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int64_t b = o0 + 32 * j + (lane & 31);
      shift[j] = rows.shift[b < owners ? b : owners - 1];
      any_large = any_large || __any(rows.top[b < owners ? b : owners - 1] != 0.f);
    }
  }
  float next_shift = 0.f, next_top = 0.f, next_factor = 0.f;               // of row `lane` of the coming step
  int next_label = -1;
  const auto fetch_rows = [&](int64_t t) {
    // a 32-bit offset from a uniform base: no address registers (at most 2^30 rows)
    const int64_t first = t * kStreamRows;
    next_shift = (rows.shift + first)[unsigned(lane)];
    next_top = (rows.top + first)[unsigned(lane)];
    if constexpr (PER_ROW) next_factor = (rows.factor + first)[unsigned(lane)];
    next_label = (rows.label + first)[unsigned(lane)];
  };
  const unsigned stages = lds_offset(lds);
  if (t0 < t1) {
    stage_stream<KD, kWaves>(streamed, t0 * kStreamRows, stages, wave, lane);
    if constexpr (BY_CLASS) fetch_rows(t0);
  }
  // A half step's logits become p while the half step before is multiplied: p of -1 is 0
  bf16x8 p[NB][2];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) p[j][e >> 3][e & 7] = static_cast<__bf16>(0.f);
  int label = -1;
  const auto half_step = [&](int64_t t, const char* tile, int sub, const char* before) {
    f32x16 z[NB];
    StreamLane here = at;                        // its variants are made where they are used, not kept
    asm volatile("" : "+v"(here.direct), "+v"(here.across));
    stream_logits_between(tile, sub, here, own, z, [](int) {});
    if (any_large) {                             // rare
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int64_t b = o0 + 32 * j + (lane & 31);
        const float top = BY_CLASS ? 0.f : rows.top[b < owners ? b : owners - 1];
#pragma unroll
        for (int e = 0; e < 16; ++e) z[j][e] -= BY_CLASS ? row_top[wave][32 * sub + block_row(e, lane)] : top;
      }
    }
    f32x4 c[2];                                  // shifts of four rows, and of the next four
    const auto shifts = [&](int e) {
      return *reinterpret_cast<const f32x4*>(&row_shift[wave][32 * sub + block_row(e, lane)]);
    };
    if constexpr (BY_CLASS) c[0] = shifts(0);
    const auto weigh = [&](int i) {
      const int j = i % NB, e = i / NB;
      if (BY_CLASS && j == 0 && e % 4 == 0 && e < 12) c[(e / 4 + 1) & 1] = shifts(e + 4);
      z[j][e] = exp2_raw(fmaf(z[j][e], kLog2e, -(BY_CLASS ? c[e / 4 & 1][e & 3] : shift[j])));
      float now = z[j][e];
      asm volatile("" : "+v"(now));              // now, not where it is used
      z[j][e] = now;
    };
    if constexpr (kTurns) {
      stream_gather_between<KD, NB>(before, sub ^ 1, here, p, acc, weigh);
    } else {
#pragma unroll
      for (int i = 0; i < 16 * NB; ++i) weigh(i);
    }
    bool with_label = false;
    if constexpr (BY_CLASS) {
      // 0 x infinity in rows without a class and beyond the last, whose shift is infinite: p is 0 there
      if (wild) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const f32x4 its_shift = shifts(e);
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < NB; ++j) z[j][e + q] = its_shift[q] == INFINITY ? 0.f : z[j][e + q];
        }
      }
      // rows whose label is among the owned classes: rare
      uint64_t h = __ballot(label >= o0 && label < o0 + 32 * NB) >> (32 * sub) & 0xffffffffull;
      with_label = h != 0;
      for (; h != 0; h &= h - 1) {
        const int r = __builtin_ctzll(h);
        const int col = int(__shfl(label, 32 * sub + r) - o0);
        int mine = r - 4 * (lane >> 5);          // compared with constants
        asm("" : "+v"(mine));
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) z[j][e] -= block_row(e, 0) == mine && 32 * j + (lane & 31) == col ? 1.f : 0.f;
      }
      if constexpr (PER_ROW) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const f32x4 g = *reinterpret_cast<const f32x4*>(&row_factor[wave][32 * sub + block_row(e, lane)]);
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < NB; ++j) z[j][e + q] *= g[q];
        }
      }
    } else if (t * kStreamRows + 32 * sub + 32 > streams) {                // classes beyond the last
      int left = int(streams - t * kStreamRows) - 32 * sub - 4 * (lane >> 5);
      asm("" : "+v"(left));
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) z[j][e] = block_row(e, 0) < left ? z[j][e] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) p[j][e >> 3][e & 7] = static_cast<__bf16>(z[j][e]);
    // The label's element is nearly all of a class's gradient, and what rounding takes off it would be
    // felt: a half step that holds one is multiplied by that, too.
    bf16x8 off[NB][2];
    if (BY_CLASS && with_label) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          off[j][e >> 3][e & 7] = static_cast<__bf16>(z[j][e] - static_cast<float>(p[j][e >> 3][e & 7]));
    }
    if constexpr (kTurns) {
      if (BY_CLASS && with_label) stream_gather_between<KD, NB>(tile, sub, here, off, acc, [](int) {});
    } else {
      for (bool again = BY_CLASS && with_label;; again = false) {
        stream_gather_between<KD, NB>(tile, sub, here, p, acc, [](int) {});
        if (!again) break;
#pragma unroll
        for (int j = 0; j < NB; ++j) p[j][0] = off[j][0], p[j][1] = off[j][1];
      }
    }
  };
  const char* tile = lds;
  for (int64_t t = t0; t < t1; ++t) {
    landed();
    __syncthreads();
    const int cur = int(t - t0) & 1;
    tile = lds + cur * stream_bytes<KD>();
    if constexpr (BY_CLASS) {                    // a wavefront's own copy: no barrier
      row_shift[wave][lane] = next_shift;
      row_top[wave][lane] = next_top;
      any_large = __any(next_top != 0.f);
      if constexpr (PER_ROW) row_factor[wave][lane] = next_factor;
      label = next_label;
      __builtin_amdgcn_wave_barrier();
    }
    // the first step has nothing before it: p is 0 and any numbers will do, its own
    half_step(t, tile, 0, t == t0 ? tile : lds + (cur ^ 1) * stream_bytes<KD>());
    if constexpr (kTurns) __syncthreads();       // everybody has left the step before
    if (t + 1 < t1) {
      stage_stream<KD, kWaves>(streamed, (t + 1) * kStreamRows, stages + (cur ^ 1) * stream_bytes<KD>(), wave, lane);
      if constexpr (BY_CLASS) fetch_rows(t + 1);
    }
    half_step(t, tile, 1, tile);
  }
  if constexpr (kTurns) stream_gather_between<KD, NB>(tile, 1, at, p, acc, [](int) {});
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t r = o0 + 32 * j + (lane & 31);
    if (r >= owners) continue;
    if (out != nullptr) {
      const float factor = share ? grad[0] * share[0] : 1.f;
      Bf16* dst = out + r * sr;
      const bool whole = sd == 1 && sr % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0;
#pragma unroll
      for (int d = 0; d < KD / 2; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int at = 32 * d + block_row(e, lane);
          Bf16 four[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) four[q] = narrow<Bf16>(factor * acc[d][j][e + q]);
          if (whole && at + 4 <= D) {
            u32x2 w;
            __builtin_memcpy(&w, &four, 8);
            *reinterpret_cast<u32x2*>(dst + at) = w;
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (at + q < D) dst[(at + q) * sd] = four[q];
          }
        }
      continue;
    }
    float* dst = part + split * plane + r * (KD * 16);
#pragma unroll
    for (int d = 0; d < KD / 2; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>(dst + 32 * d + block_row(e, lane)) =
            f32x4{acc[d][j][e], acc[d][j][e + 1], acc[d][j][e + 2], acc[d][j][e + 3]};
  }
}

// ------------------------------------------------------------------ plans
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Plan {
  int Dp, depth;                     // padded features, reduction step
  size_t elem;
  int64_t Bp, tiles_b, tiles_v;
  int stat_splits;
  // backward
  int64_t piece;                     // classes of a piece, a multiple of kTile
  int tiles_d;
  int dx_splits, dw_splits;
};

// Of dz at a time.  Larger pieces mean fewer and fuller launches; past the 256 MB of the last-level
// cache there is nothing more to gain.  Loss and gradients in fp32 at 32 / 96 / 256 MB: 4096 rows of 128
// features, 50000 classes 2025 / 1533 / 1459 us; 16384, 64, 20000: 2872 / 1970 / 1772; 512, 128, 100000:
// 581 / 451 / 417.
constexpr int64_t kPieceBytes = int64_t(256) << 20;
constexpr int kSlots = 512;                             // workgroups that run at once: two on a CU, by their LDS

// Shares of a reduction of `most` steps for `groups` workgroups a share, where `slots` workgroups
// run at once: as many as fill the slots, or, where the groups alone are more, the number up to
// four whose last round is fullest (a fifth better than none, or none).
int spread(int64_t slots, int64_t groups, int64_t most) {
  int64_t s = slots / groups;
  if (s < 1) {
    s = 1;
    double best = 0.8 * double(ceil_div(groups, slots));
    for (int64_t q = 2; q <= 4; ++q)
      if (const double rounds = double(ceil_div(groups * q, slots)) / double(q); rounds <= best) {
        best = 0.95 * rounds;                    // each share more is one more to write and to join
        s = q;
      }
  }
  if (s > most) s = most;
  return s < 1 ? 1 : int(s);
}

Plan make_plan(int dtype, int64_t B, int64_t D, int64_t V) {
  Plan p;
  p.elem = dtype == SGNN_F32 ? 4 : 2;
  p.depth = int(128 / p.elem);
  p.Dp = int(ceil_div(D, 64) * 64);
  p.tiles_b = ceil_div(B, kTile);
  p.tiles_v = ceil_div(V, kTile);
  p.Bp = p.tiles_b * kTile;
  p.stat_splits = spread(kSlots, p.tiles_b, p.tiles_v);
  int64_t tiles = kPieceBytes / (p.Bp * int64_t(p.elem) * kTile);
  if (tiles < 1) tiles = 1;
  if (tiles > p.tiles_v) tiles = p.tiles_v;
  p.piece = tiles * kTile;
  p.tiles_d = int(ceil_div(D, kTile));
  p.dx_splits = spread(kSlots, p.tiles_b * p.tiles_d, p.piece / p.depth / 2);
  p.dw_splits = spread(kSlots, tiles * p.tiles_d, p.Bp / p.depth / 2);
  return p;
}

// The kernels that keep rows in registers: sizes, KD 0 where they do not apply.
struct Wide {
  int KD;
  int64_t own_b, own_v, steps_b, steps_v;        // owners' workgroups and stream steps of either operand
  int stat_splits, dx_splits, dw_splits;
};

Wide make_wide(int dtype, int64_t B, int64_t D, int64_t V) {
  Wide f{};
  if (dtype != SGNN_BF16 || D > 256) return f;
  f.KD = int(ceil_div(D, 64) * 4);
  f.own_b = ceil_div(B, kOwnRows);
  f.own_v = ceil_div(V, kOwnRows);
  f.steps_b = ceil_div(B, kStreamRows);
  f.steps_v = ceil_div(V, kStreamRows);
  // by what a CU's registers hold: two workgroups of four wavefronts up to 192 features; of eight, one, up to 64 two
  f.stat_splits = spread(f.KD < 16 ? 512 : 256, f.own_b, f.steps_v);
  f.dx_splits = spread(f.KD > 4 ? 256 : 512, f.own_b, f.steps_v);
  f.dw_splits = spread(f.KD > 4 ? 256 : 512, f.own_v, f.steps_b);
  return f;
}

// The few-rows kernels: sizes that fit them, 0 rows where they do not apply.  Loss and gradients of 256
// features and 100003 classes: fp32 32 rows 175 us (104 at one row), 33 rows by the tiles 228 us; bf16 16
// rows 99 us, 32 rows 141 us, which the kernels with rows in registers take 114 us for.
struct Few {
  int rows, Dk, vec;
  size_t lds;
  unsigned blocks, slabs, splits;
};

Few make_few(int dtype, int64_t B, int64_t D, int64_t V, int64_t sd) {
  Few f{};
  const int P = dtype == SGNN_F32 ? 3 : 1;
  if (B > (make_wide(dtype, B, D, V).KD ? 16 : kFewRows) || sd != 1 || D > 65536) return f;
  f.Dk = int(ceil_div(D, 64) * 64);
  f.lds = size_t(P) * kFewRows * f.Dk * 2;
  if (f.lds > 150 * 1024) return f;              // of 160 KB
  f.rows = B <= 2 ? 2 : B <= 4 ? 4 : B <= 8 ? 8 : B <= 16 ? 16 : 32;
  f.vec = f.rows > 16 ? 2 : 4;
  const int64_t blocks = ceil_div(V, 128);
  f.blocks = unsigned(blocks < kFewBlocks ? blocks : kFewBlocks);
  f.slabs = unsigned(ceil_div(D, 64 * f.vec));
  const int64_t want = ceil_div(f.rows > 8 ? 512 : 1024, f.slabs), most = ceil_div(V, 16);
  f.splits = unsigned(want < most ? want : most);
  return f;
}

struct Buffers {
  char *x, *w, *dz;
  float2* part;
  float *picked, *rest, *dx, *dw;
  RowConst rows;
  size_t bytes;
};

Buffers carve(const Plan& p, int64_t B, int64_t V, bool backward, void* base) {
  sgnn::Carver c(base);
  Buffers b{};
  b.x = c.take<char>(p.elem * B * p.Dp);
  b.w = c.take<char>(p.elem * V * p.Dp);
  if (!backward) {
    b.part = c.take<float2>(size_t(p.stat_splits) * 2 * B);
    b.picked = c.take<float>(size_t(B));
  } else {
    const size_t Np = size_t(p.tiles_d) * kTile;
    b.dz = c.take<char>(p.elem * p.Bp * p.piece);
    b.rest = c.take<float>(size_t(B));
    if (p.elem == 2) b.rows.label = c.take<int>(size_t(B));
    b.dx = c.take<float>(size_t(p.dx_splits) * p.Bp * Np);
    b.dw = c.take<float>(size_t(p.dw_splits) * p.piece * Np);
  }
  b.bytes = c.off;
  return b;
}

Buffers carve_wide(const Wide& f, const Plan& p, int64_t B, int64_t V, bool backward, void* base) {
  sgnn::Carver c(base);
  Buffers b{};
  b.x = c.take<char>(p.elem * B * p.Dp);
  b.w = c.take<char>(p.elem * V * p.Dp);
  if (!backward) {
    b.part = c.take<float2>(size_t(f.stat_splits) * B);
    b.picked = c.take<float>(size_t(B));
  } else {
    static_assert(kStreamRows == 64, "rows are laid out and prepared 64 at a time");
    const size_t padded = size_t(f.steps_b) * kStreamRows;
    b.rows = RowConst{c.take<float>(padded), c.take<float>(padded), c.take<float>(padded), c.take<float>(padded),
                      c.take<int>(padded)};
    b.dx = c.take<float>(size_t(f.dx_splits) * B * p.Dp);
    b.dw = c.take<float>(size_t(f.dw_splits) * V * p.Dp);
  }
  b.bytes = c.off;
  return b;
}

Buffers carve_few(const Few& f, int64_t B, int64_t D, int64_t V, bool backward, void* base) {
  sgnn::Carver c(base);
  Buffers b{};
  if (!backward) {
    b.part = c.take<float2>(size_t(f.blocks) * B);
    b.picked = c.take<float>(size_t(B));
  } else {
    b.dw = c.take<float>(size_t(V) * f.rows);    // dz
    b.dx = c.take<float>(size_t(f.splits) * f.rows * D);
  }
  b.bytes = c.off;
  return b;
}

struct Call {
  int dtype;
  int64_t B, D, V;
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t sv, sd;
  const int64_t* labels;
  int64_t n_labels;
  const int64_t* idx;
  bool all;
  Labels of() const { return {labels, idx, n_labels, V, all}; }
};

// One launch takes fewer than 2^32 threads: a wavefront a row, a workgroup of 256 for 64 x 64 of the
// operands and for 32 x 32 of the gradients.
const char* too_large(int64_t B, int64_t D, int64_t V) {
  if (B > (int64_t(1) << 25) || V > (int64_t(1) << 28) || D > (int64_t(1) << 16))
    return "head larger than 2^25 rows, 2^28 classes or 65536 features";
  const int64_t width = ceil_div(D, 64) * 64;
  if ((B + V) * width > (int64_t(1) << 33)) return "operands of more than 2^33 elements";
  return nullptr;
}

int check_call(const Call& c) {
  using sgnn::fail;
  if (c.dtype != SGNN_F32 && c.dtype != SGNN_BF16) return fail(SGNN_ERR_INVALID, "unknown element type");
  if (c.all && c.dtype != SGNN_F32) return fail(SGNN_ERR_UNSUPPORTED, "rows without a class count in fp32 only");
  if (c.B <= 0 || c.D <= 0 || c.V <= 0) return fail(SGNN_ERR_INVALID, "need B > 0, D > 0, V > 0");
  if (const char* why = too_large(c.B, c.D, c.V)) return fail(SGNN_ERR_UNSUPPORTED, why);
  if (c.ldx < c.D) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (!((c.sd == 1 && c.sv >= c.D) || (c.sv == 1 && c.sd >= c.V)))
    return fail(SGNN_ERR_INVALID, "the weight must have unit stride along its features or its classes");
  if (c.n_labels < 0 || (!c.idx && c.n_labels < c.B)) return fail(SGNN_ERR_INVALID, "fewer labels than rows");
  if (!c.x || !c.w || !c.labels) return fail(SGNN_ERR_INVALID, "null pointer");
  return SGNN_OK;
}

// A weight whose rows are whole steps and 16-byte aligned can be staged as it lies; for stage_stream,
// whose offsets within a step have 32 bits, if they lie close enough together for that.
bool weight_as_is(const Call& c, const Plan& p, bool streamed) {
  return c.sd == 1 && c.D % p.depth == 0 && size_t(c.sv) * p.elem % 16 == 0 &&
         reinterpret_cast<uintptr_t>(c.w) % 16 == 0 &&
         (!streamed || c.sv <= int64_t(UINT32_MAX) / (kStreamRows * int64_t(p.elem)));
}

template <typename T>
int operands(const Call& c, const Plan& p, const Buffers& b, const Rows& rows, bool streamed, Operand<T>* x,
             Operand<T>* w, hipStream_t st) {
  const int across = p.Dp / 64;
  const Source sx{c.x, c.B, c.ldx, 1, b.x, ceil_div(c.B, 64) * across};
  Source sw{c.w, c.V, c.sv, c.sd, b.w, ceil_div(c.V, 64) * across};
  *x = Operand<T>{reinterpret_cast<const T*>(b.x), p.Dp, c.B, p.Dp};
  *w = Operand<T>{reinterpret_cast<const T*>(b.w), p.Dp, c.V, p.Dp};
  if (weight_as_is(c, p, streamed)) {
    sw.blocks = 0;
    *w = Operand<T>{static_cast<const T*>(c.w), c.sv, c.V, c.D};
  }
  hipLaunchKernelGGL((k_class_operands<T>), dim3(unsigned(sx.blocks + sw.blocks)), dim3(256), 0, st, int(c.D), p.Dp, sx,
                     sw, c.of(), rows);
  HIP_TRY(hipGetLastError());
  return SGNN_OK;
}

int finish_forward(const Call& c, int parts, const Buffers& b, RowStat* stats, float* row_loss, float* loss,
                   float* share, hipStream_t st) {
  hipLaunchKernelGGL(k_class_rows, dim3(unsigned(ceil_div(c.B, 4))), dim3(256), 0, st, c.B, c.V, parts, b.part, b.picked,
                     c.labels, c.idx, c.n_labels, stats, row_loss);
  HIP_TRY(hipGetLastError());
  if (loss) {
    hipLaunchKernelGGL(k_class_mean, dim3(1), dim3(1024), 0, st, c.B, c.of(), row_loss, loss, share);
    HIP_TRY(hipGetLastError());
  }
  return SGNN_OK;
}

// a kernel's dynamic LDS beyond the default limit has to be asked for
int allow_lds(const void* kernel, size_t bytes) {
  HIP_TRY(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
  return SGNN_OK;
}

template <typename T>
int forward(const Call& c, const Plan& p, const Buffers& b, RowStat* stats, float* row_loss, float* loss,
            float* share, hipStream_t st) {
  Operand<T> x, w;
  if (int rc = operands<T>(c, p, b, Rows{}, false, &x, &w, st)) return rc;
  const int depth = int(ceil_div(c.D, p.depth) * p.depth);
  hipLaunchKernelGGL((k_class_stats<T>), dim3(unsigned(p.tiles_b * p.stat_splits)), dim3(kThreads), 0, st, c.B, c.V,
                     depth, x, w, c.labels, c.idx, c.n_labels, p.tiles_v, p.stat_splits, b.part, b.picked);
  HIP_TRY(hipGetLastError());
  return finish_forward(c, 2 * p.stat_splits, b, stats, row_loss, loss, share, st);
}

template <typename T>
int launch_joins(const Join<T>& first, const Join<T>& second, hipStream_t st) {
  const unsigned blocks = first.blocks() + second.blocks();
  if (blocks == 0) return SGNN_OK;
  hipLaunchKernelGGL((k_class_join<T>), dim3(blocks), dim3(256), 0, st, first, second, first.blocks());
  HIP_TRY(hipGetLastError());
  return SGNN_OK;
}

template <typename T>
int backward(const Call& c, const Plan& p, const Buffers& b, const RowStat* stats, const float* grad,
             const float* share, void* dx, int64_t lddx, void* dw, int64_t dsv, int64_t dsd, hipStream_t st) {
  Operand<T> x, w;
  if (int rc = operands<T>(c, p, b, Rows{c.B, nullptr, nullptr, nullptr, b.rows}, false, &x, &w, st)) return rc;
  const int64_t Np = int64_t(p.tiles_d) * kTile;
  T* const dz = reinterpret_cast<T*>(b.dz);
  const int depth = int(ceil_div(c.D, p.depth) * p.depth);
  for (int64_t v0 = 0; v0 < c.V; v0 += p.piece) {
    const int64_t left = ceil_div(c.V - v0, kTile);
    const int tiles = int(left < p.piece / kTile ? left : p.piece / kTile);
    const int64_t width = int64_t(tiles) * kTile;
    hipLaunchKernelGGL((k_class_dz<T>), dim3(unsigned(p.tiles_b * tiles)), dim3(kThreads), 0, st, c.B, depth, x, w,
                       c.of(), stats, share ? nullptr : grad, b.rest, v0, tiles, dz, p.piece);
    HIP_TRY(hipGetLastError());
    const Operand<T> a{dz, p.piece, p.Bp, p.piece};
    Product<T> to_dx{}, to_dw{};
    if (dx)                                      // dx[b][d] += dz[b][v] . w[v][d]
      to_dx = Product<T>{a, Operand<T>{w.base + v0 * w.ld, w.ld, c.V - v0, w.cols}, width, p.tiles_d, p.dx_splits,
                         v0 > 0 ? 1 : 0, b.dx, p.Bp * Np, Np, Direct<T>{}, unsigned(p.tiles_b * p.dx_splits * p.tiles_d), nullptr, nullptr, 0, 0};
    Join<T> join_dw{};
    if (dw) {                                    // dw[v][d] = dz[b][v] . x[b][d]
      const int64_t rows = c.V - v0 < width ? c.V - v0 : width;
      T* const out = static_cast<T*>(dw) + v0 * dsv;
      to_dw = Product<T>{a, x, p.Bp, p.tiles_d, p.dw_splits, 0, b.dw, p.piece * Np, Np, Direct<T>{},
                         unsigned(tiles * p.dw_splits * p.tiles_d), b.rest, b.rows.label, c.B, v0};
      if (p.dw_splits == 1 && dsd == 1)
        to_dw.direct = Direct<T>{out, dsv, rows, int(c.D), share ? grad : nullptr, share};
      else
        join_dw = Join<T>{rows, int(c.D), p.dw_splits, b.dw, p.piece * Np, Np, share ? grad : nullptr, share, nullptr,
                          Labels{}, nullptr, 0, 0, out, dsv, dsd};
    }
    bool together = true;
    if constexpr (sizeof(T) == 2) {
      together = dx && dw && (to_dx.blocks < kSlots / 2 || to_dw.blocks < kSlots / 2);
      if (!together && dx) {
        hipLaunchKernelGGL((k_class_products<T, true, false>), dim3(to_dx.blocks), dim3(kThreads), 0, st, to_dx, to_dw);
        HIP_TRY(hipGetLastError());
      }
      if (!together && dw)
        hipLaunchKernelGGL((k_class_products<T, false, true>), dim3(to_dw.blocks), dim3(kThreads), 0, st, Product<T>{}, to_dw);
    }
    if (together)
      hipLaunchKernelGGL((k_class_products<T, true, true>), dim3(to_dx.blocks + to_dw.blocks), dim3(kThreads), 0, st, to_dx,
                         to_dw);
    HIP_TRY(hipGetLastError());
    Join<T> join_dx{};
    if (dx && v0 + p.piece >= c.V)               // all pieces are in
      join_dx = Join<T>{c.B, int(c.D), p.dx_splits, b.dx, p.Bp * Np, Np, share ? grad : nullptr, share,
                        sizeof(T) == 2 ? b.rest : nullptr, c.of(),
                        static_cast<const T*>(c.w), c.sv, c.sd, static_cast<T*>(dx), lddx, int64_t(1)};
    if (int rc = launch_joins(join_dx, join_dw, st)) return rc;
  }
  return SGNN_OK;
}

#define SGNN_WIDE(KDS, CALL)                         \
  switch (KDS) {                                     \
    case 4: { constexpr int KD = 4; CALL; } break;   \
    case 8: { constexpr int KD = 8; CALL; } break;   \
    case 12: { constexpr int KD = 12; CALL; } break; \
    default: { constexpr int KD = 16; CALL; } break; \
  }

int wide_forward(const Call& c, const Wide& f, const Plan& p, const Buffers& b, RowStat* stats, float* row_loss,
                 float* loss, float* share, hipStream_t st) {
  Operand<Bf16> x, w;
  if (int rc = operands<Bf16>(c, p, b, Rows{}, true, &x, &w, st)) return rc;
  const Labels of = c.of();
  SGNN_WIDE(f.KD, hipLaunchKernelGGL((k_wide_stats<KD>), dim3(unsigned(f.own_b * f.stat_splits)), dim3(kThreads), 0, st,
                                     c.B, c.V, x, w, of, f.steps_v, f.stat_splits, b.part, b.picked));
  HIP_TRY(hipGetLastError());
  return finish_forward(c, f.stat_splits, b, stats, row_loss, loss, share, st);
}

int wide_backward(const Call& c, const Wide& f, const Plan& p, const Buffers& b, const RowStat* stats,
                  const float* grad, const float* share, void* dx, int64_t lddx, void* dw, int64_t dsv, int64_t dsd,
                  hipStream_t st) {
  Operand<Bf16> x, w;
  if (int rc = operands<Bf16>(c, p, b, Rows{c.B, stats, grad, share, b.rows}, true, &x, &w, st)) return rc;
  const Labels of = c.of();
  Join<Bf16> join_dx{}, join_dw{};
  if (dx) {
    SGNN_WIDE(f.KD, hipLaunchKernelGGL((k_wide_grads<KD, false, false>), dim3(unsigned(f.own_b * f.dx_splits)),
                                       dim3(kGradThreads), 0, st, c.B, c.V, x, w, b.rows, f.steps_v, f.dx_splits, b.dx,
                                       c.B * p.Dp, int(c.D), nullptr, 0, 0, nullptr, nullptr));
    HIP_TRY(hipGetLastError());
    join_dx = Join<Bf16>{c.B, int(c.D), f.dx_splits, b.dx, c.B * p.Dp, int64_t(p.Dp), b.rows.factor, nullptr, b.rows.rest,
                         of, static_cast<const Bf16*>(c.w), c.sv, c.sd, static_cast<Bf16*>(dx), lddx, int64_t(1)};
  }
  if (dw) {
    Bf16* const direct = f.dw_splits == 1 ? static_cast<Bf16*>(dw) : nullptr;
#define SGNN_DWEIGHT(PER_ROW)                                                                                           \
  SGNN_WIDE(f.KD, hipLaunchKernelGGL((k_wide_grads<KD, true, PER_ROW>), dim3(unsigned(f.own_v * f.dw_splits)),          \
                                     dim3(kGradThreads), 0, st, c.V, c.B, w, x, b.rows, f.steps_b, f.dw_splits, b.dw,   \
                                     c.V * p.Dp, int(c.D), direct, dsv, dsd, grad, share))
    if (share) {
      SGNN_DWEIGHT(false);
    } else {
      SGNN_DWEIGHT(true);
    }
#undef SGNN_DWEIGHT
    HIP_TRY(hipGetLastError());
    if (!direct)
      join_dw = Join<Bf16>{c.V, int(c.D), f.dw_splits, b.dw, c.V * p.Dp, int64_t(p.Dp), share ? grad : nullptr, share,
                           nullptr, Labels{}, nullptr, 0, 0, static_cast<Bf16*>(dw), dsv, dsd};
  }
  return launch_joins(join_dx, join_dw, st);
}

template <typename T>
int few_forward(const Call& c, const Few& f, const Buffers& b, RowStat* stats, float* row_loss, float* loss,
                float* share, hipStream_t st) {
  const Labels of = c.of();
  if (int rc = allow_lds(reinterpret_cast<const void*>(&k_few_stats<T>), f.lds)) return rc;
  hipLaunchKernelGGL((k_few_stats<T>), dim3(f.blocks), dim3(kThreads), f.lds, st, int(c.B), int(c.D), f.Dk, c.V,
                     static_cast<const T*>(c.x), c.ldx, static_cast<const T*>(c.w), c.sv, of, b.part, b.picked);
  HIP_TRY(hipGetLastError());
  return finish_forward(c, int(f.blocks), b, stats, row_loss, loss, share, st);
}

template <typename T>
int few_backward(const Call& c, const Few& f, const Buffers& b, const RowStat* stats, const float* grad,
                 const float* share, void* dx, int64_t lddx, void* dw, int64_t dsv, int64_t dsd, hipStream_t st) {
  const Labels of = c.of();
  const T* x = static_cast<const T*>(c.x);
  const T* w = static_cast<const T*>(c.w);
  if (int rc = allow_lds(reinterpret_cast<const void*>(&k_few_dz<T>), f.lds)) return rc;
  hipLaunchKernelGGL((k_few_dz<T>), dim3(f.blocks), dim3(kThreads), f.lds, st, int(c.B), f.rows, int(c.D), f.Dk, c.V,
                     x, c.ldx, w, c.sv, of, stats, grad, share, b.dw);
  HIP_TRY(hipGetLastError());
#define SGNN_FEW(ROWS, VEC)                                                                                          \
  hipLaunchKernelGGL((k_few_grads<T, ROWS, VEC>), dim3(f.slabs, f.splits), dim3(kThreads), 0, st, int(c.B), int(c.D), \
                     c.V, x, c.ldx, w, c.sv, of, b.dw, static_cast<T*>(dw), dsv, dsd, dx ? b.dx : nullptr)
  switch (f.rows) {
    case 2: SGNN_FEW(2, 4); break;
    case 4: SGNN_FEW(4, 4); break;
    case 8: SGNN_FEW(8, 4); break;
    case 16: SGNN_FEW(16, 4); break;
    default: SGNN_FEW(32, 2); break;
  }
#undef SGNN_FEW
  HIP_TRY(hipGetLastError());
  if (dx) {
    hipLaunchKernelGGL((k_few_join<T>), dim3(unsigned(c.B), unsigned(ceil_div(c.D, 32))), dim3(kThreads), 0, st, int(c.D),
                       f.rows, int(f.splits), b.dx, of, static_cast<T*>(dx), lddx);
    HIP_TRY(hipGetLastError());
  }
  return SGNN_OK;
}

}  // namespace

extern "C" size_t sgnn_class_xent_workspace_bytes(int dtype, int64_t B, int64_t D, int64_t V, int backward) {
  dtype &= ~SGNN_ALL_ROWS;
  if (B <= 0 || D <= 0 || V <= 0 || (dtype != SGNN_F32 && dtype != SGNN_BF16) || too_large(B, D, V)) return 0;
  // the weight's layout is not known here: enough for either way
  const size_t whole = carve(make_plan(dtype, B, D, V), B, V, backward != 0, nullptr).bytes;
  const Few f = make_few(dtype, B, D, V, 1);
  const size_t few = f.rows ? carve_few(f, B, D, V, backward != 0, nullptr).bytes : 0;
  const Wide wd = make_wide(dtype, B, D, V);
  const size_t plain = wd.KD ? carve_wide(wd, make_plan(dtype, B, D, V), B, V, backward != 0, nullptr).bytes : whole;
  return plain > few ? plain : few;
}

extern "C" int sgnn_class_xent_forward(int dtype, int64_t B, int64_t D, int64_t V, const void* x, int64_t ldx,
                                       const void* weight, int64_t sv, int64_t sd, const int64_t* labels,
                                       int64_t n_labels, const int64_t* idx, float* stats, float* row_loss,
                                       float* loss, float* share, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  using sgnn::fail;
  const Call c{dtype & ~SGNN_ALL_ROWS, B, D, V, x, ldx, weight, sv, sd, labels, n_labels, idx, (dtype & SGNN_ALL_ROWS) != 0};
  dtype = c.dtype;
  if (int rc = check_call(c)) return rc;
  if (!stats || !row_loss || !workspace || (loss && !share)) return fail(SGNN_ERR_INVALID, "null pointer");
  if (workspace_bytes < sgnn_class_xent_workspace_bytes(dtype, B, D, V, 0))
    return fail(SGNN_ERR_WORKSPACE, "class-loss workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  RowStat* s = reinterpret_cast<RowStat*>(stats);
  if (const Few f = make_few(dtype, B, D, V, sd); f.rows) {
    const Buffers b = carve_few(f, B, D, V, false, workspace);
    if (dtype == SGNN_F32) return few_forward<float>(c, f, b, s, row_loss, loss, share, st);
    return few_forward<Bf16>(c, f, b, s, row_loss, loss, share, st);
  }
  const Plan p = make_plan(dtype, B, D, V);
  if (const Wide f = make_wide(dtype, B, D, V); f.KD)
    return wide_forward(c, f, p, carve_wide(f, p, B, V, false, workspace), s, row_loss, loss, share, st);
  const Buffers b = carve(p, B, V, false, workspace);
  if (dtype == SGNN_F32) return forward<float>(c, p, b, s, row_loss, loss, share, st);
  return forward<Bf16>(c, p, b, s, row_loss, loss, share, st);
}

extern "C" int sgnn_class_xent_backward(int dtype, int64_t B, int64_t D, int64_t V, const void* x, int64_t ldx,
                                        const void* weight, int64_t sv, int64_t sd, const int64_t* labels,
                                        int64_t n_labels, const int64_t* idx, const float* stats, const float* grad,
                                        const float* share, void* dx, int64_t lddx, void* dweight, int64_t dsv,
                                        int64_t dsd, void* workspace, size_t workspace_bytes, void* stream) {
  using sgnn::fail;
  const Call c{dtype & ~SGNN_ALL_ROWS, B, D, V, x, ldx, weight, sv, sd, labels, n_labels, idx, (dtype & SGNN_ALL_ROWS) != 0};
  dtype = c.dtype;
  if (int rc = check_call(c)) return rc;
  if (!stats || !grad || !workspace) return fail(SGNN_ERR_INVALID, "null pointer");
  if (dx && lddx < D) return fail(SGNN_ERR_INVALID, "row stride smaller than the width");
  if (dweight && !((dsd == 1 && dsv >= D) || (dsv == 1 && dsd >= V)))
    return fail(SGNN_ERR_INVALID, "the weight's gradient must have unit stride along its features or its classes");
  if (!dx && !dweight) return SGNN_OK;
  if (workspace_bytes < sgnn_class_xent_workspace_bytes(dtype, B, D, V, 1))
    return fail(SGNN_ERR_WORKSPACE, "class-loss workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const RowStat* s = reinterpret_cast<const RowStat*>(stats);
  if (const Few f = make_few(dtype, B, D, V, sd); f.rows) {
    const Buffers b = carve_few(f, B, D, V, true, workspace);
    if (dtype == SGNN_F32) return few_backward<float>(c, f, b, s, grad, share, dx, lddx, dweight, dsv, dsd, st);
    return few_backward<Bf16>(c, f, b, s, grad, share, dx, lddx, dweight, dsv, dsd, st);
  }
  const Plan p = make_plan(dtype, B, D, V);
  if (const Wide f = make_wide(dtype, B, D, V); f.KD)
    return wide_backward(c, f, p, carve_wide(f, p, B, V, true, workspace), s, grad, share, dx, lddx, dweight, dsv, dsd, st);
  const Buffers b = carve(p, B, V, true, workspace);
  if (dtype == SGNN_F32) return backward<float>(c, p, b, s, grad, share, dx, lddx, dweight, dsv, dsd, st);
  return backward<Bf16>(c, p, b, s, grad, share, dx, lddx, dweight, dsv, dsd, st);
}
