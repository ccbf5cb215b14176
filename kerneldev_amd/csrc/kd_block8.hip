// The transformer block's elementwise passes with results in 8-bit blocks
// (kd_block8.h): rows and weights quantised, RMSNorm after the residual's
// addition, the SwiGLU gate; and the backward passes that read what those kept
// in 8 bits instead of the 16-bit activations.
//
// All are bound by memory.  A lane takes 8 values (16 bytes of a 16-bit
// operand), so a block of 128 is a DPP row of 16 lanes and its maximum needs
// four exchanges and no LDS; the values stay in registers between the maximum
// and the rounding, so every operand is read once.
#include <algorithm>

#include "kd_block8.h"

namespace kd {
namespace {

// One operand's 8 values as floats; F32: 32 bytes
template <class E>
KD_DEV void load8(const void* p, int64_t at, float (&f)[8]) {
  unpack8<E>(*reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at), f);
}
template <>
KD_DEV void load8<F32>(const void* p, int64_t at, float (&f)[8]) {
  const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
  const f32x4 u = q[0], v = q[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = u[i], f[4 + i] = v[i];
}
KD_DEV void zero8(float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.f;
}

// x[p], p < 4 (an index into a kernel argument would copy the array to scratch memory)
template <class T>
KD_DEV T pick(const T (&x)[4], int p) {
  return p == 0 ? x[0] : p == 1 ? x[1] : p == 2 ? x[2] : x[3];
}

// The lane's 8 values at column col of row `row` as part of their block, and
// the block's scale byte by its first lane.  All lanes of a DPP row call it
// together; those at or behind column `cols` hold zeros.
KD_DEV void store_block(const float (&f)[8], uint8_t* y, int64_t y_stride, uint8_t* scale, int64_t nb, int64_t row,
                        int col, int cols) {
  const uint32_t b = scale_byte(row16_max(finite_max(f)));
  if (col < y_stride && col < (cols + 15) / 16 * 16)  // (the row's 16-byte words whole: zeros behind its end)
    *reinterpret_cast<u32x2*>(y + row * y_stride + col) = pack_e4m3(f, scale_inverse(b));
  if ((threadIdx.x & 15) == 0 && col < cols) scale[row * nb + col / QB] = uint8_t(b);
}

template <class E>
__global__ __launch_bounds__(256) void k_quant_rows(kd_rows8_args a, int64_t row0, uint32_t blocks, uint32_t nb) {
  const uint32_t blk = blockIdx.x * 16u + (threadIdx.x >> 4);
  const uint32_t r = blk / nb, kb = blk - r * nb;
  const int64_t row = row0 + r;
  const int col = int(kb) * QB + int(threadIdx.x & 15) * 8;
  float f[8];
  zero8(f);
  // the part that holds the column (parts before the last end on a block's edge)
  int p = 0, c = col;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (p == i && i + 1 < a.n && c >= a.cols[i]) c -= a.cols[i], p = i + 1;
  if (blk < blocks && col < a.total) load8<E>(pick(a.x, p), row * pick(a.x_stride, p) + c, f);
  if (blk < blocks) store_block(f, a.y, a.y_stride, a.scale, nb, row, col, a.total);
}

// A workgroup a block of 128 x 128: 16 threads a row, 8 rows a thread; the
// bytes go out as they are, and through LDS transposed.  Byte (r, c) lies at
// row c of the transposed tile, whose rows are 132 bytes so that 16 of them
// start in different banks.
template <class E>
__global__ __launch_bounds__(256) void k_quant_weight(kd_weight8_args a, uint32_t kblocks, uint32_t nblocks) {
  __shared__ uint32_t s_max[4];
  __shared__ __attribute__((aligned(16))) uint8_t s_t[QB * 132];
  const int tid = threadIdx.x, nb = blockIdx.x / kblocks, kb = blockIdx.x - nb * kblocks;
  int part = 0, first = nb * QB;  // rows of the part that holds this block (parts before the last: whole blocks)
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (part == i && i + 1 < a.n && first >= a.rows[i]) first -= a.rows[i], part = i + 1;
  const int rows = min(QB, pick(a.rows, part) - first), col = kb * QB + (tid & 15) * 8;
  float f[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = (tid >> 4) + 16 * i;
    zero8(f[i]);
    if (r < rows && col < a.K) load8<E>(pick(a.w, part), int64_t(first + r) * pick(a.w_stride, part) + col, f[i]);
    m = max(m, finite_max(f[i]));
  }
  m = row16_max(m);
  m = max(m, uint32_t(__shfl_xor(int(m), 16, 64)));
  m = max(m, uint32_t(__shfl_xor(int(m), 32, 64)));
  if ((tid & 63) == 0) s_max[tid >> 6] = m;
  __syncthreads();
  m = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
  const uint32_t b = scale_byte(m);
  const float inv = scale_inverse(b);
  if (tid == 0) {
    a.scale[int64_t(nb) * kblocks + kb] = uint8_t(b);
    if (a.scale_t != nullptr) a.scale_t[int64_t(kb) * nblocks + nb] = uint8_t(b);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = (tid >> 4) + 16 * i;
    const u32x2 w = pack_e4m3(f[i], inv);
    if (r < rows && col < (a.K + 15) / 16 * 16 && col < a.y_stride)
      *reinterpret_cast<u32x2*>(a.y + (int64_t(nb) * QB + r) * a.y_stride + col) = w;
    if (a.yt != nullptr) {
#pragma unroll
      for (int k = 0; k < 8; ++k) s_t[((tid & 15) * 8 + k) * 132 + r] = uint8_t(w[k >> 2] >> (8 * (k & 3)));
    }
  }
  if (a.yt == nullptr) return;  // (uniform)
  __syncthreads();
  const int total16 = (a.total + 15) / 16 * 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = (tid >> 4) + 16 * i, n = (tid & 15) * 8;
    if (kb * QB + k < a.K && nb * QB + n < total16 && nb * QB + n < a.yt_stride) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(s_t + k * 132 + n);
      *reinterpret_cast<u32x2*>(a.yt + int64_t(kb * QB + k) * a.yt_stride + nb * QB + n) = u32x2{p[0], p[1]};
    }
  }
}

// Sum over the WPR waves that share a row
template <int WPR>
KD_DEV float row_sum(float x, float* s_part) {
  x = wave_sum(x);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) x += s_part[i];
  }
  return x;
}

// s = x + delta rounded to its type (what the next layer adds to), y = s
// rsqrt(mean(s^2) + eps) in 8 bits.  WPR waves a row, lane l of the row holds the
// 8-value words l, l + 64 WPR, ...: the row stays in registers.
template <class E, int NCH, int WPR>
__global__ __launch_bounds__(256) void k_norm8(kd_norm8_args a, int64_t row0, int64_t end) {
  __shared__ float s_part[4];
  const int lane = threadIdx.x & (64 * WPR - 1);
  const int64_t at = row0 + int64_t(blockIdx.x) * (4 / WPR) + threadIdx.x / (64 * WPR);
  const int64_t row = at < end ? at : end - 1;  // (a wave without a row follows the last, storing nothing)
  const bool live = at < end;
  const int words = a.D / 8;
  const u32x4 *x = static_cast<const u32x4*>(a.x) + row * words, *d = static_cast<const u32x4*>(a.delta) + row * words;
  float f[NCH][8], sum = 0.f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int w = lane + 64 * WPR * c;
    unpack8<E>(w < words ? x[w] : u32x4{}, f[c]);
  }
  if (a.delta != nullptr) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int w = lane + 64 * WPR * c;
      float g[8];
      unpack8<E>(w < words ? d[w] : u32x4{}, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[c][i] += g[i];
      const u32x4 s = pack8<E>(f[c]);
      if (live && w < words) static_cast<u32x4*>(a.sum)[row * words + w] = s;
      unpack8<E>(s, f[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(f[c][i], f[c][i], sum);
  const float r = 1.f / sqrtf(row_sum<WPR>(sum, s_part) / float(a.D) + a.eps);
  if (live && lane == 0 && a.rstd != nullptr) a.rstd[row] = r;
  const int64_t nb = (a.D + QB - 1) / QB;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[c][i] *= r;
    if (live) store_block(f[c], a.y, a.y_stride, a.scale, nb, row, (lane + 64 * WPR * c) * 8, a.D);
  }
}

// dx = ds + r (g - y mean(g y)), y from its 8 bits; g in E or (EG) fp32
template <class E, class EG, int NCH, int WPR>
__global__ __launch_bounds__(256) void k_norm8_bwd(kd_norm8_bwd_args a, int64_t row0, int64_t end) {
  __shared__ float s_part[4];
  const int lane = threadIdx.x & (64 * WPR - 1);
  const int64_t at = row0 + int64_t(blockIdx.x) * (4 / WPR) + threadIdx.x / (64 * WPR);
  const int64_t row = at < end ? at : end - 1;
  const int words = a.D / 8;
  const int64_t nb = (a.D + QB - 1) / QB;
  float f[NCH][8], g[NCH][8], dot = 0.f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int w = lane + 64 * WPR * c;
    zero8(g[c]);
    if (w < words) load8<EG>(a.g, row * a.D + 8 * w, g[c]);
    unpack_e4m3(w < words ? *reinterpret_cast<const u32x2*>(a.y + row * a.y_stride + 8 * w) : u32x2{}, f[c]);
    const float s = w < words ? scale_value(a.scale[row * nb + w / 16]) : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[c][i] *= s;
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) dot = __builtin_fmaf(f[c][i], g[c][i], dot);
  const float r = a.rstd[row], m = row_sum<WPR>(dot, s_part) / float(a.D);
  if (at >= end) return;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int w = lane + 64 * WPR * c;
    float s[8];
    zero8(s);
    if (a.ds != nullptr) unpack8<E>(w < words ? (static_cast<const u32x4*>(a.ds) + row * words)[w] : u32x4{}, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[c][i] = s[i] + r * (g[c][i] - f[c][i] * m);
    if (w < words) static_cast<u32x4*>(a.dx)[row * words + w] = pack8<E>(g[c]);
  }
}

KD_DEV float sigmoid8(float x) { return 1.f / (1.f + fast_exp2(x * -1.4426950408889634f)); }

// y = silu(a) b, and a and b themselves, in 8 bits
template <class E>
__global__ __launch_bounds__(256) void k_gate8(kd_gate8_args g, int64_t row0, uint32_t blocks, uint32_t nb) {
  const uint32_t blk = blockIdx.x * 16u + (threadIdx.x >> 4);
  const uint32_t r = blk / nb, kb = blk - r * nb;
  const int64_t row = row0 + r;
  const int col = int(kb) * QB + int(threadIdx.x & 15) * 8;
  float a[8], b[8], y[8];
  zero8(a), zero8(b);
  if (blk < blocks && col < g.H) load8<E>(g.a, row * g.a_stride + col, a), load8<E>(g.b, row * g.b_stride + col, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = a[i] * sigmoid8(a[i]) * b[i];
  if (blk >= blocks) return;  // (whole DPP rows)
  store_block(y, g.y8, g.stride, g.y_scale, nb, row, col, g.H);
  if (g.a8 == nullptr) return;
  store_block(a, g.a8, g.stride, g.a_scale, nb, row, col, g.H);
  store_block(b, g.b8, g.stride, g.b_scale, nb, row, col, g.H);
}

// da = dy b s (1 + a (1 - s)), db = dy a s, s = sigmoid(a); a and b from their 8 bits
template <class E, class EG>
__global__ __launch_bounds__(256) void k_gate8_bwd(kd_gate8_args g, int64_t row0, uint32_t words_all, uint32_t words,
                                                   uint32_t nb) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= words_all) return;
  const uint32_t r = i / words, w = i - r * words;
  const int64_t row = row0 + r, at = row * g.H + w * 8;
  float a[8], b[8], d[8], da[8], db[8];
  unpack_e4m3(*reinterpret_cast<const u32x2*>(g.a8 + row * g.stride + w * 8), a);
  unpack_e4m3(*reinterpret_cast<const u32x2*>(g.b8 + row * g.stride + w * 8), b);
  load8<EG>(g.dy, at, d);
  const float sa = scale_value(g.a_scale[row * nb + w / 16]), sb = scale_value(g.b_scale[row * nb + w / 16]);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float u = a[k] * sa, v = b[k] * sb, s = sigmoid8(u);
    da[k] = d[k] * v * s * (1.f + u * (1.f - s));
    db[k] = d[k] * (u * s);
  }
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(g.da) + at) = pack8<E>(da);
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(g.db) + at) = pack8<E>(db);
}

template <class F>
int by_type(int dtype, F f) {
  if (dtype == KD_BF16) f(BF16{});
  else f(F16{});
  return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
}

// Rows in launches of less than 2^32 threads each, `per` threads a row: f(first, rows)
template <class F>
void in_launches(int64_t rows, int64_t per, F f) {
  const int64_t most = std::max<int64_t>(4, (int64_t(1) << 31) / per / 4 * 4);
  for (int64_t r = 0; r < rows; r += most) f(r, std::min(most, rows - r));
}

template <class E, class G>
void norm_variant(int D, G go) {  // waves a row and words a lane
  const int words = D / 8;
  using one = std::integral_constant<int, 1>;
  using two = std::integral_constant<int, 2>;
  using four = std::integral_constant<int, 4>;
  if (words <= 64) go(one{}, one{});
  else if (words <= 128) go(two{}, one{});
  else if (words <= 256) go(four{}, one{});
  else if (words <= 512) go(two{}, four{});
  else go(four{}, four{});
}

}  // namespace

int launch_quant_rows(const kd_rows8_args& a, hipStream_t st) {
  const uint32_t nb = uint32_t((a.total + QB - 1) / QB);
  auto go = [&](auto e) {
    in_launches(a.rows, 16 * int64_t(nb), [&](int64_t r, int64_t n) {
      const uint32_t blocks = uint32_t(n) * nb;
      hipLaunchKernelGGL(k_quant_rows<decltype(e)>, dim3((blocks + 15) / 16), dim3(256), 0, st, a, r, blocks, nb);
    });
  };
  if (a.dtype == KD_F32) {
    go(F32{});
    return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
  }
  return by_type(a.dtype, go);
}

int launch_quant_weight(const kd_weight8_args& a, hipStream_t st) {
  const uint32_t kb = uint32_t((a.K + QB - 1) / QB), nb = uint32_t((a.total + QB - 1) / QB);
  auto go = [&](auto e) {
    hipLaunchKernelGGL(k_quant_weight<decltype(e)>, dim3(kb * nb), dim3(256), 0, st, a, kb, nb);
  };
  if (a.dtype == KD_F32) {
    go(F32{});
    return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
  }
  return by_type(a.dtype, go);
}

int launch_norm8(const kd_norm8_args& a, hipStream_t st) {
  return by_type(a.dtype, [&](auto e) {
    using E = decltype(e);
    norm_variant<E>(a.D, [&](auto nch, auto wpr) {
      constexpr int W = decltype(wpr)::value;
      in_launches(a.rows, 64 * W, [&](int64_t r, int64_t n) {
        hipLaunchKernelGGL((k_norm8<E, decltype(nch)::value, W>), dim3(unsigned((n * W + 3) / 4)), dim3(256), 0, st, a, r,
                           r + n);
      });
    });
  });
}

int launch_norm8_bwd(const kd_norm8_bwd_args& a, hipStream_t st) {
  return by_type(a.dtype, [&](auto e) {
    using E = decltype(e);
    norm_variant<E>(a.D, [&](auto nch, auto wpr) {
      constexpr int W = decltype(wpr)::value;
      in_launches(a.rows, 64 * W, [&](int64_t r, int64_t n) {
        auto k = a.g_dtype == KD_F32 ? k_norm8_bwd<E, F32, decltype(nch)::value, W> : k_norm8_bwd<E, E, decltype(nch)::value, W>;
        hipLaunchKernelGGL(k, dim3(unsigned((n * W + 3) / 4)), dim3(256), 0, st, a, r, r + n);
      });
    });
  });
}

int launch_gate8(const kd_gate8_args& a, hipStream_t st) {
  const uint32_t nb = uint32_t((a.H + QB - 1) / QB);
  return by_type(a.dtype, [&](auto e) {
    in_launches(a.rows, 16 * int64_t(nb), [&](int64_t r, int64_t n) {
      const uint32_t blocks = uint32_t(n) * nb;
      hipLaunchKernelGGL(k_gate8<decltype(e)>, dim3((blocks + 15) / 16), dim3(256), 0, st, a, r, blocks, nb);
    });
  });
}

int launch_gate8_bwd(const kd_gate8_args& a, hipStream_t st) {
  const uint32_t nb = uint32_t((a.H + QB - 1) / QB), words = uint32_t(a.H / 8);
  return by_type(a.dtype, [&](auto e) {
    in_launches(a.rows, int64_t(words), [&](int64_t r, int64_t n) {
      const uint32_t all = uint32_t(n) * words;
      auto k = a.dy_dtype == KD_F32 ? k_gate8_bwd<decltype(e), F32> : k_gate8_bwd<decltype(e), decltype(e)>;
      hipLaunchKernelGGL(k, dim3((all + 255) / 256), dim3(256), 0, st, a, r, all, words, nb);
    });
  });
}

}  // namespace kd
