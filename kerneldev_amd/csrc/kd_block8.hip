// The transformer block's elementwise passes with results in 8-bit blocks
// (kd_block8.h): rows and weights quantised, RMSNorm after the residual's
// addition, the SwiGLU gate; and the backward passes that read what those kept
// in 8 bits instead of the 16-bit activations.
//
// All are bound by memory.  A lane takes 8 values (16 bytes of a 16-bit
// operand), so a block of 128 is a DPP row of 16 lanes and its maximum needs
// four exchanges and no LDS; the values stay in registers between the maximum
// and the rounding, so every operand is read once.  At 16384 rows, bf16, with what
// a pass has to read and write (a 64 MiB copy reaches 7.2 TB/s here, one of 1 GiB 5.1):
//   rows of 2304 quantised     20 us  5.6 TB/s
//   norm after addition, 768   16 us  5.5 TB/s, its backward 15 us  5.9 TB/s
//   gate kept, 2048            43 us  5.5 TB/s, its backward 46 us  5.8 TB/s
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

// The scale's byte and the e4m3 bytes of the lane's 8 values, the block's lanes (a
// DPP row) together.  Blocks that hold a NaN or an infinity take the longer way, and
// with them their wave.
KD_DEV u32x2 quantise(const float (&f)[8], uint32_t* byte) {
  uint32_t m = row16_max(any_max(f));
  if (__builtin_amdgcn_ballot_w64(m >= 0x7F800000u) != 0) {
    *byte = scale_byte(row16_max(finite_max(f)));
    return pack_e4m3(f, scale_inverse(*byte));
  }
  *byte = scale_byte(m);
  return pack_finite(f, scale_value(*byte));
}
template <class E>
KD_DEV u32x2 quantise(const u32x4& v, uint32_t* byte) {
  constexpr bool B = std::is_same_v<E, BF16>;
  const uint32_t m = row16_max(any_max(v));
  float f[8];
  unpack8<E>(v, f);
  if (__builtin_amdgcn_ballot_w64(m >= (B ? 0x7F80u : 0x7C00u)) != 0) {
    *byte = scale_byte(row16_max(finite_max(f)));
    return pack_e4m3(f, scale_inverse(*byte));
  }
  *byte = scale_byte(B ? m << 16 : __float_as_uint(to_f32<E>(uint16_t(m))));
  return pack_finite(f, scale_value(*byte));
}

// Results of 16 MiB and more pass by the L2, which holds 32 (us, through it and past
// it, sizes as above: rows 24.1 and 20.1, norm 18.3 and 15.5, its backward 16.2 and 14.8,
// gate 45.0 and 42.6, its backward 48.6 and 46.1); smaller ones are read from it at once.
constexpr int64_t PAST_BYTES = int64_t(1) << 24;
template <class V>
KD_DEV void put(V* p, const V& v, bool past) {
  if (past) __builtin_nontemporal_store(v, p);
  else *p = v;
}

// The lane's 8 values at column col of row `row` as part of their block, and
// the block's scale byte by its first lane.  All lanes of a DPP row call it
// together; those at or behind column `cols` hold zeros.
KD_DEV void store_bytes(const u32x2& w, uint32_t byte, uint8_t* y, int64_t y_stride, uint8_t* scale, int64_t nb, int64_t row,
                        int col, int cols, bool past) {
  if (col < (cols + 15) / 16 * 16)  // (the row's 16-byte words whole: zeros behind its end)
    put(reinterpret_cast<u32x2*>(y + row * y_stride + col), w, past);
  if ((threadIdx.x & 15) == 0 && col < cols) scale[row * nb + col / QB] = uint8_t(byte);
}
KD_DEV void store_block(const float (&f)[8], uint8_t* y, int64_t y_stride, uint8_t* scale, int64_t nb, int64_t row,
                        int col, int cols, bool past) {
  uint32_t b;
  const u32x2 w = quantise(f, &b);
  store_bytes(w, b, y, y_stride, scale, nb, row, col, cols, past);
}
template <class E>
KD_DEV void store_block(const u32x4& v, uint8_t* y, int64_t y_stride, uint8_t* scale, int64_t nb, int64_t row, int col,
                        int cols, bool past) {
  uint32_t b;
  const u32x2 w = quantise<E>(v, &b);
  store_bytes(w, b, y, y_stride, scale, nb, row, col, cols, past);
}

// U blocks a DPP row of lanes, 16 apart: their loads go out together
template <class E, int U>
__global__ __launch_bounds__(256) void k_quant_rows(kd_rows8_args a, int64_t row0, uint32_t blocks, uint32_t nb, bool past) {
  u32x4 v[U], hi[U];
  int64_t row[U];
  int col[U];
  const uint32_t blk0 = blockIdx.x * (16u * U) + (threadIdx.x >> 4);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t blk = min(blk0 + 16u * u, blocks - 1), r = blk / nb, kb = blk - r * nb;  // (behind the last: the last)
    row[u] = row0 + r, col[u] = int(kb) * QB + int(threadIdx.x & 15) * 8;
    // the part that holds the column (parts before the last end on a block's edge)
    const void* x = a.x[0];
    int64_t stride = a.x_stride[0];
    int c = col[u], cols = a.cols[0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (i < a.n && c >= cols) c -= cols, x = a.x[i], stride = a.x_stride[i], cols = a.cols[i];
    const int64_t at = row[u] * stride + c;
    v[u] = hi[u] = u32x4{};
    if (col[u] < a.total) {
      if constexpr (std::is_same_v<E, F32>) {
        const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const float*>(x) + at);
        v[u] = p[0], hi[u] = p[1];
      } else {
        v[u] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(x) + at);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (blk0 + 16u * u >= blocks) return;  // (whole DPP rows)
    if constexpr (std::is_same_v<E, F32>) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[u][i]), f[4 + i] = __uint_as_float(hi[u][i]);
      store_block(f, a.y, a.y_stride, a.scale, nb, row[u], col[u], a.total, past);
    } else {
      store_block<E>(v[u], a.y, a.y_stride, a.scale, nb, row[u], col[u], a.total, past);
    }
  }
}

// The bytes of a 4 x 4 block turned over: word j of the result holds byte j of the four words
KD_DEV void turn4(const uint32_t (&r)[4], uint32_t (&c)[4]) {
  const uint32_t t0 = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), t1 = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u),
                 t2 = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u), t3 = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
  c[0] = __builtin_amdgcn_perm(t1, t0, 0x05040100u), c[1] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
  c[2] = __builtin_amdgcn_perm(t3, t2, 0x05040100u), c[3] = __builtin_amdgcn_perm(t3, t2, 0x07060302u);
}

// A workgroup a block of 128 x 128, a thread 4 rows of 8 columns: the bytes go out
// as they are and, turned over in registers, transposed.  Latency bounds it (a
// model's weight is some hundred blocks): one round of loads, one exchange of the
// maximum (2304 x 768: 8.0 us, with 256 threads of 8 rows 10.5).
template <class E>
__global__ __launch_bounds__(512) void k_quant_weight(kd_weight8_args a, uint32_t kblocks, uint32_t nblocks) {
  __shared__ uint32_t s_max[8];
  const int tid = threadIdx.x, nb = blockIdx.x / kblocks, kb = blockIdx.x - nb * kblocks;
  const void* src = a.w[0];  // the part that holds this block (parts before the last: whole blocks)
  int64_t stride = a.w_stride[0];
  int first = nb * QB, height = a.rows[0];
#pragma unroll
  for (int i = 1; i < 4; ++i)
    if (i < a.n && first >= height) first -= height, src = a.w[i], stride = a.w_stride[i], height = a.rows[i];
  const int rows = min(QB, height - first), r0 = (tid >> 4) * 4, col = kb * QB + (tid & 15) * 8;
  float f[4][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    zero8(f[i]);
    if (r0 + i < rows && col < a.K) load8<E>(src, int64_t(first + r0 + i) * stride + col, f[i]);
  }
  auto block_max = [&](uint32_t v) {
    v = row16_max(v);
    v = max(v, uint32_t(__shfl_xor(int(v), 16, 64)));
    v = max(v, uint32_t(__shfl_xor(int(v), 32, 64)));
    if ((tid & 63) == 0) s_max[tid >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) v = max(v, s_max[i]);
    return v;
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, any_max(f[i]));
  m = block_max(m);
  const bool finite = m < 0x7F800000u;  // (the same in every thread; blocks that hold a NaN or an infinity take the longer way)
  if (!finite) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, finite_max(f[i]));
    __syncthreads();  // (the maxima above are read)
    m = block_max(m);
  }
  const uint32_t b = scale_byte(m);
  if (tid == 0) {
    a.scale[int64_t(nb) * kblocks + kb] = uint8_t(b);
    if (a.scale_t != nullptr) a.scale_t[int64_t(kb) * nblocks + nb] = uint8_t(b);
  }
  u32x2 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = finite ? pack_finite(f[i], scale_value(b)) : pack_e4m3(f[i], scale_inverse(b));
    if (r0 + i < rows && col < (a.K + 15) / 16 * 16)
      *reinterpret_cast<u32x2*>(a.y + (int64_t(nb) * QB + r0 + i) * a.y_stride + col) = w[i];
  }
  if (a.yt == nullptr || nb * QB + r0 >= (a.total + 15) / 16 * 16) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t t[4];
    turn4({w[0][h], w[1][h], w[2][h], w[3][h]}, t);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + 4 * h + j < a.K) *reinterpret_cast<uint32_t*>(a.yt + int64_t(col + 4 * h + j) * a.yt_stride + nb * QB + r0) = t[j];
  }
}

// Sum over the WPR waves that share a row
template <int WPR, class T>
KD_DEV T row_sum(T x, T* s_part) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int i = 0; i < WPR; ++i) x += s_part[i];
  }
  return x;
}

// s = x + delta rounded to its type (what the next layer adds to), y = s
// rsqrt(mean(s^2) + eps) in 8 bits.  WPR waves a row, lane l of the row holds the
// 8-value words l, l + 64 WPR, ...: the row stays in registers.  The sum of
// squares and its root are formed in 64 bits and y = s r with r as two floats: y is
// the exact value's fp32 rounding, nearly always, and its 8 bits those of the exact
// value (rounded from an fp32 root, some ten of 10^7 were not).  Memory bounds it all
// the same.
template <class E, int NCH, int WPR>
__global__ __launch_bounds__(256) void k_norm8(kd_norm8_args a, int64_t row0, int64_t end, bool past) {
  __shared__ double s_part[4];
  const int lane = threadIdx.x & (64 * WPR - 1);
  const int64_t at = row0 + int64_t(blockIdx.x) * (4 / WPR) + threadIdx.x / (64 * WPR);
  const int64_t row = at < end ? at : end - 1;  // (a wave without a row follows the last, storing nothing)
  const bool live = at < end;
  const int words = a.D / 8;
  const u32x4 *x = static_cast<const u32x4*>(a.x) + row * words, *d = static_cast<const u32x4*>(a.delta) + row * words;
  float f[NCH][8];
  double sum = 0.0;
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
      if (live && w < words) put(static_cast<u32x4*>(a.sum) + row * words + w, s, past);
      unpack8<E>(s, f[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fma(double(f[c][i]), double(f[c][i]), sum);
  const double v = row_sum<WPR>(sum, s_part) / double(a.D) + double(a.eps);
  const double g = double(1.f / sqrtf(float(v))), root = g * (1.5 - 0.5 * v * g * g);  // one step of Newton's
  const bool fine = g > 0.0 && g < double(__builtin_inff());                           // (else 0, infinite or NaN, as g is)
  const float r = fine ? float(root) : float(g), rest = fine ? float(root - double(r)) : 0.f;
  if (live && lane == 0 && a.rstd != nullptr) a.rstd[row] = r;
  const int64_t nb = (a.D + QB - 1) / QB;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[c][i] = __builtin_fmaf(f[c][i], r, f[c][i] * rest);
    if (live) store_block(f[c], a.y, a.y_stride, a.scale, nb, row, (lane + 64 * WPR * c) * 8, a.D, past);
  }
}

// dx = ds + r (g - y mean(g y)), y from its 8 bits; g in E or (EG) fp32
template <class E, class EG, int NCH, int WPR>
__global__ __launch_bounds__(256) void k_norm8_bwd(kd_norm8_bwd_args a, int64_t row0, int64_t end, bool past) {
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
    if (w < words) put(static_cast<u32x4*>(a.dx) + row * words + w, pack8<E>(g[c]), past);
  }
}

// (the reciprocal within 1 ulp; of infinity 0)
KD_DEV float sigmoid8(float x) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(x * -1.4426950408889634f)); }

// y = silu(a) b, and a and b themselves, in 8 bits
template <class E>
__global__ __launch_bounds__(256) void k_gate8(kd_gate8_args g, int64_t row0, uint32_t blocks, uint32_t nb, bool past) {
  const uint32_t blk = blockIdx.x * 16u + (threadIdx.x >> 4);
  const uint32_t r = blk / nb, kb = blk - r * nb;
  const int64_t row = row0 + r;
  const int col = int(kb) * QB + int(threadIdx.x & 15) * 8;
  if (blk >= blocks) return;  // (whole DPP rows)
  u32x4 va{}, vb{};
  if (col < g.H) {
    va = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(g.a) + row * g.a_stride + col);
    vb = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(g.b) + row * g.b_stride + col);
  }
  float a[8], b[8], y[8];
  unpack8<E>(va, a), unpack8<E>(vb, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = a[i] * sigmoid8(a[i]) * b[i];
  store_block(y, g.y8, g.stride, g.y_scale, nb, row, col, g.H, past);
  if (g.a8 == nullptr) return;
  store_block<E>(va, g.a8, g.stride, g.a_scale, nb, row, col, g.H, past);
  store_block<E>(vb, g.b8, g.stride, g.b_scale, nb, row, col, g.H, past);
}

// da = dy b s (1 + a (1 - s)), db = dy a s, s = sigmoid(a); a and b from their 8 bits
template <class E, class EG>
__global__ __launch_bounds__(256) void k_gate8_bwd(kd_gate8_args g, int64_t row0, uint32_t words_all, uint32_t words,
                                                   uint32_t nb, bool past) {
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
  put(reinterpret_cast<u32x4*>(static_cast<uint16_t*>(g.da) + at), pack8<E>(da), past);
  put(reinterpret_cast<u32x4*>(static_cast<uint16_t*>(g.db) + at), pack8<E>(db), past);
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

// Two blocks a thread where there are many, 16 bits (us, one and two): 16384 x 2304 26.9 and 24.2, 16384 x 768 8.8 and
// 8.3, but 2048 x 768 2.6 and 2.9, 633 x 1000 2.3 and 2.7; four 27.3, 9.1, 3.9, 3.9.  fp32: 16384 x 768 11.4 and 11.7.
int launch_quant_rows(const kd_rows8_args& a, hipStream_t st) {
  const uint32_t nb = uint32_t((a.total + QB - 1) / QB);
  const bool past = a.rows * a.total >= PAST_BYTES;
  auto go = [&](auto e, auto u) {
    constexpr int U = decltype(u)::value;
    in_launches(a.rows, 16 * int64_t(nb), [&](int64_t r, int64_t n) {
      const uint32_t blocks = uint32_t(n) * nb;
      hipLaunchKernelGGL((k_quant_rows<decltype(e), U>), dim3((blocks + 16 * U - 1) / (16 * U)), dim3(256), 0, st, a, r, blocks, nb, past);
    });
  };
  using one = std::integral_constant<int, 1>;
  using two = std::integral_constant<int, 2>;
  if (a.dtype == KD_F32) {
    go(F32{}, one{});
    return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
  }
  return by_type(a.dtype, [&](auto e) { a.rows * nb >= (1 << 16) ? go(e, two{}) : go(e, one{}); });
}

int launch_quant_weight(const kd_weight8_args& a, hipStream_t st) {
  const uint32_t kb = uint32_t((a.K + QB - 1) / QB), nb = uint32_t((a.total + QB - 1) / QB);
  auto go = [&](auto e) {
    hipLaunchKernelGGL(k_quant_weight<decltype(e)>, dim3(kb * nb), dim3(512), 0, st, a, kb, nb);
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
                           r + n, a.rows * a.D * (a.delta != nullptr ? 3 : 1) >= PAST_BYTES);
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
        hipLaunchKernelGGL(k, dim3(unsigned((n * W + 3) / 4)), dim3(256), 0, st, a, r, r + n, 2 * a.rows * a.D >= PAST_BYTES);
      });
    });
  });
}

int launch_gate8(const kd_gate8_args& a, hipStream_t st) {
  const uint32_t nb = uint32_t((a.H + QB - 1) / QB);
  return by_type(a.dtype, [&](auto e) {
    in_launches(a.rows, 16 * int64_t(nb), [&](int64_t r, int64_t n) {
      const uint32_t blocks = uint32_t(n) * nb;
      hipLaunchKernelGGL(k_gate8<decltype(e)>, dim3((blocks + 15) / 16), dim3(256), 0, st, a, r, blocks, nb,
                         a.rows * a.H * (a.a8 != nullptr ? 3 : 1) >= PAST_BYTES);
    });
  });
}

int launch_gate8_bwd(const kd_gate8_args& a, hipStream_t st) {
  const uint32_t nb = uint32_t((a.H + QB - 1) / QB), words = uint32_t(a.H / 8);
  return by_type(a.dtype, [&](auto e) {
    in_launches(a.rows, int64_t(words), [&](int64_t r, int64_t n) {
      const uint32_t all = uint32_t(n) * words;
      auto k = a.dy_dtype == KD_F32 ? k_gate8_bwd<decltype(e), F32> : k_gate8_bwd<decltype(e), decltype(e)>;
      hipLaunchKernelGGL(k, dim3((all + 255) / 256), dim3(256), 0, st, a, r, all, words, nb, 4 * a.rows * a.H >= PAST_BYTES);
    });
  });
}

}  // namespace kd
