// Weight gradients of the block's projections: dW [N, K] = dY^T X over M
// tokens, dY [M, N] and X [M, K] in bf16 or fp16, row-major.
//
// The contraction runs over the tokens, the slow dimension of both operands,
// and the result is small (768 x 768 .. 2048 x 768 against 16384 tokens), so a
// product needs its tokens split to fill the chip.  A workgroup takes 128 x 128
// of dW over one piece of the tokens: 64 tokens a step of both operands go to
// LDS (two slots of 2 x 16 KiB, so two workgroups share a CU), and both MFMA
// operands are read transposed from there (ds_read_b64_tr_b16), four waves
// taking 64 x 64 each: one operand read a MFMA, at which the LDS keeps the
// matrix cores about three quarters busy.  The pieces' fp32 results are added
// in ascending order by a second kernel and rounded once.  Items are
// piece-major, so an XCD's workgroups read the same tokens through its L2.
#include <algorithm>
#include <cmath>

#include "kd_block8.h"

namespace kd {
namespace {

constexpr int WT = 128;  // rows and columns of dW a workgroup takes

struct WgradArgs {
  const void *dy, *x;
  float* part;      // [S][N][K]
  int M, N, K, S;   // S pieces of the tokens
  int tn, tk;       // tiles of dW
};

template <class E>
__global__ __launch_bounds__(256, 2) void k_wgrad(WgradArgs w) {
  using TL = Tile<WT, 4>;
  __shared__ __attribute__((aligned(1024))) uint8_t s_y[2][TL::BYTES];
  __shared__ __attribute__((aligned(1024))) uint8_t s_x[2][TL::BYTES];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hf = lane >> 5,
            c = lane & 31;
  const int item = xcd_remap(blockIdx.x, gridDim.x), tiles = w.tn * w.tk;
  const int piece = item / tiles, tile = item - piece * tiles;
  const int n0 = (tile / w.tk) * WT, k0 = (tile - (tile / w.tk) * w.tk) * WT;
  const int steps_all = (w.M + 63) / 64;
  const int e0 = int(int64_t(steps_all) * piece / w.S), e1 = int(int64_t(steps_all) * (piece + 1) / w.S);
  const uint32_t yrb = uint32_t(w.N) * 2u, xrb = uint32_t(w.K) * 2u;
  const u32x4 rs_y = rsrc_words(w.dy, uint32_t(w.M) * yrb), rs_x = rsrc_words(w.x, uint32_t(w.M) * xrb);
  uint32_t yoff[TL::LOADS_PER_WAVE], xoff[TL::LOADS_PER_WAVE];  // (columns past N, K read as zeros)
  TL::load_offsets(wave, lane, yrb, yoff, yrb - uint32_t(n0) * 2u);
  TL::load_offsets(wave, lane, xrb, xoff, xrb - uint32_t(k0) * 2u);
  auto load = [&](int e, int slot) {
    TL::load_async(rs_y, uint32_t(e) * 64u * yrb + uint32_t(n0) * 2u, yoff, lds_addr(s_y[slot]), wave);
    TL::load_async(rs_x, uint32_t(e) * 64u * xrb + uint32_t(k0) * 2u, xoff, lds_addr(s_x[slot]), wave);
  };
  // this wave's 64 x 64: column blocks 2 wn, 2 wn + 1 of the dY tile against 2 wk, 2 wk + 1 of the X tile
  const int wn = wave >> 1, wk = wave & 1;
  int ya[2][2], xa[2][2];  // transposed-read offsets [column block][half], a k-step adds 16 rows
  {
    const int i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = 8 * (g >> 1) + 4 * half + (i >> 2), ch = 2 * (g & 1) + ((i & 3) >> 1);
        ya[b][half] = TL::at(r, 4 * (2 * wn + b) + ch) + 8 * (i & 1);
        xa[b][half] = TL::at(r, 4 * (2 * wk + b) + ch) + 8 * (i & 1);
      }
  }
  f32x16 acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) acc[a][b] = f32x16{};

  if (e0 < e1) load(e0, 0);
  auto step = [&](int e, auto slot_c) {
    constexpr int slot = decltype(slot_c)::value;
    wait_vmem();
    barrier_raw();  // step e's tiles landed for every wave; every wave is done with the other slot
    if (e + 1 < e1) load(e + 1, slot ^ 1);
    lds_u8 *ty = to_lds(s_y[slot]), *tx = to_lds(s_x[slot]);
    auto read = [&](lds_u8* t, const int (&at)[2], int ks) {
      const u32x2 lo = ds_read_tr16(t + at[0] + ks * 16 * TL::ROWB);
      const u32x2 hi = ds_read_tr16(t + at[1] + ks * 16 * TL::ROWB);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    // operands of k-step ks + 1 are read before the MFMAs of k-step ks
    u32x4 av[2][2], bv[2][2];  // [k-step parity][block]
#pragma unroll
    for (int b = 0; b < 2; ++b) av[0][b] = read(ty, ya[b], 0), bv[0][b] = read(tx, xa[b], 0);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      __builtin_amdgcn_sched_barrier(0x406);
      if (ks + 1 < 4) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
          av[(ks + 1) & 1][b] = read(ty, ya[b], ks + 1), bv[(ks + 1) & 1][b] = read(tx, xa[b], ks + 1);
      }
      __builtin_amdgcn_sched_barrier(0x406);
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = mfma32x32x16<E>(av[ks & 1][a], bv[ks & 1][b], acc[a][b]);
    }
    __builtin_amdgcn_sched_barrier(0x406);
  };
  for (int e = e0; e < e1; e += 2) {
    step(e, std::integral_constant<int, 0>{});
    if (e + 1 < e1) step(e + 1, std::integral_constant<int, 1>{});
  }
  float* out = w.part + int64_t(piece) * w.N * w.K;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int k = k0 + 64 * wk + 32 * b + c;
#pragma unroll
      for (int r = 0; r < 16; ++r) {  // register r: row 8 (r / 4) + 4 hf + r % 4 of the 32 x 32 block
        const int n = n0 + 64 * wn + 32 * a + 8 * (r >> 2) + 4 * hf + (r & 3);
        if (n < w.N && k < w.K) out[int64_t(n) * w.K + k] = acc[a][b][r];
      }
    }
}

// dW = the pieces' sum, rounded once; four elements a thread (N K is a multiple of 64)
template <class E>
__global__ __launch_bounds__(256) void k_wgrad_sum(const float* __restrict__ part, uint16_t* __restrict__ dw, int64_t n,
                                                   int S) {
  const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  f32x4 f{};
#pragma unroll 8
  for (int s = 0; s < S; ++s) f += *reinterpret_cast<const f32x4*>(part + s * n + i);
  *reinterpret_cast<u32x2*>(dw + i) = u32x2{pack2<E>(f[0], f[1]), pack2<E>(f[2], f[3])};
}

// The same with X in 8-bit blocks (kd_block8.h), the checkpoint that a forward
// kept: dW [N, K] = dY^T X, dY in up to four parts side by side.  X's values are
// multiplied out to bf16 on their way -- exactly, 4 bits and a power of two -- and
// lie in the LDS as the 16-bit kernel's copy would have put them.  A dY in fp16
// enters as two bf16 (8 + 8 of its 11 bits), since X's range does not fit fp16.
//
// Four waves take 256 x 256 of dW over a piece of the tokens, 128 x 128 each, whose
// sums fill half of a wave's registers: half an operand read a product, at which the
// LDS is half as busy as the matrix cores, and half the copies of a 128 x 128 tile.
// One wave a SIMD has nothing to hide behind, so a step of 32 tokens is one basic
// block in which reads, copies and X's widening stand between the products that
// cover them: the first 16 tokens' products cover the reads of the second 16 and X's
// widening for the next step, the second 16's the next step's first reads, after the
// step's one barrier.  dY and X's bytes are on their way two to three steps ahead.
// What bounds it: of 4096^3's 140 us (0.98 PFLOP/s; the library's bf16 product of that
// shape 131, a 128 x 128 tile with two workgroups a CU 183) the products alone take
// 76, reads add 17, copies 17, the widening 9, the results and their sum 20.  Few
// tokens pay for the large tile: 633 by 1000 x 528 17.5 us, 128 x 128 13.
struct Wgrad8Args {
  const void* dy[4];
  int64_t ldy[4];
  int cols[4], n;
  const uint8_t *x, *scale;
  int64_t ldx;
  float* part;
  int M, N, K, S, tn, tk, nb;
};
constexpr int W8 = 256, T8 = 32;  // rows and columns of dW a workgroup takes, tokens a step

// 8 e4m3 bytes times the scale as 8 bf16
KD_DEV u32x4 widen8(uint32_t v0, uint32_t v1, float scale) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = i < 2 ? v0 : v1;
    w[i] = __builtin_bit_cast(uint32_t, (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, scale, true)
                                                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, scale, false));
  }
  return w;
}

template <class E>
__global__ __launch_bounds__(256, 1) void k_wgrad8(Wgrad8Args w) {
  using TL = Tile<WT, 4>;                                     // (its rows: 128 columns in 16 bits)
  constexpr int HALF = T8 * TL::ROWB, TILE = 2 * HALF;        // a step's tile of one operand in 16 bits
  constexpr int X8 = T8 * W8, SLOTS = 4, YL = 4, XL = 2;      // X's bytes; slots of the copies; copies a wave and step
  constexpr int CHUNK = 128, SROW = 2 * T8;                   // steps whose scales lie in the LDS; bytes of a step
  __shared__ __attribute__((aligned(1024))) uint8_t s_y[SLOTS * TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t s_x8[SLOTS * X8];
  __shared__ __attribute__((aligned(1024))) uint8_t s_x[2 * TILE];
  __shared__ __attribute__((aligned(16))) uint8_t s_scale[CHUNK * SROW];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hf = lane >> 5,
            c = lane & 31;
  const int item = xcd_remap(blockIdx.x, gridDim.x), tiles = w.tn * w.tk;
  const int piece = item / tiles, tile = item - piece * tiles;
  const int n0 = (tile / w.tk) * W8, k0 = (tile - (tile / w.tk) * w.tk) * W8;
  const int steps_all = int((int64_t(w.M) + T8 - 1) / T8);
  const int e0 = int(int64_t(steps_all) * piece / w.S), e1 = int(int64_t(steps_all) * (piece + 1) / w.S);
  // This wave's copies of dY: half of the rows of one half of the tile's columns, which
  // lie in one part (parts before the last are whole halves)
  const int yh = wave >> 1;
  const uint8_t* dy = static_cast<const uint8_t*>(w.dy[0]);
  int64_t yrb = w.ldy[0];
  int cols = w.cols[0], first = n0 + yh * WT;
#pragma unroll
  for (int i = 1; i < 4; ++i)
    if (i < w.n && first >= cols) first -= cols, dy = static_cast<const uint8_t*>(w.dy[i]), yrb = w.ldy[i], cols = w.cols[i];
  yrb *= 2;
  const bool none = first >= cols;  // (a half behind N)
  uint32_t yoff[YL];
#pragma unroll
  for (int j = 0; j < YL; ++j) {
    const int r = ((wave & 1) * YL + j) * 4 + (lane >> 4), col = first + 8 * ((lane & 15) ^ TL::swz(r));
    yoff[j] = !none && col < cols ? uint32_t(r) * uint32_t(yrb) + uint32_t(col) * 2u : OFF_OUTSIDE;
  }
  // ... and of X's bytes: rows tid / 16 and 16 on, 16 columns each, where this thread reads them
  const int xr = tid >> 4, xc = tid & 15;
  const uint32_t xoff = k0 + 16 * xc < w.K ? uint32_t(xr) * uint32_t(w.ldx) + uint32_t(k0 + 16 * xc) : OFF_OUTSIDE;
  const uint32_t kw = uint32_t((w.K + 15) / 16 * 16);
  // Both operands' next steps to copy (behind the piece's end, and behind M: zeros; products
  // and no selects, which would end the basic block)
  const int end = e1 == steps_all ? w.M : e1 * T8;
  const uint32_t ylast = none ? 0u : uint32_t(cols) * 2u, ystep = none ? 0u : uint32_t(yrb), xstep = uint32_t(w.ldx);
  const uint8_t *ynext = dy + int64_t(e0) * T8 * yrb, *xnext = w.x + int64_t(e0) * T8 * w.ldx;
  int yleft = end - e0 * T8, xleft = yleft;  // tokens
  u32x4 rs_y, rs_x;
  auto next_y = [&] {
    const int rows = max(0, min(T8, yleft));
    rs_y = rsrc_words(ynext, uint32_t(min(rows, 1)) * (uint32_t(rows - 1) * ystep + ylast));
    ynext += T8 * yrb, yleft -= T8;
  };
  auto next_x = [&] {
    const int rows = max(0, min(T8, xleft));
    rs_x = rsrc_words(xnext, uint32_t(min(rows, 1)) * (uint32_t(rows - 1) * xstep + kw));
    xnext += T8 * w.ldx, xleft -= T8;
  };
  auto load_y = [&](int slot, int j) {
    dma_b128(rs_y, yoff[j], lds_addr(s_y) + uint32_t(slot * TILE + (wave * YL + j) * 1024));
  };
  auto load_x = [&](int slot, int j) {
    dma_b128(rs_x, xoff + (xoff < OFF_OUTSIDE ? uint32_t(j * 16) * uint32_t(w.ldx) : 0u),
             lds_addr(s_x8) + uint32_t(slot * X8 + j * 4096 + wave * 1024));
  };
  auto load = [&](int slot) {
    next_x(), next_y();
#pragma unroll
    for (int j = 0; j < XL; ++j) load_x(slot, j);
#pragma unroll
    for (int j = 0; j < YL; ++j) load_y(slot, j);
  };
  // Scales of the steps p0 on, of rows r and r + 16 side by side
  const int kb = k0 / QB;
  auto fetch_scales = [&](int p0) {
#pragma unroll 8
    for (int i = tid; i < min(CHUNK, e1 - p0) * T8; i += 256) {
      const int p = p0 + i / T8, b = (i >> 4) & 1;
      const int64_t row = int64_t(p) * T8 + (i & 15);
      const uint8_t* s = w.scale + row * w.nb + kb + b;
      const bool in = kb + b < w.nb;
      const uint32_t lo = in && row < w.M ? s[0] : 127u, hi = in && row + 16 < w.M ? s[int64_t(16) * w.nb] : 127u;
      reinterpret_cast<uint16_t*>(s_scale)[i] = uint16_t(lo | hi << 8);
    }
  };
  // (a thread's two words of a row in 16 bits; 16 lanes write one row, and those of its
  // second half take their second word first, so that they meet every bank once)
  const int odd = xc >> 3;
  u32x2 xv[XL][2];
  uint32_t xs;
  auto take_x = [&](int slot, int p) {
#pragma unroll
    for (int j = 0; j < XL; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        xv[j][h] = *reinterpret_cast<const u32x2*>(s_x8 + slot * X8 + j * 4096 + tid * 16 + 8 * (odd ^ h));
    xs = reinterpret_cast<const uint16_t*>(s_scale)[p * T8 + odd * 16 + xr];
  };
  const int xto[2] = {odd * HALF + TL::at(xr, 2 * (xc & 7) + odd), odd * HALF + TL::at(xr, 2 * (xc & 7) + (odd ^ 1))};
  auto put_x = [&](int to, int j, int h) {
    if (j == 0 && h == 0) settle(xs);  // (nothing of it is formed earlier, where it would wait for the read)
    const float s = scale_value(j == 0 ? xs & 255u : xs >> 8);
    *reinterpret_cast<u32x4*>(s_x + to * TILE + j * 16 * TL::ROWB + xto[h]) = widen8(xv[j][h][0], xv[j][h][1], s);
  };
  // this wave's 128 x 128: half wn of the dY tile against half wk of the X tile
  const int wn = wave >> 1, wk = wave & 1;
  int at[4][2];  // of a tile's half: [32 columns][4 tokens more]
  {
    const int i = lane & 15, q = lane >> 4;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        at[b][half] = TL::at(8 * (q >> 1) + 4 * half + (i >> 2), 4 * b + 2 * (q & 1) + ((i & 3) >> 1)) + 8 * (i & 1);
  }
  f32x16 acc[4][4];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = f32x16{};
  u32x4 av[2][4], bv[2][4];  // [16 tokens' parity][32 columns]
  auto read = [&](lds_u8* t, int b, int ks) {
    const u32x2 lo = ds_read_tr16(t + at[b][0] + ks * 16 * TL::ROWB), hi = ds_read_tr16(t + at[b][1] + ks * 16 * TL::ROWB);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  // 16 tokens' products in 16 lots of one block, between(m) before each
  auto multiply = [&](int ks, auto between) {
    u32x4 hi, lo;
#pragma unroll
    for (int m = 0; m < 16; ++m) {
      const int a = m >> 2, b = m & 3;
      __builtin_amdgcn_sched_barrier(0);
      between(m);
      if (b == 0) {
        hi = av[ks][a];
        if constexpr (std::is_same_v<E, F16>) {
          float f[8];
          unpack8<F16>(hi, f);
          hi = pack8<BF16>(f);
          lo = pack8_residual<BF16>(f, hi);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (std::is_same_v<E, F16>) acc[a][b] = mfma32x32x16<BF16>(lo, bv[ks][b], acc[a][b]);
      acc[a][b] = mfma32x32x16<BF16>(hi, bv[ks][b], acc[a][b]);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // the m-th of the reads of 16 tokens, in the order of their use
  auto read_next = [&](lds_u8* ty, lds_u8* tx, int to, int from_ks, int m) {
    if (m == 0 || m == 2 || m == 3 || m == 4) bv[to][m == 0 ? 0 : m - 1] = read(tx, m == 0 ? 0 : m - 1, from_ks);
    else if (m < 8) av[to][m == 1 ? 0 : m - 4] = read(ty, m == 1 ? 0 : m - 4, from_ks);
  };
  fetch_scales(e0);
  for (int i = 0; i < SLOTS - 1; ++i) load(i);
  wait_vmem_n<2 * (YL + XL)>();  // the first step's (copies of steps behind the piece fill with zeros, so counts hold)
  barrier_lds();
  take_x(0, 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) put_x(0, j >> 1, j & 1);
  barrier_lds();
  next_x();
  load_x(SLOTS - 1, 0), load_x(SLOTS - 1, 1);
#pragma unroll
  for (int b = 0; b < 4; ++b)
    av[0][b] = read(to_lds(s_y) + wn * HALF, b, 0), bv[0][b] = read(to_lds(s_x) + wk * HALF, b, 0);
  for (int c0 = e0, p0 = e0; c0 < e1; p0 += CHUNK) {  // p0: the first step whose scales are there
    const int c1 = min(e1, p0 + CHUNK - 1);
    for (int e = c0; e < c1; ++e) {  // (one basic block)
      const int i = e - e0;
      lds_u8 *ty = to_lds(s_y) + (i & 3) * TILE + wn * HALF, *tx = to_lds(s_x) + (i & 1) * TILE + wk * HALF;
      wait_vmem_n<2 * YL + 2 * XL>();  // X of e + 1; behind it dY of e + 1, X and dY of e + 2, X of e + 3
      multiply(0, [&](int m) {
        read_next(ty, tx, 1, 1, m);
        if (m == 7) take_x((i + 1) & 3, e + 1 - p0);
        if (m == 8) next_y();
        if (m == 9) next_x();
        if (m >= 10 && m < 14) put_x((i + 1) & 1, (m - 10) >> 1, m & 1);
      });
      wait_vmem_n<YL + 2 * XL>();  // dY of e + 1; behind it X and dY of e + 2, X of e + 3
      barrier_lds();  // the next step's tiles are in place for every wave, and every wave has read this one's
      lds_u8 *ny = to_lds(s_y) + ((i + 1) & 3) * TILE + wn * HALF, *nx = to_lds(s_x) + ((i + 1) & 1) * TILE + wk * HALF;
      multiply(1, [&](int m) {
        read_next(ny, nx, 0, 0, m);
        if (m >= 8 && m < 8 + YL) load_y((i + 3) & 3, m - 8);
        if (m >= 8 + YL && m < 8 + YL + XL) load_x(i & 3, m - 8 - YL);
      });
    }
    c0 = c1;
    if (c0 < e1) {
      fetch_scales(p0 + CHUNK);  // (every wave has taken its last of those that were there before the step's barrier)
      barrier_lds();
    }
  }
  wait_vmem();  // (the copies behind the piece land before the LDS is given back)
  float* out = w.part + int64_t(piece) * w.N * w.K;
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int k = k0 + WT * wk + 32 * b + c, nb = n0 + WT * wn + 32 * a, n = nb + 4 * hf;
      float* p = out + int64_t(n) * w.K + k;
      if (nb + 32 <= w.N) {  // (uniform: one test for the block's rows)
        if (k < w.K) {
#pragma unroll
          for (int r = 0; r < 16; ++r) p[int64_t(8 * (r >> 2) + (r & 3)) * w.K] = acc[a][b][r];
        }
      } else if (k < w.K) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (n + 8 * (r >> 2) + (r & 3) < w.N) p[int64_t(8 * (r >> 2) + (r & 3)) * w.K] = acc[a][b][r];
      }
    }
}

}  // namespace

// Pieces: a step of 64 tokens takes a workgroup 0.45 us with two on a CU, and a
// piece's N K floats go to memory and back at about 5 TB/s; steps / S * 0.45 us +
// S N K 1.6e-6 us is least at the root below.  No more than two workgroups a CU.
int wgrad_pieces(int M, int N, int K) {
  const int tiles = ((N + WT - 1) / WT) * ((K + WT - 1) / WT), steps = (M + 63) / 64;
  const int best = int(std::sqrt(281250.0 * steps / (double(N) * K)) + 0.5);
  return std::max(1, std::min(std::min(best, steps), 512 / tiles));
}

int launch_wgrad(const void* dy, const void* x, void* dw, float* part, int M, int N, int K, int dtype, hipStream_t st) {
  WgradArgs w{dy, x, part, M, N, K, wgrad_pieces(M, N, K), (N + WT - 1) / WT, (K + WT - 1) / WT};
  const int64_t n = int64_t(N) * K;
  auto go = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL(k_wgrad<E>, dim3(unsigned(w.tn * w.tk * w.S)), dim3(256), 0, st, w);
    hipLaunchKernelGGL(k_wgrad_sum<E>, dim3(unsigned((n / 4 + 255) / 256)), dim3(256), 0, st, part,
                       static_cast<uint16_t*>(dw), n, w.S);
  };
  if (dtype == KD_BF16) go(BF16{});
  else go(F16{});
  return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
}

// The same for tiles of 256 x 256, one a CU: rounds of workgroups over the chip times
// a round's cost, and the pieces' way through memory, in us.  Fitted to 1 to 28 pieces
// of six shapes, which it meets within 4 us but where a piece is a few steps: 16384
// tokens by 768 x 768 take 63 us in 8 pieces, 45.7 in 14, 40.8 in 21 and 41.0 in 28.
int wgrad8_pieces(int M, int N, int K) {
  constexpr double START = 7.0, STEP = 0.80, ELEMENT = 1.2e-6;
  const int64_t tiles = int64_t((N + W8 - 1) / W8) * ((K + W8 - 1) / W8), steps = (int64_t(M) + T8 - 1) / T8;
  int best = 1;
  double least = 1e30;
  for (int64_t S = 1; S <= std::min<int64_t>(steps, 256); ++S) {
    const double us = double((tiles * S + 255) / 256) * (START + STEP * double((steps + S - 1) / S)) + ELEMENT * double(S) * N * K;
    if (us < least) least = us, best = int(S);
  }
  return best;
}
int64_t wgrad8_ws_bytes(int M, int N, int K) { return int64_t(4) * wgrad8_pieces(M, N, K) * N * K; }

int launch_wgrad8(const kd_wgrad8_args& a, hipStream_t st) {
  const int S = wgrad8_pieces(a.M, a.N, a.K);
  Wgrad8Args g{};
  for (int i = 0; i < a.n; ++i) g.dy[i] = a.dy[i], g.ldy[i] = a.ldy[i], g.cols[i] = a.cols[i];
  g.n = a.n, g.x = a.x, g.scale = a.x_scale, g.ldx = a.ldx, g.part = a.ws;
  g.M = a.M, g.N = a.N, g.K = a.K, g.S = S;
  g.tn = (a.N + W8 - 1) / W8, g.tk = (a.K + W8 - 1) / W8, g.nb = (a.K + QB - 1) / QB;
  const int64_t n = int64_t(a.N) * a.K;
  auto go = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL(k_wgrad8<E>, dim3(unsigned(g.tn * g.tk * S)), dim3(256), 0, st, g);
    hipLaunchKernelGGL(k_wgrad_sum<E>, dim3(unsigned((n / 4 + 255) / 256)), dim3(256), 0, st, a.ws,
                       static_cast<uint16_t*>(a.dw), n, S);
  };
  if (a.dtype == KD_BF16) go(BF16{});
  else go(F16{});
  return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
}

}  // namespace kd
