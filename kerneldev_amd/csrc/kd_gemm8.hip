// C [M, N] = A B^T of 8-bit blocks (kd_block8.h): A [M, K] rows with a scale for
// each 128 columns, B [N, K] with a scale for each 128 x 128, fp32 sums, one
// rounding to the output's type.
//
// Two products.  The 8-bit MFMA adds eight neighbouring products aligned to the
// largest of them, what lies under 2^-13 of its power of two cut off, and the
// groups' sums in fp32 (found by sending pairs of values through it); on normal
// data that leaves 1.4e-5 of a result, against the 1.7e-3 of its rounding to bf16 and 2.1e-4 to fp16,
// so 16-bit results take it.  A result in fp32 takes the same tiles through the
// bf16 MFMA (e4m3 is exact in bf16, the products in fp32), each block's sum
// multiplied by its scales afterwards: half the rate, and fp32's precision.
#include "kd_block8.h"

namespace kd {
namespace {

struct F32Q {};  // fp32 results of the 8-bit product (kd_matmul8_args.fast)

// Eight of an operand's 32 e4m3 values (words 2 q and 2 q + 1) as bf16
KD_DEV u32x4 as_bf16(const i32x8& v, int q) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t from = uint32_t(v[2 * q + (i >> 1)]);
    w[i] = __builtin_bit_cast(uint32_t, (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(from, 1.f, true)
                                                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(from, 1.f, false));
  }
  return w;
}

KD_DEV i32x8 join8(const u32x4& lo, const u32x4& hi) {
  return i32x8{int(lo[0]), int(lo[1]), int(lo[2]), int(lo[3]), int(hi[0]), int(hi[1]), int(hi[2]), int(hi[3])};
}

// The workgroup's tile.  Each XCD takes one contiguous range of the items
// (xcd_remap), which run down `group` rows of tiles before the next column of
// tiles, so that the tiles in flight on an XCD share rows of both operands in its L2.
KD_DEV void tile_of(int item, int tiles_m, int tiles_n, int group, int* tm, int* tn) {
  const int per = group * tiles_n, g = item / per, first = g * group;
  const int rows = min(group, tiles_m - first), local = item - g * per;
  *tn = local / rows;
  *tm = first + (local - *tn * rows);
}

// A workgroup of WM x WN waves takes BM x BN of C, 128 columns of K a step (whole
// cache lines, one block's scales) through two tiles of both operands in LDS.  A
// wave takes BM / WM x BN / WN with the 32 x 32 x 64 MFMA; B's rows are the
// instruction's rows, so that a lane ends with four consecutive columns of a row
// of C.  A step is 2 FA parts, 32 rows of A and half of K each, whose operands are
// read while the products of the part before run; before the last part, when every
// wave has read all of the step's, the next step's tiles must have landed and the
// copies of the step behind it start: about a step's products to arrive in, and one
// barrier a step.  Reads and copies stand between single products (all ahead of a
// part's products: 5 % slower).  C leaves through LDS in whole rows.
//
// What bounds it: in 8192^3, 450 us or 2.4 PFLOP/s, the products are issued half of the
// time; the waves' reads keep the LDS three quarters busy and the copies' writes the
// rest.  Four waves of 128 x 128, which read two thirds of that, have nobody to take
// over while they wait: 487 us.  Workgroups that go on to a next tile, with its copies
// on their way while C is stored from registers: 489, and 50 against 47 in 16384 x
// 2304 x 768.
template <class O, int BM, int BN, int WM, int WN, int PER_CU>
struct Gemm8 {
  static constexpr bool F = std::is_same_v<O, F32>, WIDE = F || std::is_same_v<O, F32Q>;
  static constexpr int NW = WM * WN, THREADS = 64 * NW, TM = BM / WM, TN = BN / WN, FA = TM / 32, FB = TN / 32;
  using TL = Tile<64>;  // 64 rows of 128 bytes, 8 KiB
  static constexpr int SLOT = (BM + BN) * 128, LOADS = SLOT / 1024 / NW;  // wave-wide 1 KiB copies a wave and step
  static constexpr int SB = 16, SROW = SB + 4;                            // blocks of K with scales in LDS
  static constexpr int ESIZE = WIDE ? 4 : 2, OROW = BN * ESIZE + 16;         // C in LDS
  static constexpr int NBT = (BN + QB - 1) / QB;                          // B's blocks of rows in a tile
  static constexpr int POOL = 2 * SLOT > BM * OROW ? 2 * SLOT : BM * OROW;
  static constexpr int SCALES = (BM + NBT) * SROW, LDS = POOL + 2 * SCALES;
  static_assert(SLOT % (1024 * NW) == 0 && (BM / 8) % LOADS == 0 && LOADS % 2 == 0 && LDS * PER_CU <= 160 * 1024 && TN <= QB &&
                    THREADS % BM == 0 && SB * BM % (4 * THREADS) == 0 && NBT * SB <= THREADS,
                "tile shape");
};

template <class O, int BM, int BN, int WM, int WN, int PER_CU>
__global__ __launch_bounds__(64 * WM * WN, (PER_CU * WM * WN + 3) / 4) void k_gemm8(kd_matmul8_args g, int tiles_m,
                                                                                    int tiles_n, int group) {
  using G = Gemm8<O, BM, BN, WM, WN, PER_CU>;
  using TL = typename G::TL;
  constexpr bool F = G::F;
  constexpr int FA = G::FA, FB = G::FB, LOADS = G::LOADS;
  __shared__ __attribute__((aligned(1024))) uint8_t s_pool[G::LDS];
  uint8_t* s_scale = s_pool + G::POOL;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hf = lane >> 5, c = lane & 31;
  int tm, tn;
  tile_of(xcd_remap(blockIdx.x, gridDim.x), tiles_m, tiles_n, group, &tm, &tn);
  const int m0 = tm * BM, n0 = tn * BN, nb = (g.K + QB - 1) / QB;
  const int rows_a = min(BM, g.M - m0), rows_b = min(BN, g.N - n0);
  // This wave's copies: 1 KiB pieces of 8 rows, of A or of B.  A lane's 16 bytes lie
  // at its own row of a piece, and at a chunk whose swizzle the piece's parity flips.
  const bool is_a = wave * LOADS < BM / 8;
  const int piece0 = is_a ? wave * LOADS : wave * LOADS - BM / 8;
  const uint32_t ld = uint32_t(is_a ? g.lda : g.ldb);
  const u32x4 rs = is_a ? rsrc_words(g.a + int64_t(m0) * g.lda, uint32_t(int64_t(rows_a - 1) * g.lda + g.K))
                        : rsrc_words(g.b + int64_t(n0) * g.ldb, uint32_t(int64_t(rows_b - 1) * g.ldb + g.K));
  const uint32_t arow = uint32_t(piece0 * 8 + lane / TL::CPR) * ld,
                 c16 = uint32_t((lane % TL::CPR) ^ TL::swz(lane / TL::CPR)) * 16u;
  auto load = [&](int e, int from, int to) {  // copies from .. to - 1 of step e (of a step behind the last: zeros)
    const uint32_t k0 = uint32_t(e) * QB;
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_addr(s_pool) + uint32_t(e & 1) * G::SLOT + uint32_t(wave * LOADS) * 1024u);
#pragma unroll
    for (int j = from; j < to; ++j) {
      const uint32_t col = k0 + (c16 ^ ((j & 1) * uint32_t(TL::swz(8)) * 16u));
      dma_b128(rs, col < uint32_t(g.K) ? arow + uint32_t(j * 8) * ld + col : OFF_OUTSIDE, at + uint32_t(j) * 1024u);
    }
  };
  // Scales, SB blocks of K at a time, in two buffers: a thread takes SPT bytes of a
  // row of A, the first ones a byte of B's too.  Fetched a chunk ahead.
  constexpr int TPR = G::THREADS / BM, SPT = G::SB / TPR;
  const int srow = tid / TPR, sb0 = (tid - srow * TPR) * SPT;
  uint32_t sv[SPT], sw = 0;
  auto fetch_scales = [&](int b0) {
    const uint8_t* p = g.a_scale + int64_t(m0 + min(srow, rows_a - 1)) * nb + b0 + sb0;
#pragma unroll
    for (int i = 0; i < SPT; ++i) sv[i] = b0 + sb0 + i < nb ? p[i] : 0u;
    const int r = tid / G::SB, b = b0 + tid % G::SB;
    if (r < G::NBT && r * QB < rows_b && b < nb) sw = g.b_scale[int64_t(n0 / QB + r) * nb + b];
  };
  auto put_scales = [&](int chunk) {
    uint8_t* to = s_scale + (chunk & 1) * G::SCALES;
#pragma unroll
    for (int i = 0; i < SPT; i += 4)
      *reinterpret_cast<uint32_t*>(to + srow * G::SROW + sb0 + i) = sv[i] | sv[i + 1] << 8 | sv[i + 2] << 16 | sv[i + 3] << 24;
    if (tid < G::NBT * G::SB) to[(BM + tid / G::SB) * G::SROW + tid % G::SB] = uint8_t(sw);
  };
  fetch_scales(0);
  load(0, 0, LOADS);
  put_scales(0);
  const int wn = wave / WM, wm = wave - wn * WM;
  f32x16 acc[FB][FA];  // [32 rows of B][32 rows of A]
#pragma unroll
  for (int i = 0; i < FB; ++i)
#pragma unroll
    for (int j = 0; j < FA; ++j) acc[i][j] = f32x16{};
  const int at0 = TL::at(c, 2 * hf), at1 = TL::at(c, 2 * hf + 1);  // this lane's chunks of the first half (of the second: bit 6 flipped); 32 rows on: 4 KiB
  const int scale_a = (wm * G::TM + c) * G::SROW, scale_b = (BM + wn * G::TN / QB) * G::SROW;
  auto frag = [&](int e, int h, int row) {
    lds_u8* t = to_lds(s_pool) + (e & 1) * G::SLOT + row * 128;
    return join8(ds_read16(t + (at0 ^ (64 * h))), ds_read16(t + (at1 ^ (64 * h))));
  };
  uint32_t xs[FA], ws = 0;  // scale bytes, the current block's lowest
  auto multiply = [&](const i32x8& a, const i32x8& b, int i, int j) {
    if constexpr (F) {
      f32x16 part{};  // without the scales
#pragma unroll
      for (int q = 0; q < 4; ++q) part = mfma32x32x16<BF16>(as_bf16(b, q), as_bf16(a, q), part);
      const int e2 = int(ws & 255u) + int(xs[j] & 255u) - 254;
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] += __builtin_amdgcn_ldexpf(part[q], e2);
    } else {
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc[i][j], 0, 0, 0, int(ws), 0, int(xs[j]));
    }
  };
  i32x8 fa[2], fb[2][FB];  // A's 32 rows of this part and the next; B's of this half and the next
  auto read_b = [&](int e, int h, int i) { fb[h][i] = frag(e, h, BM + wn * G::TN + 32 * i); };
  wait_vmem();
  barrier_lds();  // the first step's tiles and scales are in place for every wave
  load(1, 0, LOADS);  // (copies of steps behind the last write zeros)
#pragma unroll
  for (int i = 0; i < FB; ++i) read_b(0, 0, i);
  fa[0] = frag(0, 0, wm * G::TM);
  for (int e0 = 0; e0 < nb; e0 += G::SB) {
    const int chunk = e0 / G::SB, e1 = min(nb, e0 + G::SB);
    if (e0 > 0) {
      put_scales(chunk);
      barrier_lds();
    }
    if (e1 < nb) fetch_scales(e1);
    const uint8_t* from = s_scale + (chunk & 1) * G::SCALES;
    auto scales = [&](int b) {
#pragma unroll
      for (int j = 0; j < FA; ++j) xs[j] = from[scale_a + j * 32 * G::SROW + b];
      ws = from[scale_b + b];
    };
    scales(0);
    // One basic block: products would otherwise sink past the barrier, behind the reads they are to cover
    for (int e = e0; e < e1; ++e) {
#pragma unroll
      for (int t = 0; t < 2 * FA; ++t)  // part t: half t / FA, A's rows 32 (t % FA) on
#pragma unroll
        for (int i = 0; i < FB; ++i) {
          if (t == 2 * FA - 1) {
            if (i == 0) {
              wait_vmem();
              barrier_lds();  // step e + 1's tiles have landed for every wave, and every wave has read step e's
              fa[0] = frag(e + 1, 0, wm * G::TM);
            }
            read_b(e + 1, 0, i);
            load(e + 2, i * LOADS / FB, (i + 1) * LOADS / FB);
          } else {
            if (i == 0) fa[(t + 1) & 1] = frag(e, (t + 1) / FA, wm * G::TM + 32 * ((t + 1) % FA));
            if (t == FA - 1 - (FA > 1)) read_b(e, 1, i);
          }
          __builtin_amdgcn_sched_barrier(0);
          multiply(fa[t & 1], fb[t / FA][i], i, t % FA);
          __builtin_amdgcn_sched_barrier(0);
        }
      scales(e - e0 + 1);  // (a chunk's first are read anew)
    }
  }
  wait_vmem();
  barrier_lds();
  // C through LDS: [BM] rows of OROW bytes
#pragma unroll
  for (int i = 0; i < FB; ++i)
#pragma unroll
    for (int j = 0; j < FA; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // registers 4 q ..: columns 8 q + 4 hf .. of the 32
        const f32x16& v = acc[i][j];
        uint8_t* p = s_pool + (wm * G::TM + 32 * j + c) * G::OROW + (wn * G::TN + 32 * i + 8 * q + 4 * hf) * G::ESIZE;
        if constexpr (G::WIDE) *reinterpret_cast<f32x4*>(p) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        else *reinterpret_cast<u32x2*>(p) = u32x2{pack2<O>(v[4 * q], v[4 * q + 1]), pack2<O>(v[4 * q + 2], v[4 * q + 3])};
      }
  barrier_lds();
  constexpr int PER = 16 / G::ESIZE, CH = BN / PER;  // values and words of a row
  uint8_t* out = static_cast<uint8_t*>(g.out) + (int64_t(m0) * g.ldo + n0) * G::ESIZE;
  if ((g.ldo * G::ESIZE) % 16 == 0) {
    for (int i = tid; i < rows_a * CH; i += G::THREADS) {
      const int r = i / CH, w = i - r * CH, left = rows_b - w * PER;
      const uint8_t* p = s_pool + r * G::OROW + w * 16;
      uint8_t* q = out + (int64_t(r) * g.ldo + w * PER) * G::ESIZE;
      if (left >= PER) {
        // (C of large tiles passes by the L2, which the operands' rows need: 16384 x 2304 x 768 47 and 43 us, x 4096 76 and 71;
        // with 64 x 64 300 x 1000 x 528 4.1 and 4.5)
        if constexpr (BM > 64) __builtin_nontemporal_store(*reinterpret_cast<const u32x4*>(p), reinterpret_cast<u32x4*>(q));
        else *reinterpret_cast<u32x4*>(q) = *reinterpret_cast<const u32x4*>(p);
      } else {
        for (int k = 0; k < left; ++k) {
          if constexpr (G::WIDE) reinterpret_cast<float*>(q)[k] = reinterpret_cast<const float*>(p)[k];
          else reinterpret_cast<uint16_t*>(q)[k] = reinterpret_cast<const uint16_t*>(p)[k];
        }
      }
    }
  } else {  // rows that do not start on 16 bytes: value by value
    for (int i = tid; i < rows_a * BN; i += G::THREADS) {
      const int r = i / BN, n = i - r * BN;
      if (n >= rows_b) continue;
      const uint8_t* p = s_pool + r * G::OROW + n * G::ESIZE;
      uint8_t* q = out + (int64_t(r) * g.ldo + n) * G::ESIZE;
      if constexpr (G::WIDE) *reinterpret_cast<float*>(q) = *reinterpret_cast<const float*>(p);
      else *reinterpret_cast<uint16_t*>(q) = *reinterpret_cast<const uint16_t*>(p);
    }
  }
}

// Few rows of A: a workgroup of W waves takes 16 rows of B, each wave every W-th
// block of K straight from memory into the 16 x 16 x 128 MFMA (a lane holds 32
// bytes of a row, four lanes a block's 128), against MT x 16 rows of A; the waves'
// sums meet in LDS, in order.  What bounds it is reading B once, and latency.
template <class O, int MT, int W>
__global__ __launch_bounds__(64 * W) void k_gemm8_rows(kd_matmul8_args g) {
  constexpr bool F = std::is_same_v<O, F32>;
  __shared__ f32x4 s_part[W][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, nb = (g.K + QB - 1) / QB;
  const uint8_t* b = g.b + int64_t(min(n0 + r, g.N - 1)) * g.ldb + 32 * q;
  const uint8_t* bs = g.b_scale + int64_t(n0 / QB) * nb;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{};
  auto read = [&](const uint8_t* p, int k) {  // 32 bytes at column k + 32 q, zeros behind K
    u32x4 lo{}, hi{};
    if (k + 32 * q < g.K) lo = *reinterpret_cast<const u32x4*>(p + k);
    if (k + 32 * q + 16 < g.K) hi = *reinterpret_cast<const u32x4*>(p + k + 16);
    return join8(lo, hi);
  };
#pragma unroll 4
  for (int kb = wave; kb < nb; kb += W) {
    const i32x8 bv = read(b, kb * QB);
    const int wsc = bs[kb];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int64_t row = min(16 * t + r, g.M - 1);
      const i32x8 av = read(g.a + row * g.lda + 32 * q, kb * QB);
      const int xsc = g.a_scale[row * nb + kb];
      if constexpr (F) {
        // the 16 x 16 x 32 bf16 product takes 8 values a lane: any four lanes of a row hold the same places of both operands
        f32x4 part{};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, as_bf16(bv, i)),
                                                         __builtin_bit_cast(bf16x8, as_bf16(av, i)), part, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] += __builtin_amdgcn_ldexpf(part[i], wsc + xsc - 254);
      } else {
        acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bv, av, acc[t], 0, 0, 0, wsc, 0, xsc);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) s_part[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < MT; t += W) {
    f32x4 v = s_part[0][t][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += s_part[w][t][lane];
    const int m = 16 * t + r, n = n0 + 4 * q;  // lane (r, q): row r of A's tile, columns 4 q ..
    if (m >= g.M) continue;
    const int64_t at = int64_t(m) * g.ldo + n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < g.N) {
        if constexpr (F || std::is_same_v<O, F32Q>) static_cast<float*>(g.out)[at + i] = v[i];
        else static_cast<uint16_t*>(g.out)[at + i] = uint16_t(pack2<O>(v[i], 0.f) & 0xFFFFu);
      }
  }
}

template <class O, int BM, int BN, int WM, int WN, int PER_CU>
int go_tiles(const kd_matmul8_args& g, int group, hipStream_t st) {
  using G = Gemm8<O, BM, BN, WM, WN, PER_CU>;
  const auto k = k_gemm8<O, BM, BN, WM, WN, PER_CU>;
  const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN;
  hipLaunchKernelGGL(k, dim3(unsigned(tm * tn)), dim3(G::THREADS), 0, st, g, tm, tn, group);
  return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
}

template <class O, int MT>
int go_rows(const kd_matmul8_args& g, hipStream_t st) {
  hipLaunchKernelGGL((k_gemm8_rows<O, MT, 8>), dim3(unsigned((g.N + 15) / 16)), dim3(512), 0, st, g);
  return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
}

// Which tile: rounds of workgroups over the chip times a round's cost, in us, from
// 8192^3 (a step of 128 columns) and 16384 x 4096 x 768 (start and end of a tile):
//   256 x 256, one a CU:   450 us and 79 us
//   128 x 128, two:        564        88
//   64 x 64, four:         864       118, but 4.1 us against 5.7 and 12.5 where one round does (128 x 2048 x 768)
// (columns of 64 instead of 128 a step: 16 TB/s instead of 25 from the L2, 528 us at best in the first;
// four waves instead of eight in the 128 x 128 tile: 595 and 94.)
template <class O>
int go(const kd_matmul8_args& g, hipStream_t st) {
  // Few rows, us, rows / tiles: 32 x 2048 x 768 3.2 / 4.3, 32 x 768 x 2048 5.1 / 6.5, 48 x 768 x 2048 6.9 / 6.5, 64 x 8192 x 8192
  // 53 / 46; fp32, whose tiles are slower, 64 x 768 x 2048 7.8 / 13.5
  // (a launch is less than 2^32 threads: up to 2^27 rows of B, or 2^23 tiles of 512 threads)
  const bool rows = g.N < (1 << 27);
  if (rows && g.M <= 16) return go_rows<O, 1>(g, st);
  if (rows && g.M <= 32) return go_rows<O, 2>(g, st);
  if (std::is_same_v<O, F32> && rows && g.M <= 64) return go_rows<O, 4>(g, st);
  const int64_t nb = (g.K + QB - 1) / QB;
  auto cost = [&](int64_t tile, int64_t at_once, double ends, double step) {
    const int64_t tiles = (g.M + tile - 1) / tile * ((g.N + tile - 1) / tile);
    return tiles >= (1 << 23) ? 1e300 : double((tiles + at_once - 1) / at_once) * (ends + step * double(nb));
  };
  const double large = cost(256, 256, 9.0, 1.70), mid = cost(128, 512, 4.3, 1.10), small = cost(64, 1024, 2.3, 0.84);
  if constexpr (std::is_same_v<O, BF16> || std::is_same_v<O, F16>)  // (an fp32 tile of 256 x 256 does not fit the LDS on its way out)
    if (large < mid && large < small) return go_tiles<O, 256, 256, 2, 4, 1>(g, 4, st);
  if (mid < small) {
    if constexpr (std::is_same_v<O, F32>) return go_tiles<O, 128, 128, 2, 2, 2>(g, 8, st);  // (its registers do not fit eight waves)
    else return go_tiles<O, 128, 128, 4, 2, 2>(g, 8, st);
  }
  return go_tiles<O, 64, 64, 2, 2, 4>(g, 8, st);
}

}  // namespace

int launch_matmul8(const kd_matmul8_args& g, hipStream_t st) {
  if (g.dtype == KD_F32) return g.fast ? go<F32Q>(g, st) : go<F32>(g, st);
  return g.dtype == KD_BF16 ? go<BF16>(g, st) : go<F16>(g, st);
}

}  // namespace kd
