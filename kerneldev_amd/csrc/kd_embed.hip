// Embedding lookup with a scale, y_i = c W[t_i], and its gradient by sorted
// tokens, dW[v] = c sum over the i with t_i = v of dy_i.
//
// The lookup is one pass over the rows.  The gradient sorts (token, position) by
// the token, stable, so that equal tokens become a run whose rows are added in
// fp32 in the order of their positions: no atomics, and a result that does not
// change from run to run.  A row of dy is read once.  The sorted list is cut into
// chunks of 16 positions, one wave a chunk and 256 columns, eight rows in flight at
// once, so that a token that fills the batch costs what short runs cost; runs that cross a chunk's edge
// leave partial sums, which a last launch adds in order.  32656 tokens of 50021, rows
// of 1024 bf16: lookup 24 us (5.6 TB/s), two sorting passes 36 with dW's clearing, sums
// 24, joins 13, where latency and the launches' starts count more than bytes.  A token outside the
// vocabulary reads nothing: its row of y is NaN and it takes no part in dW.
#include <algorithm>
#include <initializer_list>

#include "kd_block8.h"

namespace kd {
namespace {

constexpr int CHUNK = 16;       // sorted positions a wave adds
constexpr int SORT_T = 1024;    // threads of a sorting workgroup
constexpr int SORT_N = 1024;    // positions it takes: one a thread
constexpr int MAX_BINS = 2048;  // a pass sorts by up to 11 bits
constexpr int JOIN_W = 8;       // waves that share a long run's partial sums

KD_DEV int64_t token_at(const kd_embed_args& a, int64_t i) {
  return a.tokens_dtype == KD_I64 ? static_cast<const int64_t*>(a.tokens)[i] : static_cast<const int32_t*>(a.tokens)[i];
}
// A position's key: its token, or vocab (sorted behind all) where it takes no part
KD_DEV uint32_t key_at(const kd_embed_args& a, int64_t i) {
  const int64_t t = token_at(a, i);
  return t < 0 || t >= a.vocab || t == a.padding_idx ? uint32_t(a.vocab) : uint32_t(t);
}

// ---- values of E, V of them at a time -------------------------------------
template <class E, int V>
KD_DEV void load_v(const void* p, int64_t at, float (&f)[V]) {
  if constexpr (std::is_same_v<E, F32>) {
    const float* q = static_cast<const float*>(p) + at;
    if constexpr (V == 4) {
      const f32x4 u = *reinterpret_cast<const f32x4*>(q);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = u[i];
    } else {
      f[0] = q[0];
    }
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
    if constexpr (V == 8) {
      unpack8<E>(*reinterpret_cast<const u32x4*>(q), f);
    } else if constexpr (V == 4) {
      const u32x2 u = *reinterpret_cast<const u32x2*>(q);
#pragma unroll
      for (int i = 0; i < 2; ++i) f[2 * i] = to_f32<E>(uint16_t(u[i] & 0xFFFFu)), f[2 * i + 1] = to_f32<E>(uint16_t(u[i] >> 16));
    } else {
      f[0] = to_f32<E>(q[0]);
    }
  }
}
// f times the scale, rounded to fp32 before the rounding to E: fp16's conversion
// would otherwise take the multiplication into itself in some of the kernels
template <int V>
KD_DEV void scaled(float (&f)[V], float scale) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    f[k] *= scale;
    settle(f[k]);
  }
}
template <class E, int V>
KD_DEV void store_v(void* p, int64_t at, const float (&f)[V]) {
  if constexpr (std::is_same_v<E, F32>) {
    float* q = static_cast<float*>(p) + at;
    if constexpr (V == 4) *reinterpret_cast<f32x4*>(q) = f32x4{f[0], f[1], f[2], f[3]};
    else q[0] = f[0];
  } else {
    uint16_t* q = static_cast<uint16_t*>(p) + at;
    if constexpr (V == 8) *reinterpret_cast<u32x4*>(q) = pack8<E>(f);
    else if constexpr (V == 4) *reinterpret_cast<u32x2*>(q) = u32x2{pack2<E>(f[0], f[1]), pack2<E>(f[2], f[3])};
    else q[0] = uint16_t(pack2<E>(f[0], 0.f) & 0xFFFFu);
  }
}

// ---- lookup -----------------------------------------------------------------
template <class E, int V>
__global__ __launch_bounds__(256) void k_embed(kd_embed_args a, int64_t row0, uint32_t words_all, uint32_t words) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= words_all) return;
  const uint32_t r = i / words;
  const int64_t row = row0 + r, col = int64_t(i - r * words) * V, t = token_at(a, row);
  float f[V];
#pragma unroll
  for (int k = 0; k < V; ++k) f[k] = __uint_as_float(0x7FC00000u);
  if (t >= 0 && t < a.vocab) load_v<E, V>(a.weight, t * a.dim + col, f);
  scaled<V>(f, a.scale);
  store_v<E, V>(a.out, row * a.dim + col, f);
}

// ---- sort -------------------------------------------------------------------
struct SortPass {
  const uint32_t *keys, *idx;   // NULL: the tokens themselves, in order
  uint32_t *keys_out, *idx_out;
  uint32_t* hist;               // [blocks][bins]: counts; from k_sort_scan on, first positions
  int shift, bits, blocks;      // the digit; workgroups of SORT_N positions
  bool scanned;
};

KD_DEV uint32_t sort_key(const kd_embed_args& a, const SortPass& s, int64_t i) {
  return s.keys != nullptr ? s.keys[i] : key_at(a, i);
}

// Workgroups below s.blocks count their positions' digits; those behind clear dW
// (rows of tokens that do not occur)
__global__ __launch_bounds__(SORT_T) void k_sort_count(kd_embed_args a, SortPass s, int64_t fill_bytes, int count_blocks) {
  __shared__ uint32_t s_hist[MAX_BINS];
  const int bins = 1 << s.bits;
  if (int(blockIdx.x) >= count_blocks) {
    const int64_t step = int64_t(gridDim.x - count_blocks) * SORT_T;
    const int64_t i = int64_t(blockIdx.x - count_blocks) * SORT_T + threadIdx.x;
    const int64_t whole = fill_bytes / 16;
    for (int64_t w = i; w < whole; w += step) static_cast<u32x4*>(a.dw)[w] = u32x4{};
    for (int64_t w = whole * 8 + i; w < fill_bytes / 2; w += step) static_cast<uint16_t*>(a.dw)[w] = 0;
    return;
  }
  for (int b = threadIdx.x; b < bins; b += SORT_T) s_hist[b] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < SORT_N / SORT_T; ++k) {
    const int64_t i = int64_t(blockIdx.x) * SORT_N + k * SORT_T + threadIdx.x;
    if (i < a.n) atomicAdd(&s_hist[(sort_key(a, s, i) >> s.shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += SORT_T) s.hist[int64_t(blockIdx.x) * bins + b] = s_hist[b];
}

// hist's counts to first positions, one workgroup: where many blocks would each
// add up all the others' counts
__global__ __launch_bounds__(SORT_T) void k_sort_scan(SortPass s) {
  __shared__ int s_warp[16];
  const int bins = 1 << s.bits, b0 = 2 * threadIdx.x;
  uint32_t sum[2] = {};
  for (int k = 0; k < s.blocks; ++k)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (b0 + j < bins) sum[j] += s.hist[int64_t(k) * bins + b0 + j];
  uint32_t at[2];
  at[0] = uint32_t(block_scan(int(sum[0] + sum[1]), s_warp)) - sum[0] - sum[1];
  at[1] = at[0] + sum[0];
  for (int k = 0; k < s.blocks; ++k)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (b0 + j < bins) {
        uint32_t* p = s.hist + int64_t(k) * bins + b0 + j;
        const uint32_t n = *p;
        *p = at[j], at[j] += n;
      }
}

// Moves a block's positions behind those of smaller digits, of earlier blocks and
// of earlier places: a wave takes 256 consecutive positions, 64 at a time, and
// ranks equal digits among them with ballots and a count of its own a digit.
__global__ __launch_bounds__(SORT_T) void k_sort_move(kd_embed_args a, SortPass s) {
  constexpr int W = SORT_T / 64, ROUNDS = SORT_N / SORT_T;
  __shared__ uint16_t s_wave[W][MAX_BINS];
  __shared__ uint32_t s_base[MAX_BINS];
  __shared__ int s_warp[16];
  const int bins = 1 << s.bits, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, blk = blockIdx.x;
  for (int b = tid; b < bins; b += SORT_T)
#pragma unroll
    for (int w = 0; w < W; ++w) s_wave[w][b] = 0;
  __syncthreads();
  uint32_t key[ROUNDS], pos[ROUNDS];
  uint16_t rank[ROUNDS];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int64_t i = int64_t(blk) * SORT_N + wave * (64 * ROUNDS) + k * 64 + lane;
    const bool in = i < a.n;
    key[k] = in ? sort_key(a, s, i) : 0u;
    pos[k] = in ? (s.idx != nullptr ? s.idx[i] : uint32_t(i)) : 0u;
  }
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int64_t i = int64_t(blk) * SORT_N + wave * (64 * ROUNDS) + k * 64 + lane;
    const uint32_t d = (key[k] >> s.shift) & uint32_t(bins - 1);
    uint64_t same = __builtin_amdgcn_ballot_w64(i < a.n);
    for (int b = 0; b < s.bits; ++b) {
      const uint64_t one = __builtin_amdgcn_ballot_w64((d >> b) & 1u);
      same &= (d >> b) & 1u ? one : ~one;
    }
    const int before = __builtin_popcountll(same & ((uint64_t(1) << lane) - 1u));
    if (i < a.n) {
      const uint16_t had = s_wave[wave][d];
      rank[k] = uint16_t(had + before);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // every lane has read before the first one writes
      if (before == 0) s_wave[wave][d] = uint16_t(had + __builtin_popcountll(same));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  // thread t: digits 2 t and 2 t + 1.  Counts of the waves to first ranks, then
  // the digits' first positions
  uint32_t total[2] = {}, before[2] = {};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int b = 2 * tid + j;
    if (b >= bins) continue;
    uint32_t run = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t n = s_wave[w][b];
      s_wave[w][b] = uint16_t(run);
      run += n;
    }
    total[j] = run;
    if (s.scanned) {
      before[j] = s.hist[int64_t(blk) * bins + b];
    } else if (s.blocks > 1) {
      total[j] = 0;
#pragma unroll 8
      for (int k = 0; k < s.blocks; ++k) {
        const uint32_t n = s.hist[int64_t(k) * bins + b];
        total[j] += n;
        before[j] += k < blk ? n : 0u;
      }
    }
  }
  if (!s.scanned) {  // (uniform)
    const uint32_t at = uint32_t(block_scan(int(total[0] + total[1]), s_warp)) - total[0] - total[1];
    before[0] += at, before[1] += at + total[0];
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (2 * tid + j < bins) s_base[2 * tid + j] = before[j];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int64_t i = int64_t(blk) * SORT_N + wave * (64 * ROUNDS) + k * 64 + lane;
    if (i >= a.n) continue;
    const uint32_t d = (key[k] >> s.shift) & uint32_t(bins - 1);
    const uint32_t to = s_base[d] + s_wave[wave][d] + rank[k];
    s.keys_out[to] = key[k], s.idx_out[to] = pos[k];
  }
}

// ---- sums of runs -----------------------------------------------------------
struct Runs {
  const uint32_t *keys, *idx;
  float* part;  // [chunk][2][dim]: the run that comes in from the chunk before; the one that starts here and goes on
  int64_t chunks;
  int tiles;
  int64_t first;  // unit (a chunk's tile of columns) of this launch
};

template <class E, int V>
__global__ __launch_bounds__(256) void k_embed_runs(kd_embed_args a, Runs s) {
  const int64_t unit = s.first + int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (unit >= s.chunks * s.tiles) return;
  const int64_t chunk = unit / s.tiles;
  const int lane = threadIdx.x & 63, col = int(unit - chunk * s.tiles) * 64 * V + lane * V;
  const int64_t i0 = chunk * CHUNK;
  const int n = int(min(int64_t(CHUNK), a.n - i0));
  const bool in = col < a.dim;
  // lane 0: the key before the chunk; lane 1 + r: position r; lane 1 + n: the key behind
  const int64_t at = i0 + lane - 1;
  const uint32_t none = 0xFFFFFFFFu;
  const uint32_t key = at >= 0 && at < a.n && lane <= n + 1 ? s.keys[at] : none;
  const uint32_t pos = lane >= 1 && lane <= n ? s.idx[at] : 0u;
  auto key_of = [&](int r) { return uint32_t(__builtin_amdgcn_readlane(int(key), r + 1)); };
  const uint32_t prev = key_of(-1), next = key_of(n);
  float sum[V];
  uint32_t run = key_of(0);
  auto zero = [&] {
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] = 0.f;
  };
  auto flush = [&](bool last) {  // (uniform) the run ends here, or with the chunk
    if (run == uint32_t(a.vocab) || !in) return;
    const bool from = run == prev, on = last && run == next;
    if (from || on) {
      float* p = s.part + (2 * chunk + (from ? 0 : 1)) * a.dim + col;
#pragma unroll
      for (int k = 0; k < V; ++k) p[k] = sum[k];
      return;
    }
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = sum[k];
    scaled<V>(f, a.scale);
    store_v<E, V>(a.dw, int64_t(run) * a.dim + col, f);
  };
  zero();
#pragma unroll
  for (int r0 = 0; r0 < CHUNK; r0 += 8) {
    if (r0 >= n) break;
    float v[8][V];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[j][k] = 0.f;
      const int64_t row = int64_t(uint32_t(__builtin_amdgcn_readlane(int(pos), min(r0 + j, n - 1) + 1)));
      if (r0 + j < n && in) load_v<E, V>(a.dy, row * a.dim + col, v[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (r0 + j < n) {
        const uint32_t k0 = key_of(r0 + j);
        if (k0 != run) {
          flush(false);
          run = k0;
          zero();
        }
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] += v[j][k];
      }
    }
  }
  flush(true);
}

// A run that starts in a chunk and goes on: its partial sums in order, the
// chunks behind the first split over JOIN_W waves
template <class E, int V>
__global__ __launch_bounds__(64 * JOIN_W) void k_embed_join(kd_embed_args a, Runs s) {
  __shared__ float s_sum[JOIN_W][64 * V];
  const int64_t unit = s.first + blockIdx.x, chunk = unit / s.tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = int(unit - chunk * s.tiles) * 64 * V + lane * V;
  const int64_t i0 = chunk * CHUNK, i1 = i0 + CHUNK;
  if (i1 >= a.n) return;  // (all uniform up to the sums)
  const uint32_t run = s.keys[i1 - 1];
  if (run == uint32_t(a.vocab) || s.keys[i1] != run || (i0 > 0 && s.keys[i0 - 1] == run)) return;
  int64_t more = 0;  // chunks behind this one that begin with the run
  for (;;) {
    const int64_t c = chunk + 1 + more + lane;
    const uint64_t in = __builtin_amdgcn_ballot_w64(c < s.chunks && s.keys[c * CHUNK] == run);
    const int k = in == ~uint64_t(0) ? 64 : __builtin_ctzll(~in);
    more += k;
    if (k < 64) break;
  }
  const int64_t c0 = chunk + 1 + more * wave / JOIN_W, c1 = chunk + 1 + more * (wave + 1) / JOIN_W;
  float sum[V];
#pragma unroll
  for (int k = 0; k < V; ++k) sum[k] = 0.f;
  if (col < a.dim) {
#pragma unroll 8
    for (int64_t c = c0; c < c1; ++c) {
      const float* p = s.part + 2 * c * a.dim + col;
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] += p[k];
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) s_sum[wave][lane * V + k] = sum[k];
  __syncthreads();
  if (wave != 0 || col >= a.dim) return;
  float f[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    f[k] = s.part[(2 * chunk + 1) * a.dim + col + k];
#pragma unroll
    for (int w = 0; w < JOIN_W; ++w) f[k] += s_sum[w][lane * V + k];
  }
  scaled<V>(f, a.scale);
  store_v<E, V>(a.dw, int64_t(run) * a.dim + col, f);
}

// Few positions: one launch.  A workgroup takes R rows of dW, lists in order the
// positions whose tokens lie among them, and for each row adds the listed rows of
// dy, eight in flight; rows without a token are written as zeros.
constexpr int SMALL_N = 512;
template <class E, int V>
__global__ __launch_bounds__(256) void k_embed_small(kd_embed_args a, int R) {
  __shared__ uint32_t s_list[SMALL_N + 64];  // position << 8 | row
  __shared__ int s_count[SMALL_N / 64 + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = int(a.n);
  const int64_t v0 = int64_t(blockIdx.x) * R;
  const int rows = int(min(int64_t(R), a.vocab - v0));
  // groups of 64 positions, two a wave
  uint64_t found[2];
  int row[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int i = (2 * wave + g) * 64 + lane;
    const int64_t at = i < n ? int64_t(key_at(a, i)) - v0 : -1;
    row[g] = int(at);
    const bool in = at >= 0 && at < rows;
    found[g] = __builtin_amdgcn_ballot_w64(in);
    if (lane == 0) s_count[2 * wave + g] = __builtin_popcountll(found[g]);
  }
  __syncthreads();
  int total = 0, before[2] = {0, 0};
#pragma unroll
  for (int g = 0; g < SMALL_N / 64; ++g) {
    if (g == 2 * wave) before[0] = total;
    if (g == 2 * wave + 1) before[1] = total;
    total += s_count[g];
  }
#pragma unroll
  for (int g = 0; g < 2; ++g)
    if ((found[g] >> lane) & 1u)
      s_list[before[g] + __builtin_popcountll(found[g] & ((uint64_t(1) << lane) - 1u))] =
          uint32_t((2 * wave + g) * 64 + lane) << 8 | uint32_t(row[g]);
  __syncthreads();
  for (int r = 0; r < rows; ++r) {
    for (int64_t c0 = 0; c0 < a.dim; c0 += 256 * V) {
      const int64_t col = c0 + tid * V;
      const bool in = col < a.dim;
      float sum[V];
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = 0.f;
      for (int g = 0; g < total; g += 64) {
        const uint32_t e = g + lane < total ? s_list[g + lane] : 0xFFFFFFFFu;
        uint64_t todo = __builtin_amdgcn_ballot_w64((e & 255u) == uint32_t(r) && g + lane < total);
        while (todo != 0) {  // (uniform, at most 8 rounds)
          float f[8][V];
          int m = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int k = 0; k < V; ++k) f[j][k] = 0.f;
            if (todo != 0) {
              const uint32_t p = uint32_t(__builtin_amdgcn_readlane(int(e), __builtin_ctzll(todo))) >> 8;
              todo &= todo - 1;
              m = j + 1;
              if (in) load_v<E, V>(a.dy, int64_t(p) * a.dim + col, f[j]);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < m)
#pragma unroll
              for (int k = 0; k < V; ++k) sum[k] += f[j][k];
        }
      }
      scaled<V>(sum, a.scale);
      if (in) store_v<E, V>(a.dw, (v0 + r) * a.dim + col, sum);
    }
  }
}

struct EmbedLayout {
  int64_t keys[2], idx[2], hist, part, total;  // bytes from the workspace's start
  int64_t chunks;
  int blocks, passes, bits;
};

EmbedLayout embed_layout(int64_t n, int64_t vocab, int64_t dim) {
  EmbedLayout L{};
  if (n <= SMALL_N) {
    L.total = 256;  // (nothing is needed; a pointer is)
    return L;
  }
  int bits = 1;
  while ((int64_t(1) << bits) <= vocab) ++bits;  // keys are 0 .. vocab
  L.passes = (bits + 10) / 11;
  L.bits = (bits + L.passes - 1) / L.passes;
  L.blocks = int((n + SORT_N - 1) / SORT_N);
  L.chunks = (n + CHUNK - 1) / CHUNK;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += (bytes + 255) / 256 * 256;
    return was;
  };
  for (int i = 0; i < 2; ++i) L.keys[i] = take(4 * n), L.idx[i] = take(4 * n);
  L.hist = take(int64_t(4) * L.blocks << L.bits);
  L.part = take(8 * L.chunks * dim);
  L.total = at;
  return L;
}

template <class F>
int by_type(int dtype, F f) {
  if (dtype == KD_BF16) f(BF16{});
  else if (dtype == KD_F16) f(F16{});
  else f(F32{});
  return hipGetLastError() == hipSuccess ? KD_OK : KD_ERR_LAUNCH;
}
template <int V>
using int_c = std::integral_constant<int, V>;

// Four values at a time where rows and bases allow it
bool by_four(const kd_embed_args& a, std::initializer_list<const void*> ps) {
  bool ok = a.dim % 4 == 0;
  for (const void* p : ps) ok &= reinterpret_cast<uintptr_t>(p) % 16 == 0;
  return ok;
}

}  // namespace

int64_t embed_grad_ws_bytes(int64_t n, int64_t vocab, int64_t dim) { return embed_layout(n, vocab, dim).total; }

int launch_embed(const kd_embed_args& a, hipStream_t st) {
  return by_type(a.dtype, [&](auto e) {
    using E = decltype(e);
    auto go = [&](auto v) {
      constexpr int V = decltype(v)::value;
      const int64_t words = a.dim / V, most = std::max<int64_t>(1, (int64_t(1) << 31) / words);
      for (int64_t r = 0; r < a.n; r += most) {
        const int64_t all = std::min(most, a.n - r) * words;
        hipLaunchKernelGGL((k_embed<E, V>), dim3(unsigned((all + 255) / 256)), dim3(256), 0, st, a, r, uint32_t(all),
                           uint32_t(words));
      }
    };
    if constexpr (!std::is_same_v<E, F32>)
      if (a.dim % 8 == 0 && by_four(a, {a.weight, a.out})) return go(int_c<8>{});
    if (by_four(a, {a.weight, a.out})) go(int_c<4>{});
    else go(int_c<1>{});
  });
}

int launch_embed_grad(const kd_embed_args& a, uint8_t* ws, hipStream_t st) {
  if (a.n <= SMALL_N)
    return by_type(a.dtype, [&](auto e) {
      using E = decltype(e);
      // (255 rows at most fit the list; a launch is less than 2^32 threads)
      const int R = a.vocab >= (int64_t(1) << 29) ? 255 : int(std::max<int64_t>(1, std::min<int64_t>(64, a.vocab / 1024)));
      auto go = [&](auto v) {
        hipLaunchKernelGGL((k_embed_small<E, decltype(v)::value>), dim3(unsigned((a.vocab + R - 1) / R)), dim3(256), 0, st, a, R);
      };
      if (by_four(a, {a.dy, a.dw})) go(int_c<4>{});
      else go(int_c<1>{});
    });
  const EmbedLayout L = embed_layout(a.n, a.vocab, a.dim);
  auto u32 = [&](int64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
  const int64_t bytes = a.vocab * a.dim * (a.dtype == KD_F32 ? 4 : 2);
  SortPass s{};
  s.bits = L.bits, s.blocks = L.blocks, s.hist = u32(L.hist);
  s.scanned = L.blocks > 64;
  for (int p = 0; p < L.passes; ++p) {
    s.keys = p == 0 ? nullptr : u32(L.keys[(p - 1) & 1]), s.idx = p == 0 ? nullptr : u32(L.idx[(p - 1) & 1]);
    s.keys_out = u32(L.keys[p & 1]), s.idx_out = u32(L.idx[p & 1]);
    s.shift = p * L.bits;
    const int count = L.blocks > 1 ? L.blocks : 0;
    const int fill = p == 0 ? int(std::min<int64_t>(1024, (bytes / 16 + SORT_T - 1) / SORT_T) + 1) : 0;
    if (count + fill > 0)
      hipLaunchKernelGGL(k_sort_count, dim3(count + fill), dim3(SORT_T), 0, st, a, s, bytes, count);
    if (s.scanned) hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(SORT_T), 0, st, s);
    hipLaunchKernelGGL(k_sort_move, dim3(L.blocks), dim3(SORT_T), 0, st, a, s);
  }
  return by_type(a.dtype, [&](auto e) {
    using E = decltype(e);
    auto go = [&](auto v) {
      constexpr int V = decltype(v)::value;
      Runs r{s.keys_out, s.idx_out, reinterpret_cast<float*>(ws + L.part), L.chunks, int((a.dim + 64 * V - 1) / (64 * V)), 0};
      const int64_t units = L.chunks * r.tiles, most = 1 << 22;  // (a launch is less than 2^32 threads)
      for (r.first = 0; r.first < units; r.first += 4 * most)
        hipLaunchKernelGGL((k_embed_runs<E, V>), dim3(unsigned((std::min(4 * most, units - r.first) + 3) / 4)), dim3(256), 0, st, a, r);
      for (r.first = 0; r.first < units; r.first += most)
        hipLaunchKernelGGL((k_embed_join<E, V>), dim3(unsigned(std::min(most, units - r.first))), dim3(64 * JOIN_W), 0, st, a, r);
    };
    if (by_four(a, {a.dy, a.dw})) go(int_c<4>{});
    else go(int_c<1>{});
  });
}

}  // namespace kd
