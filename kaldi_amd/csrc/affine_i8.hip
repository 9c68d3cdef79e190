// affine_i8.hip -- the affine product in 8-bit integers (kamd_component_i8_*):
//
//   out[m][n] = map(sum_k q[m][k] w[n][k] * scale[m] * w_scale[n] + bias[n]),   map(z) = mul[n] * relu(z) + add[n]
//
// The sum is exact: products of 8-bit codes in 32-bit integers (at most 131071 of them), by v_mfma_i32_16x16x64_i8.  It is
// turned into a 32-bit float once and rounded to the output's type once.
//
// The weights are laid out once, when the handle is made, in the order in which the matrix units take them: blocks of 16
// channels x 64 codes, 1 KB each, lane l of a wave holding channel l % 16, codes 16 (l / 16) .. +15, one 16-byte load per lane.
// A block is contiguous in memory, contiguous in LDS, and read from LDS without a bank conflict.  The 16 blocks of 256 channels
// that meet the same 64 codes lie side by side: a tile's stage is one stretch of memory, spread over all channels of the L2
// (with the blocks of one channel group side by side instead, they lay a power of two apart).  Channels are padded to
// kPadN and codes to kPadK with zeros, so that no kernel has to guard a weight, and so that whatever the activations' row holds
// beyond its last code meets a zero.
//
// The weights are operand A (rows = channels) and the activations operand B (columns = rows of the call): a lane then holds
// four consecutive channels of ONE row, i.e. one row scale and a contiguous piece of the output.
#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>
#include <vector>

#include "common.h"

namespace kamd {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr int kPadN = 256, kPadK = 128;
constexpr int64_t kMaxIn = 131071;        // 128 * 128 * 131071 < 2^31
constexpr int64_t kMaxLd = 1 << 23;       // a tile's rows stay within 32-bit offsets of its first
constexpr int64_t kMaxOut = 1 << 26;      // three vectors of them stay within 32-bit indexes
constexpr int64_t kMaxWeights = int64_t{1} << 35;
constexpr int64_t kMaxTiles = 1 << 22;    // per launch, of 512 threads: a launch has fewer than 2^32

struct AffineI8 {
  int device = 0, in_dim = 0, out_dim = 0, kp = 0, np = 0, relu = 0, mapped = 0;
  unsigned char *w = NULL;                // [np / 256][kp / 64][16][64 lanes][16]
  float *col = NULL;                      // [4][np]: w_scale, bias, mul, add
};

struct AffineArgs {
  const unsigned char *w;
  const int8_t *q;
  const float *scale;
  const float *col;
  void *out;
  int64_t ld_q, ld_out;
  int rows, n, np;
  int kb;                                 // 64-code blocks per channel = kp / 64
  int last_chunk;                         // byte offset of a row's last 16-byte chunk that may be read
  int relu, mapped;
  int tiles_m, tiles_n;
};

template <typename V, typename T>
__device__ inline void StoreAny(T *p, V v) { __builtin_memcpy(p, &v, sizeof(V)); }

typedef float f32x4 __attribute__((ext_vector_type(4)));

// the output of four consecutive channels n .. n + 3 (n < np) of one row, from their sums
__device__ inline f32x4 Finish(const AffineArgs &p, i32x4 acc, float scale, f32x4 w_scale, f32x4 bias, int n) {
  f32x4 z;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    z[j] = static_cast<float>(acc[j]) * w_scale[j] * scale + bias[j];
    if (p.relu) z[j] = z[j] < 0.0f ? 0.0f : z[j];                // (a NaN stays one)
  }
  if (p.mapped) {
    const f32x4 mul = *reinterpret_cast<const f32x4 *>(p.col + 2 * p.np + n), add = *reinterpret_cast<const f32x4 *>(p.col + 3 * p.np + n);
#pragma unroll
    for (int j = 0; j < 4; j++) z[j] = z[j] * mul[j] + add[j];
  }
  return z;
}

// values n .. n + VE - 1 of a row of the output; those behind its end are dropped
template <int VE, bool STREAM, typename TO, typename V>
__device__ inline void StoreRow(const AffineArgs &p, int m, int n, V v) {
  typedef V Unaligned __attribute__((aligned(sizeof(TO))));
  TO *o = static_cast<TO *>(p.out) + m * p.ld_out + n;
  if (n + VE <= p.n) {
    if (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<Unaligned *>(o));
    else StoreAny(o, v);
  } else
#pragma unroll
    for (int j = 0; j < VE; j++)
      if (n + j < p.n) o[j] = v[j];
}

// Workgroups are handed to the 8 XCDs in turn.  Each XCD takes one contiguous stretch of the tiles, and the stretch runs
// through bands of 8 row tiles, so that the tiles that are worked on at once share their operands in the XCD's L2.
__device__ inline void TileOf(int b, int tiles_m, int tiles_n, int *tm, int *tn) {
  const int all = tiles_m * tiles_n, xcd = b & 7, each = all >> 3, more = all & 7;
  const int i = xcd * each + min(xcd, more) + (b >> 3);
  constexpr int kBand = 8;
  const int band = i / (kBand * tiles_n), first = band * kBand, high = min(kBand, tiles_m - first), in = i - first * tiles_n;
  *tm = first + in % high;
  *tn = in / high;
}

// Few rows, or few tiles: what counts is how many loads are under way at once.  A workgroup computes 16 TI rows x 16 TJ channels;
// each of its 8 waves takes every 8th block of 64 codes of all of them, operands straight into registers, with no barrier until
// the sums are joined in LDS.  ONCE: the weights are read once by the call and not kept for the next.
template <int TI, int TJ, bool ONCE, typename TO>
__global__ __launch_bounds__(512) void SplitKernel(AffineArgs p) {
  constexpr int NW = 8, U = TI * TJ <= 2 ? 4 : 2;                // U blocks are loaded before the first is multiplied
  __shared__ i32x4 part[NW][TI * TJ][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  TileOf(blockIdx.x, p.tiles_m, p.tiles_n, &tm, &tn);
  const int m0 = tm * TI * 16, n0 = tn * TJ * 16;
  const unsigned char *w = p.w + (static_cast<size_t>(n0 / kPadN) * p.kb * 16 + n0 % kPadN / 16) * 1024 + lane * 16;
  const int8_t *x[TI];
#pragma unroll
  for (int i = 0; i < TI; i++) x[i] = p.q + static_cast<int64_t>(min(m0 + i * 16 + (lane & 15), p.rows - 1)) * p.ld_q;
  const int chunk = (lane >> 4) * 16;
  i32x4 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; i++)
#pragma unroll
    for (int j = 0; j < TJ; j++) acc[i][j] = i32x4{0, 0, 0, 0};
  for (int k0 = wave; k0 < p.kb; k0 += NW * U) {
    i32x4 a[U][TJ], b[U][TI];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (k0 + u * NW < p.kb) {
        const int k = k0 + u * NW, at = min(k * 64 + chunk, p.last_chunk);
#pragma unroll
        for (int j = 0; j < TJ; j++) {
          const i32x4 *block = reinterpret_cast<const i32x4 *>(w + (static_cast<size_t>(k) * 16 + j) * 1024);
          a[u][j] = ONCE ? __builtin_nontemporal_load(block) : *block;
        }
#pragma unroll
        for (int i = 0; i < TI; i++) b[u][i] = *reinterpret_cast<const i32x4 *>(x[i] + at);
      }
#pragma unroll
    for (int u = 0; u < U; u++)
      if (k0 + u * NW < p.kb)
#pragma unroll
        for (int i = 0; i < TI; i++)
#pragma unroll
          for (int j = 0; j < TJ; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][j], b[u][i], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < TI; i++)
#pragma unroll
    for (int j = 0; j < TJ; j++) part[wave][i * TJ + j][lane] = acc[i][j];
  __syncthreads();
  typedef TO OV __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int f0 = 0; f0 < TI * TJ; f0 += NW) {
    const int f = f0 + wave, m = m0 + f / TJ * 16 + (lane & 15), n = n0 + f % TJ * 16 + (lane >> 4) * 4;
    if (f >= TI * TJ || m >= p.rows || n >= p.n) continue;
    i32x4 s = part[0][f][lane];
#pragma unroll
    for (int v = 1; v < NW; v++) s += part[v][f][lane];
    const f32x4 z = Finish(p, s, p.scale[m], *reinterpret_cast<const f32x4 *>(p.col + n), *reinterpret_cast<const f32x4 *>(p.col + p.np + n), n);
    StoreRow<4, false, TO>(p, m, n, __builtin_convertvector(z, OV));
  }
}

typedef __attribute__((address_space(3))) unsigned char lds_byte;

// s_waitcnt: all but the newest LOADS * `stages` of this wave's loads are there (stages <= MOST), and its LDS reads
template <int LOADS, int MOST>
__device__ inline void WaitBut(int stages) {
  static_assert(LOADS * MOST < 64, "vmcnt has 6 bits");
  if constexpr (MOST > 0) {
    if (stages < MOST) return WaitBut<LOADS, MOST - 1>(stages);
  }
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS * MOST) : "memory");
}

// Many rows: BM rows x BN channels per workgroup of WM x WN waves, operands by DMA into a ring of NST stages of 128 codes in LDS.
// Large products are bound by the power that the matrix units draw: 16384 x 8192 x 8192 runs at 2.7 POP/s (816 us a call) with the
// clock at 1.9 GHz of 2.4 and the matrix units 67 % busy; the matrix instructions alone reach 4.6.  Sums of ~1536 codes keep them 43 % busy:
// a tile's first loads and its output take a third of its time, which the other tile on the CU covers in part.
template <int BM, int BN, int WM, int WN, int NST, bool STREAM, typename TO>
__global__ __launch_bounds__(WM * WN * 64) void TileKernel(AffineArgs p) {
  constexpr int NW = WM * WN, TI = BM / WM / 16, TJ = BN / WN / 16;
  constexpr int X_BYTES = BM * 128, W_BYTES = BN * 128, STAGE = X_BYTES + W_BYTES;
  constexpr int X_PW = BM / 8 / NW, W_PW = BN / 8 / NW, LOADS = X_PW + W_PW;       // 1 KB loads of a wave per stage
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BN <= kPadN, "tile");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[NST * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int tm, tn;
  TileOf(blockIdx.x, p.tiles_m, p.tiles_n, &tm, &tn);
  const int m0 = tm * BM, n0 = tn * BN, rows = min(BM, p.rows - m0);
  const unsigned lds = static_cast<unsigned>(reinterpret_cast<size_t>((lds_byte *)smem));

  // Buffer descriptors: base, extent, raw 32-bit data.  Every offset below stays inside by itself (rows clamped to the last
  // one, chunks to last_chunk).
  const size_t xb = reinterpret_cast<size_t>(p.q + static_cast<int64_t>(m0) * p.ld_q), wb = reinterpret_cast<size_t>(p.w + static_cast<size_t>(n0 / kPadN) * p.kb * (kPadN * 64));
  i32x4 xr = {static_cast<int>(xb), static_cast<int>((xb >> 32) & 0xffff), static_cast<int>((rows - 1) * p.ld_q + p.last_chunk + 16), 0x00027000};
  i32x4 wr = {static_cast<int>(wb), static_cast<int>((wb >> 32) & 0xffff), min(2, p.np / kPadN - n0 / kPadN) * kPadN * 64 * p.kb, 0x00027000};
#pragma unroll
  for (int i = 0; i < 4; i++) { xr[i] = __builtin_amdgcn_readfirstlane(xr[i]); wr[i] = __builtin_amdgcn_readfirstlane(wr[i]); }

  // Activations: a load covers 8 rows x 128 codes.  Chunk c (16 codes) of row r goes to slot c ^ ((r >> 1) & 7) of the row, so
  // that the 16 lanes that read one chunk of 16 rows touch all 64 banks once.
  int x_row[X_PW], x_chunk[X_PW];
#pragma unroll
  for (int i = 0; i < X_PW; i++) {
    const int r = (wave + NW * i) * 8 + (lane >> 3);
    x_row[i] = min(r, rows - 1) * static_cast<int>(p.ld_q);
    x_chunk[i] = ((lane & 7) ^ ((r >> 1) & 7)) * 16;
  }
  auto load = [&](unsigned to, i32x4 rsrc, int voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
  };
  // Where several tiles share a CU, tiles next to each other along a row start at different places of the sum, which is exact in
  // any order, so that not all of them ask for the same lines at once.  With inputs that change from call to call, us:  600 x 6000 x
  // 1536 13.2 -> 12.3, 40000 x 768 x 768 43.3 -> 41.1, but 12000 x 1536 x 1536 33.7 -> 34.8 and five other sizes 1 to 3 % slower.
  // Of no use to the other tiles.
  const int steps = p.kb >> 1, start = BM == 128 && NST == 2 ? (tn & 7) * 3 % steps : 0;
  auto issue = [&](int kt, int stage, int first, int last) {     // loads first .. last - 1 of this wave's for a stage
    kt += start;
    if (kt >= steps) kt -= steps;
    const unsigned at = lds + stage * STAGE;
#pragma unroll
    for (int l = 0; l < LOADS; l++) {
      if (l < first || l >= last) continue;
      if (l < X_PW) {
        load(at + (wave + NW * l) * 1024, xr, x_row[l] + min(kt * 128 + x_chunk[l], p.last_chunk), 0);
      } else {
        const int j = wave + NW * (l - X_PW), h = j / (BN / 16); // half h of the 128 codes, block j % (BN / 16) of 16 channels
        const int b = min(n0 / 16 + j % (BN / 16), p.np / 16 - 1) - n0 / kPadN * 16;
        load(at + X_BYTES + j * 1024, wr, lane * 16, ((((b >> 4) * p.kb + kt * 2 + h) << 4) + (b & 15)) * 1024);
      }
    }
  };

  i32x4 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; i++)
#pragma unroll
    for (int j = 0; j < TJ; j++) acc[i][j] = i32x4{0, 0, 0, 0};
  const int xoff = (wm * (BM / WM) + (lane & 15)) * 128, xslot = (lane >> 4) ^ ((lane >> 1) & 7);
  const int woff = X_BYTES + wn * (BN / WN / 16) * 1024 + lane * 16;
  struct Fragments { i32x4 w[TJ], x[TI]; } half0, half1;         // 64 codes each
  auto fetch_w = [&](int stage, int h, int j, Fragments *f) {
    f->w[j] = *reinterpret_cast<const i32x4 *>(smem + stage * STAGE + woff + (h * (BN / 16) + j) * 1024);
  };
  auto fetch_x = [&](int stage, int h, int i, Fragments *f) {
    f->x[i] = *reinterpret_cast<const i32x4 *>(smem + stage * STAGE + xoff + i * 2048 + ((xslot ^ (h * 4)) * 16));
  };
  // One half of a stage is multiplied while the next is read and a later stage is asked for: a few of each at a time, since a
  // wave issues in order and both the LDS and the load path would hold it up, the matrix unit idle, if asked all at once.
  // FETCH: the fragments of half `h` of `stage` go to `next`; LOAD: stage `kt` is loaded into `slot`.
  auto half = [&](const Fragments &now, Fragments *next, int stage, int h, auto fetch, auto load_too, int kt, int slot) {
#pragma unroll
    for (int i = 0; i < TI; i++) {
      if constexpr (decltype(fetch)::value) {
        fetch_x(stage, h, i, next);
#pragma unroll
        for (int j = i * TJ / TI; j < (i + 1) * TJ / TI; j++) fetch_w(stage, h, j, next);
      }
#pragma unroll
      for (int j = 0; j < TJ; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now.w[j], now.x[i], acc[i][j], 0, 0, 0);
      if constexpr (decltype(load_too)::value) issue(kt, slot, i * LOADS / TI, (i + 1) * LOADS / TI);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  typedef std::integral_constant<bool, true> Yes;
  typedef std::integral_constant<bool, false> No;
#pragma unroll
  for (int t = 0; t < NST; t++)
    if (t < steps) issue(t, t, 0, LOADS);
  WaitBut<LOADS, NST - 1>(min(NST, steps) - 1);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int j = 0; j < TJ; j++) fetch_w(0, 0, j, &half0);
#pragma unroll
  for (int i = 0; i < TI; i++) fetch_x(0, 0, i, &half0);
  int stage = 0, kt = 0;
  auto next_stage = [&]() {
    __builtin_amdgcn_s_barrier();                                // the next stage is there, and this one has been read by all
    asm volatile("" ::: "memory");
    stage = stage + 1 == NST ? 0 : stage + 1;
  };
  for (; kt + NST < steps; kt++) {
    half(half0, &half1, stage, 1, Yes(), No(), 0, 0);
    WaitBut<LOADS, NST - 2>(NST - 2);
    const int slot = stage;
    next_stage();
    half(half1, &half0, stage, 0, Yes(), Yes(), kt + NST, slot);
  }
  for (; kt + 1 < steps; kt++) {
    half(half0, &half1, stage, 1, Yes(), No(), 0, 0);
    WaitBut<LOADS, NST - 2>(min(NST - 2, steps - 2 - kt));
    next_stage();
    half(half1, &half0, stage, 0, Yes(), No(), 0, 0);
  }
  half(half0, &half1, stage, 1, Yes(), No(), 0, 0);
  half(half1, &half0, stage, 0, No(), No(), 0, 0);

  // The output leaves in whole cache lines: a lane holds 4 channels of one row, so that stores from the registers would touch
  // 16 rows with 8 to 16 bytes each.  Every wave turns its tile through a corner of the LDS of its own, 16 rows at a time.
  constexpr int VE = 16 / static_cast<int>(sizeof(TO)), COLS = BN / WN, PITCH = COLS * static_cast<int>(sizeof(TO)) + 16, LPR = COLS / VE, RPI = 64 / LPR;
  static_assert(NW * 16 * PITCH <= NST * STAGE && LPR <= 64 && RPI <= 16, "epilogue");
  typedef TO OV __attribute__((ext_vector_type(VE)));
  typedef TO OV4 __attribute__((ext_vector_type(4)));
  __syncthreads();
  unsigned char *mine = smem + wave * 16 * PITCH;
  const int nw = n0 + wn * COLS, n4 = nw + (lane >> 4) * 4;
  // All that it reads is asked for first: a wave's loads and stores are counted in order, so that a load between the stores
  // waits for those before it (256 x 256 tiles 3 to 6 % slower, 128 x 192 1 to 2 %).
  f32x4 w_scale[TJ], bias[TJ];
  float x_scale[TI];
#pragma unroll
  for (int j = 0; j < TJ; j++) {
    const int n = min(n4 + j * 16, p.np - 4);
    w_scale[j] = *reinterpret_cast<const f32x4 *>(p.col + n);
    bias[j] = *reinterpret_cast<const f32x4 *>(p.col + p.np + n);
  }
#pragma unroll
  for (int i = 0; i < TI; i++) x_scale[i] = p.scale[min(m0 + wm * (BM / WM) + i * 16 + (lane & 15), p.rows - 1)];
#pragma unroll
  for (int i = 0; i < TI; i++) {
    const int mi = m0 + wm * (BM / WM) + i * 16;
#pragma unroll
    for (int j = 0; j < TJ; j++) {
      const f32x4 z = Finish(p, acc[i][j], x_scale[i], w_scale[j], bias[j], min(n4 + j * 16, p.np - 4));
      StoreAny(mine + (lane & 15) * PITCH + ((lane >> 4) * 4 + j * 16) * sizeof(TO), __builtin_convertvector(z, OV4));
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += RPI) {                       // LPR lanes to a row, RPI rows at once
      const int r = r0 + lane / LPR, n = nw + lane % LPR * VE;
      if ((64 % LPR == 0 || (lane < RPI * LPR && r < 16)) && mi + r < p.rows && n < p.n) {
        OV v;
        __builtin_memcpy(&v, mine + r * PITCH + lane % LPR * 16, 16);
        StoreRow<VE, STREAM, TO>(p, mi + r, n, v);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// [n x k] codes -> the layout above; one thread per 16 codes
__global__ __launch_bounds__(256) void PackKernel(const int8_t *w, int64_t ld, int n, int k, int kb, unsigned char *to, int64_t chunks) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= chunks) return;
  const int lane = static_cast<int>(i & 63);
  const int64_t block = i >> 6, step = block >> 4;               // 16 blocks of 16 channels to a step of 64 codes
  const int row = static_cast<int>(step / kb) * kPadN + static_cast<int>(block & 15) * 16 + (lane & 15);
  const int at = static_cast<int>(step % kb) * 64 + (lane >> 4) * 16;
  int8_t v[16];
#pragma unroll
  for (int j = 0; j < 16; j++) v[j] = row < n && at + j < k ? w[row * ld + at + j] : 0;
  __builtin_memcpy(to + i * 16, v, 16);
}

// the four vectors of the output channels, padded to np; NULL = the neutral value
__global__ __launch_bounds__(256) void ColumnsKernel(const float *w_scale, const float *bias, const float *mul, const float *add, int n, int np, float *to) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= np) return;
  const bool in = i < n;
  to[i] = in ? w_scale[i] : 0.0f;
  to[np + i] = in && bias ? bias[i] : 0.0f;
  to[2 * np + i] = in && mul ? mul[i] : 1.0f;
  to[3 * np + i] = in && add ? add[i] : 0.0f;
}

// Weights that the L2s (8 x 4 MB) cannot hold until the next call pass them by where a split kernel reads them for at most 16 rows
// (us from HBM, in brackets from the last-level cache):  1 x 8192 x 8192  13.7 -> 12.1 (11.1 -> 11.3),  16 x 8192 x 8192  14.6 -> 13.3
// (11.9 -> 12.8).  Not from 24 rows on, 16.3 -> 15.1 (12.3 -> 14.6), nor smaller ones:  1 x 4096 x 4096  5.0 -> 4.8 (L2s 3.1 -> 4.5).
// From some 12000 channels on the cost rule below, which counts no bytes, takes LDS tiles for such calls, which read the weights
// through the caches:  1 x 16384 x 4096  11.6 (16 x 16 split 9.9),  1 x 65536 x 8192  96 (75).
constexpr int64_t kL2Bytes = 32 << 20;

template <int TI, int TJ, typename TO>
void LaunchSplit(AffineArgs p, hipStream_t st) {
  p.tiles_m = CeilDiv(p.rows, TI * 16); p.tiles_n = CeilDiv(p.n, TJ * 16);
  const dim3 grid(p.tiles_m * p.tiles_n), block(512);
  if (p.rows <= 16 && static_cast<int64_t>(p.np) * p.kb * 64 > kL2Bytes)
    hipLaunchKernelGGL((SplitKernel<TI, TJ, true, TO>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((SplitKernel<TI, TJ, false, TO>), grid, block, 0, st, p);
}

// An output that the last-level cache (256 MB) could not keep for the next layer anyway goes past the caches, whose lines the
// operands need more.  A smaller one does not: the next layer would have to fetch it.  256 x 256 tiles with the coding of the rows
// behind them, us, kept -> past:  98 MB 80 -> 88,  134 MB 145 -> 149,  164 MB 199 -> 196,  201 MB 249 -> 234,  268 MB (16384 x 8192
// x 8192) 893 -> 883, that product alone 830 -> 738.
constexpr int64_t kStreamBytes = 128 << 20;

template <int BM, int BN, int WM, int WN, int NST, typename TO>
void LaunchTile(AffineArgs p, hipStream_t st) {
  p.tiles_m = CeilDiv(p.rows, BM); p.tiles_n = CeilDiv(p.n, BN);
  const dim3 grid(p.tiles_m * p.tiles_n), block(WM * WN * 64);
  if (static_cast<int64_t>(p.rows) * p.n * static_cast<int64_t>(sizeof(TO)) > kStreamBytes)
    hipLaunchKernelGGL((TileKernel<BM, BN, WM, WN, NST, true, TO>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((TileKernel<BM, BN, WM, WN, NST, false, TO>), grid, block, 0, st, p);
}

// Which kernel.  A call takes about  2 us + c (s step + fixed),  c = tiles per CU, s = steps of 128 codes, with the two constants
// of each kernel measured on MI355X; the cheapest is taken.  Over 200 random sizes that is 1.3 % from the fastest of them in the
// mean, 14 % at most in calls of over 5 us (12000 x 6000 x 256).  Bytes are not counted, see above.
// What the kernels are for, each against its neighbour (us, in a loop over the same operands):
//   16 x 16 split    1 x 4096 x 4096  3.1 (32 x 32  4.1)          20 x 320 x 7840  5.3 (7.5)
//   32 x 32 split    24 x 6000 x 1536  3.7 (16 x 16  4.8)         64 x 4096 x 4096  6.8 (64 x 64  8.8)
//   64 x 64, 4 st.   256 x 4096 x 4096  9.4   (64 x 128 11.6)     1000 x 768 x 768  4.0 (4.8)
//   64 x 128, 3 st.  512 x 4096 x 4096  12.5  (64 x 64 14.1)      600 x 6000 x 1536  10.2 (128 x 192 11.2)
//   128 x 192, 3 st. 1999 x 2328 x 1537 12.5  (64 x 128 14.7, 2 stages 13.6): one tile per CU, so that it can have all the LDS
//   128 x 192, 2 st. 12000 x 1536 x 1536 32.4 (256 x 256 43.2, 3 stages 33.8): two tiles per CU cover each other's waits
//   256 x 256, 2 st. 4096 x 4096 x 4096 52.3  (128 x 192 65.7)    16384 x 8192 x 8192  738 (881)
constexpr int kCus = 256;

constexpr int kMaxRows = 1 << 22;         // per launch: the grid of the smallest tile stays within its limit

template <typename TO>
int Propagate(AffineArgs p, hipStream_t st) {
  if (p.rows > kMaxRows) {
    AffineArgs rest = p;
    rest.q += static_cast<int64_t>(kMaxRows) * p.ld_q; rest.scale += kMaxRows; rest.rows -= kMaxRows;
    rest.out = static_cast<TO *>(p.out) + static_cast<int64_t>(kMaxRows) * p.ld_out;
    p.rows = kMaxRows;
    const int rc = Propagate<TO>(p, st);
    return rc != KAMD_OK ? rc : Propagate<TO>(rest, st);
  }
  struct Kernel { int bm, bn; double step, fixed; bool alone; void (*go)(AffineArgs, hipStream_t); };     // alone: at most one tile per CU
  static const Kernel kernels[] = {{16, 16, 0.065, 0.2, false, LaunchSplit<1, 1, TO>},
                                   {32, 32, 0.115, 0.3, false, LaunchSplit<2, 2, TO>},
                                   {64, 64, 0.19, 0.9, false, LaunchTile<64, 64, 4, 2, 4, TO>},
                                   {64, 128, 0.29, 1.2, false, LaunchTile<64, 128, 2, 4, 3, TO>},
                                   {128, 192, 0.40, 5.0, true, LaunchTile<128, 192, 2, 4, 3, TO>},
                                   {128, 192, 0.62, 2.8, false, LaunchTile<128, 192, 2, 4, 2, TO>},
                                   {256, 256, 1.42, 8.0, false, LaunchTile<256, 256, 2, 4, 2, TO>}};
  const Kernel *best = NULL;
  double least = 0.0;
  for (const Kernel &k : kernels) {
    const int64_t tiles = static_cast<int64_t>(CeilDiv(p.rows, k.bm)) * CeilDiv(p.n, k.bn), per_cu = (tiles + kCus - 1) / kCus;
    if ((k.alone && per_cu > 1) || tiles > kMaxTiles) continue;
    const double cost = static_cast<double>(per_cu) * (p.kb / 2 * k.step + k.fixed);
    if (!best || cost < least) { best = &k; least = cost; }
  }
  if (!best) return SetError(KAMD_ERR_ARG, "kamd_component_i8_propagate: %d rows of %d outputs are too many for one call", p.rows, p.n);
  best->go(p, st);
  KAMD_HIP(hipGetLastError());
  return KAMD_OK;
}

// An error that is told to the caller, or of no consequence, is not left to be found as the thread's last one by whoever asks next
// (torch does after each of its launches).
hipError_t Told(hipError_t e) {
  if (e != hipSuccess) (void)hipGetLastError();
  return e;
}

// For this thread, in this scope: allocating and freeing do not break a capture that is under way on some stream (a handle goes
// when its last owner lets go of it, from the garbage collector perhaps, and hipFree would invalidate the capture and free nothing).
struct OutsideCaptures {
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  OutsideCaptures() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
  ~OutsideCaptures() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
};

void Free(AffineI8 *c) {
  if (!c) return;
  const OutsideCaptures guard;
  for (void *p : {static_cast<void *>(c->w), static_cast<void *>(c->col)})
    if (p) Told(hipFree(p));
  delete c;
}

// A handle is filled here and now; a stream that is being captured does nothing now, and allocating would invalidate the capture.
bool RefuseCapture(const char *who, hipStream_t st) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(st, &status) == hipSuccess && status == hipStreamCaptureStatusNone) return false;
  (void)hipGetLastError();
  SetError(KAMD_ERR_STATE, "%s: the stream is being captured: layers are made before", who);
  return true;
}

int CheckSizes(const char *who, int64_t in_dim, int64_t out_dim) {
  if (in_dim < 1 || out_dim < 1) return SetError(KAMD_ERR_ARG, "%s: bad sizes (%lld -> %lld)", who, static_cast<long long>(in_dim), static_cast<long long>(out_dim));
  if (in_dim > kMaxIn) return SetError(KAMD_ERR_ARG, "%s: %lld inputs: a 32-bit sum of 8-bit products holds at most %lld", who, static_cast<long long>(in_dim), static_cast<long long>(kMaxIn));
  if (out_dim > kMaxOut || static_cast<int64_t>(RoundUp(out_dim, kPadN)) * RoundUp(in_dim, kPadK) > kMaxWeights)
    return SetError(KAMD_ERR_ARG, "%s: too many outputs (%lld of %lld inputs)", who, static_cast<long long>(out_dim), static_cast<long long>(in_dim));
  return KAMD_OK;
}

}  // namespace
}  // namespace kamd
using kamd::AffineI8;
using kamd::SetError;

extern "C" {

kamd_component_i8 *kamd_component_i8_create_quantized(const int8_t *d_w, int64_t ld_w, const float *d_w_scale, int in_dim, int out_dim,
                                                      const float *d_bias, int relu, const float *d_mul, const float *d_add, void *stream) {
  if (kamd::CheckSizes("kamd_component_i8_create_quantized", in_dim, out_dim) != KAMD_OK) return NULL;
  if (!d_w || !d_w_scale || ld_w < in_dim) { SetError(KAMD_ERR_ARG, "kamd_component_i8_create_quantized: null argument or leading dimension smaller than the matrix"); return NULL; }
  if (!kamd::RequireDevice() || kamd::RefuseCapture("kamd_component_i8_create_quantized", static_cast<hipStream_t>(stream))) return NULL;
  AffineI8 *c = new (std::nothrow) AffineI8();
  if (!c) { SetError(KAMD_ERR_HIP, "kamd_component_i8_create_quantized: out of memory"); return NULL; }
  c->in_dim = in_dim; c->out_dim = out_dim; c->kp = kamd::RoundUp(in_dim, kamd::kPadK); c->np = kamd::RoundUp(out_dim, kamd::kPadN);
  c->relu = relu != 0; c->mapped = d_mul || d_add;
  const size_t bytes = static_cast<size_t>(c->np) * c->kp;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = hipGetDevice(&c->device);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&c->w), bytes);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&c->col), sizeof(float) * 4 * c->np);
  if (e == hipSuccess) {
    hipLaunchKernelGGL(kamd::PackKernel, dim3(kamd::CeilDiv(static_cast<int64_t>(bytes / 16), 256)), dim3(256), 0, st, d_w, ld_w, out_dim, in_dim, c->kp / 64,
                       c->w, static_cast<int64_t>(bytes / 16));
    hipLaunchKernelGGL(kamd::ColumnsKernel, dim3(kamd::CeilDiv(c->np, 256)), dim3(256), 0, st, d_w_scale, d_bias, d_mul, d_add, out_dim, c->np, c->col);
    e = hipGetLastError();
  }
  if (e == hipSuccess) e = hipStreamSynchronize(st);             // the caller's arrays may go, and any stream may use the handle
  if (kamd::Told(e) != hipSuccess) {
    SetError(KAMD_ERR_HIP, "kamd_component_i8_create_quantized: %s", hipGetErrorString(e));
    kamd::Free(c);
    return NULL;
  }
  return reinterpret_cast<kamd_component_i8 *>(c);
}

kamd_component_i8 *kamd_component_i8_create(const kamd_layer_desc *layer) {
  if (!layer || layer->ivector_dim != 0 || layer->multi_input || layer->log_softmax || layer->n_offsets < 1 || layer->n_offsets > KAMD_MAX_OFFSETS || !layer->W) {
    SetError(KAMD_ERR_ARG, "kamd_component_i8_create: a plain fused layer is expected (weights; no ivector, multi_input or log-softmax)");
    return NULL;
  }
  const int64_t k = static_cast<int64_t>(layer->in_dim) * layer->n_offsets;
  const int n = layer->out_dim;
  if (kamd::CheckSizes("kamd_component_i8_create", layer->in_dim < 1 ? 0 : k, n) != KAMD_OK) return NULL;
  const size_t values = static_cast<size_t>(n) * k;
  for (size_t i = 0; i < values; i++)
    if (!std::isfinite(layer->W[i])) { SetError(KAMD_ERR_ARG, "kamd_component_i8_create: weight %zu is not finite", i); return NULL; }
  if (!kamd::RequireDevice() || kamd::RefuseCapture("kamd_component_i8_create", NULL)) return NULL;
  // weights, their codes and scales, and the channel vectors: one allocation, released below
  const size_t f_w = values, f_col = static_cast<size_t>(n) * 4, bytes = (f_w + f_col) * 4 + values;
  float *d = NULL;
  hipError_t e = hipMalloc(reinterpret_cast<void **>(&d), bytes);
  if (kamd::Told(e) != hipSuccess) { SetError(KAMD_ERR_HIP, "kamd_component_i8_create: %s", hipGetErrorString(e)); return NULL; }
  float *d_scale = d + f_w, *d_bias = d_scale + n, *d_mul = d_bias + n, *d_add = d_mul + n;
  int8_t *d_q = reinterpret_cast<int8_t *>(d_add + n);
  // BatchNorm and post maps: (bn_scale * z + bn_offset + post_offset) * post_scale
  const bool mapped = layer->bn_scale || layer->bn_offset || layer->post_offset || layer->post_scale != 1.0f;
  kamd_component_i8 *c = NULL;
  try {
    std::vector<float> mul(n), add(n);
    for (int i = 0; i < n; i++) {
      mul[i] = (layer->bn_scale ? layer->bn_scale[i] : 1.0f) * layer->post_scale;
      add[i] = ((layer->bn_offset ? layer->bn_offset[i] : 0.0f) + (layer->post_offset ? layer->post_offset[i] : 0.0f)) * layer->post_scale;
    }
    e = hipMemcpy(d, layer->W, values * 4, hipMemcpyHostToDevice);
    if (e == hipSuccess && layer->bias) e = hipMemcpy(d_bias, layer->bias, sizeof(float) * n, hipMemcpyHostToDevice);
    if (e == hipSuccess && mapped) e = hipMemcpy(d_mul, mul.data(), sizeof(float) * n, hipMemcpyHostToDevice);
    if (e == hipSuccess && mapped) e = hipMemcpy(d_add, add.data(), sizeof(float) * n, hipMemcpyHostToDevice);
    const int32_t zero = 0;
    if (kamd::Told(e) != hipSuccess) SetError(KAMD_ERR_HIP, "kamd_component_i8_create: %s", hipGetErrorString(e));
    else if (kamd_quantize_rows_device(d, k, KAMD_F32, n, static_cast<int>(k), &zero, 1, d_q, k, d_scale, NULL) == KAMD_OK)
      c = kamd_component_i8_create_quantized(d_q, k, d_scale, static_cast<int>(k), n, layer->bias ? d_bias : NULL, layer->relu, mapped ? d_mul : NULL,
                                             mapped ? d_add : NULL, NULL);
  } catch (const std::exception &) {
    SetError(KAMD_ERR_HIP, "kamd_component_i8_create: out of memory");
  }
  kamd::Told(hipFree(d));
  return c;
}

void kamd_component_i8_destroy(kamd_component_i8 *h) { kamd::Free(reinterpret_cast<AffineI8 *>(h)); }
int kamd_component_i8_input_dim(const kamd_component_i8 *h) { return reinterpret_cast<const AffineI8 *>(h)->in_dim; }
int kamd_component_i8_output_dim(const kamd_component_i8 *h) { return reinterpret_cast<const AffineI8 *>(h)->out_dim; }

int kamd_component_i8_propagate(const kamd_component_i8 *h, const int8_t *d_q, int64_t ld_q, const float *d_scale, int64_t rows, void *d_out,
                                int64_t ld_out, int out_type, void *stream) {
  const AffineI8 *c = reinterpret_cast<const AffineI8 *>(h);
  if (!c || rows < 0 || rows > INT32_MAX - kamd::kPadN) return SetError(KAMD_ERR_ARG, "kamd_component_i8_propagate: null handle or bad number of rows (%lld)", static_cast<long long>(rows));
  if (out_type != KAMD_F32 && out_type != KAMD_BF16 && out_type != KAMD_F16) return SetError(KAMD_ERR_ARG, "kamd_component_i8_propagate: unknown output type %d", out_type);
  if (ld_q < c->in_dim || ld_out < c->out_dim) return SetError(KAMD_ERR_ARG, "kamd_component_i8_propagate: leading dimension smaller than the matrix");
  if (ld_q % 16 != 0 || ld_q > kamd::kMaxLd || reinterpret_cast<uintptr_t>(d_q) % 16 != 0)
    return SetError(KAMD_ERR_ARG, "kamd_component_i8_propagate: rows of codes begin on multiples of 16 bytes, at most %lld apart", static_cast<long long>(kamd::kMaxLd));
  if (rows == 0) return KAMD_OK;
  if (!d_q || !d_scale || !d_out) return SetError(KAMD_ERR_ARG, "kamd_component_i8_propagate: null argument");
  const kamd::MemoryRows out = kamd::RowsOf(d_out, ld_out, c->out_dim, out_type == KAMD_F32 ? 4 : 2, rows);
  if (RowsMeet(out, kamd::RowsOf(d_q, ld_q, c->in_dim, 1, rows)) || RowsMeet(out, kamd::RowsOf(d_scale, rows, rows, 4, 1)))
    return SetError(KAMD_ERR_ARG, "kamd_component_i8_propagate: the output overlaps another argument");
  int device = -1;
  KAMD_HIP(hipGetDevice(&device));
  if (device != c->device) return SetError(KAMD_ERR_STATE, "kamd_component_i8_propagate: the handle belongs to device %d, the current one is %d", c->device, device);
  kamd::AffineArgs a = {};
  a.w = c->w; a.q = d_q; a.scale = d_scale; a.col = c->col; a.out = d_out; a.ld_q = ld_q; a.ld_out = ld_out;
  a.rows = static_cast<int>(rows); a.n = c->out_dim; a.np = c->np; a.kb = c->kp / 64; a.last_chunk = kamd::RoundUp(c->in_dim, 16) - 16;
  a.relu = c->relu; a.mapped = c->mapped;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (out_type == KAMD_F32) return kamd::Propagate<float>(a, st);
  if (out_type == KAMD_BF16) return kamd::Propagate<__bf16>(a, st);
  return kamd::Propagate<_Float16>(a, st);
}

}  // extern "C"
