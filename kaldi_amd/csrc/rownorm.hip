// rownorm.hip -- rows of a matrix normalised by their root mean square, and rows coded in 8 bits.
//
//   kamd_rms_norm_device       h = x + residual,  y = h / sqrt(mean(h^2) + eps) * gain      (NormalizeComponent's kernel,
//                              nnet3/nnet-normalize-component.cc, cudamatrix/cu-math.cc NormalizePerRow, with the gain and
//                              the residual of a pre-norm layer); y in the input's type, or in 8 bits with a scale per row
//   kamd_quantize_rows_device  the 8-bit form of a (spliced) matrix, for layers whose input is not normalised
//
// 8-bit rows.  With t = h * gain, r = 1 / sqrt(mean(h^2) + eps) and a = max |t|, the row y = t * r is held as
//   code q = rint(t * (127 / a)),   scale = a * r / 127,   y ~ q * scale,   |y - q * scale| <= scale / 2.
// r > 0 cancels in the codes: they need a alone, so the sum of squares and the maximum are reduced TOGETHER, in one pass and
// one exchange between the threads of a row, and y itself is never formed or rounded.
//
// Numbers: h and t are 32-bit; squares are summed in 64 bits (a row of bf16 values near 1e20 has no 32-bit sum of squares, and
// the conversion hides behind the loads); every output is rounded once.
//
// What bounds it: the bytes, for rows of some hundred columns and splices of up to 3 such pieces.  Each row is read once and stays in registers (up to 48
// elements per thread) between the reduction and the output, rows longer than 32768 elements excepted, which are read twice, and
// splices of many pieces, each of which is rounded up to a pass of all the row's threads (RunRows).
#include <cfloat>
#include <cmath>

#include "common.h"

namespace kamd {

struct RowArgs {
  const void *x, *residual;
  void *sum, *out;
  float *out_scale;
  const float *gain;
  int64_t ld_x, ld_residual, ld_sum, ld_out;
  int64_t rows;
  float eps;
  // a spliced row is n_parts pieces of part_dim columns; piece p of output row r begins at x[r * ld_x + part_at[p]]
  int part_dim, n_parts;
  int64_t part_at[KAMD_MAX_OFFSETS];
};

// The widest access is used whatever the address: rows of odd length start anywhere, and MI355X's global loads and stores
// need no more than the element's own alignment.
template <typename V, typename T>
__device__ inline V LoadAny(const T *p) { V v; __builtin_memcpy(&v, p, sizeof(V)); return v; }
// v without its first `skip` elements
template <int VE, typename V, typename T>
__device__ inline void StoreFrom(T *p, V v, int skip, bool whole) {
  if (whole || skip == 0) { __builtin_memcpy(p, &v, sizeof(V)); return; }
#pragma unroll
  for (int j = 1; j < VE; j++)
    if (j >= skip) p[j] = v[j];
}

// Over the 64 lanes, without going through the LDS: shifts inside rows of 16 lanes, then lane 15 of a row to the next row and
// lane 31 to the upper half; lane 63 holds the result and hands it to all.  Lanes that receive nothing keep 0.
template <int CTRL, int ROWS>
__device__ inline uint32_t Moved(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false)); }
template <int CTRL, int ROWS>
__device__ inline double Moved(double v) {
  uint32_t w[2];
  __builtin_memcpy(w, &v, 8);
  w[0] = Moved<CTRL, ROWS>(w[0]); w[1] = Moved<CTRL, ROWS>(w[1]);
  __builtin_memcpy(&v, w, 8);
  return v;
}
__device__ inline double WaveSum(double v) {
  v += Moved<0x111, 0xf>(v); v += Moved<0x112, 0xf>(v); v += Moved<0x114, 0xf>(v); v += Moved<0x118, 0xf>(v);
  v += Moved<0x142, 0xa>(v); v += Moved<0x143, 0xc>(v);
  uint32_t w[2];
  __builtin_memcpy(w, &v, 8);
  w[0] = __builtin_amdgcn_readlane(w[0], 63); w[1] = __builtin_amdgcn_readlane(w[1], 63);
  __builtin_memcpy(&v, w, 8);
  return v;
}
__device__ inline uint32_t WaveMax(uint32_t v) {
  v = max(v, Moved<0x111, 0xf>(v)); v = max(v, Moved<0x112, 0xf>(v)); v = max(v, Moved<0x114, 0xf>(v)); v = max(v, Moved<0x118, 0xf>(v));
  v = max(v, Moved<0x142, 0xa>(v)); v = max(v, Moved<0x143, 0xc>(v));
  return __builtin_amdgcn_readlane(v, 63);
}

// T: the input's type; TO: the output's (T or int8_t); NORM: false = coding alone; VE: elements per access; TPR: threads per row;
// NV: accesses per thread, held in registers; 0 = as many as it takes, the row being read twice.
//
// A row (each piece of a spliced one) is cut into accesses of VE elements.  The last one is moved back to end where the piece
// ends; what it has in common with the one before stays that one's: it counts as zero and is not stored.  Threads beyond the
// last access repeat it in the same way, with nothing of their own.  So no length needs loads of single elements, and nothing
// that is held in registers is written under a condition (which costs a copy of all of them).  Every element is read and
// written by one thread, which is what lets outputs lie over inputs.
template <typename T, typename TO, bool NORM, int VE, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void RowKernel(RowArgs a) {
  constexpr bool I8 = sizeof(TO) == 1;
  constexpr int BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR, NW = TPR / 64;
  typedef T TV __attribute__((ext_vector_type(VE)));
  typedef TO OV __attribute__((ext_vector_type(VE)));
  typedef float FV __attribute__((ext_vector_type(VE)));
  const int t = RPB == 1 ? threadIdx.x : threadIdx.x & (TPR - 1);
  // Spliced rows share their pieces with rows near them: each of the 8 XCDs, which are handed workgroups in turn, takes one
  // stretch of the rows, so that the pieces are found in its L2.
  const unsigned group = !NORM && a.n_parts > 1 ? (blockIdx.x & 7) * (gridDim.x >> 3) + min(blockIdx.x & 7, gridDim.x & 7) + (blockIdx.x >> 3) : blockIdx.x;
  const int64_t row = static_cast<int64_t>(group) * RPB + (RPB == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR));
  if (row >= a.rows) return;                                     // (a whole wave; a whole workgroup where there is a barrier)
  const T *x = static_cast<const T *>(a.x) + row * a.ld_x;
  const T *res = NORM && a.residual ? static_cast<const T *>(a.residual) + row * a.ld_residual : NULL;
  T *sum = NORM && a.sum ? static_cast<T *>(a.sum) + row * a.ld_sum : NULL;
  TO *out = static_cast<TO *>(a.out) + row * a.ld_out;
  // Access c of piece p takes columns k .. k + VE - 1 of the piece for every thread, k = (c TPR + t) VE: p and c are the same for
  // all threads, so that finding one's place is scalar work.  `skip`: the first elements that are not this access's own.
  const int per_part = (a.part_dim + TPR * VE - 1) / (TPR * VE);                 // accesses per piece
  const int parts = NORM ? 1 : a.n_parts;
  struct Place { int64_t from; int to, skip; bool whole; };
  auto place = [&](int p, int c) {
    Place w;
    const int k = (c * TPR + t) * VE, at = min(k, a.part_dim - VE);
    w.from = (NORM ? 0 : a.part_at[p]) + at;
    w.to = p * a.part_dim + at;
    w.skip = k - at;
    w.whole = (c + 1) * TPR * VE <= a.part_dim;                  // nobody skips anything
    return w;
  };
  // (p, c) of the register slots in turn; slots that are left over repeat the last piece behind its end
  struct Slot { int p, c; };
  auto next = [&](Slot s) {
    s.c++;
    if (s.c == per_part && s.p + 1 < parts) { s.c = 0; s.p++; }
    return s;
  };
  auto gains = [&](int k) {
    FV g;
    if (NORM && a.gain) return LoadAny<FV>(a.gain + k);
#pragma unroll
    for (int j = 0; j < VE; j++) g[j] = 1.0f;
    return g;
  };

  double ss = 0.0;
  uint32_t most = 0;                                             // bits of max |t|: ordered like the values, NaN on top
  // h into the row's statistics and, with its place, to `sum`; returns what the output is made of: h, or t = h * gain for codes
  auto take = [&](TV xv, TV rv, const Place &w, bool store) {
    FV h = __builtin_convertvector(xv, FV);
    if (res) h += __builtin_convertvector(rv, FV);
    if (store && sum) StoreFrom<VE>(sum + w.to, __builtin_convertvector(h, TV), w.skip, w.whole);
    if (NORM && !w.whole)                                        // (a repeated element changes no maximum; a residual that is
#pragma unroll                                                   //  updated in place may have changed under it, though)
      for (int j = 0; j < VE; j++) h[j] = j >= w.skip ? h[j] : 0.0f;
    if (NORM)
#pragma unroll
      for (int j = 0; j < VE; j++) ss += static_cast<double>(h[j]) * static_cast<double>(h[j]);
    if (I8) {
      if (NORM) h *= gains(w.to);
#pragma unroll
      for (int j = 0; j < VE; j++) most = max(most, __float_as_uint(h[j]) & 0x7fffffffu);
    }
    return h;
  };

  FV v[NV > 0 ? NV : 1];
  if constexpr (NV > 0) {
    TV xr[NV], rr[NV];                                           // all loads are under way before the first is waited for
    Slot s = {0, 0};
#pragma unroll
    for (int i = 0; i < NV; i++, s = next(s)) {
      const Place w = place(s.p, s.c);
      xr[i] = LoadAny<TV>(x + w.from);
      rr[i] = xr[i];
      if (res) rr[i] = LoadAny<TV>(res + w.to);
    }
    s = {0, 0};
#pragma unroll
    for (int i = 0; i < NV; i++, s = next(s)) v[i] = take(xr[i], rr[i], place(s.p, s.c), true);
  } else {
    for (int p = 0; p < parts; p++)
      for (int c = 0; c < per_part; c++) {
        const Place w = place(p, c);
        const TV xv = LoadAny<TV>(x + w.from);
        (void)take(xv, res ? LoadAny<TV>(res + w.to) : xv, w, false);
      }
  }

  // over the wave, then over the row's waves (the same order for every thread: one value)
  if (NORM) ss = WaveSum(ss);
  if (I8) most = WaveMax(most);
  if constexpr (NW > 1) {
    __shared__ double part_ss[NW];
    __shared__ uint32_t part_most[NW];
    if ((t & 63) == 0) { part_ss[t >> 6] = ss; part_most[t >> 6] = most; }
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      if (NORM) ss += part_ss[w];
      if (I8) most = max(most, part_most[w]);
    }
  }
  const double r = NORM ? 1.0 / sqrt(ss / a.part_dim + static_cast<double>(a.eps)) : 1.0;
  const float rf = static_cast<float>(r);
  // A row that holds an infinity or a NaN has no codes: zeros under a NaN scale.  Rows below 2^-100 are lifted first (an exact
  // product), so that 127 / a stays finite down to the smallest denormal.
  const bool bad = I8 && most >= 0x7f800000u;
  const float top = __uint_as_float(most), lift = top < 7.8886090522101181e-31f ? 1.2676506002282294e+30f : 1.0f;
  const float to_code = I8 && !bad && most != 0 ? 127.0f / (top * lift) : 0.0f;
  if (I8 && t == 0) a.out_scale[row] = bad ? __uint_as_float(0x7fc00000u) : static_cast<float>(static_cast<double>(top) * r / 127.0);

  const uint32_t keep = bad ? 0u : 0xffffffffu;
  auto give = [&](FV w, const Place &at) {
    OV o;
    if constexpr (I8) {
      w = w * lift * to_code;
      // 1.5 * 2^23 + v, rounded to the nearest even integer by the sum itself, has v's code in its lowest byte
      uint32_t code[VE];
#pragma unroll
      for (int j = 0; j < VE; j++) code[j] = __float_as_uint(w[j] + 12582912.0f) & keep;
      if constexpr (VE % 4 == 0) {
        uint32_t word[VE / 4];
#pragma unroll
        for (int j = 0; j < VE / 4; j++)
          word[j] = __builtin_amdgcn_perm(code[4 * j + 1], code[4 * j], 0x0c0c0400u) | __builtin_amdgcn_perm(code[4 * j + 3], code[4 * j + 2], 0x04000c0cu);
        __builtin_memcpy(&o, word, sizeof(o));
      } else {
#pragma unroll
        for (int j = 0; j < VE; j++) o[j] = static_cast<TO>(code[j] & 0xff);
      }
    } else {
      o = __builtin_convertvector(w * rf * gains(at.to), OV);
    }
    StoreFrom<VE>(out + at.to, o, at.skip, at.whole);
  };
  if constexpr (NV > 0) {
    Slot s = {0, 0};
#pragma unroll
    for (int i = 0; i < NV; i++, s = next(s)) give(v[i], place(s.p, s.c));
  } else {
    for (int p = 0; p < parts; p++)
      for (int c = 0; c < per_part; c++) {                       // (the sum is stored here, its parts being read for the last time)
        const Place w = place(p, c);
        const TV xv = LoadAny<TV>(x + w.from);
        give(take(xv, res ? LoadAny<TV>(res + w.to) : xv, w, true), w);
      }
  }
}

constexpr int kMaxDim = 1 << 30;
// At most this many workgroups per launch (rows beyond go to a launch of their own): a launch has fewer than 2^32 threads.
constexpr int64_t kMaxGroups = 1 << 21;
static_assert(kMaxGroups * 1024 < int64_t{1} << 32, "threads of a launch");

template <typename T, typename TO, bool NORM, int VE, int TPR, int NV>
static int LaunchRows(RowArgs a, hipStream_t st) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR;
  const int64_t rows = a.rows, most = kMaxGroups * RPB;
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    RowArgs b = a;
    b.rows = rows - r0 < most ? rows - r0 : most;
    b.x = static_cast<const T *>(a.x) + r0 * a.ld_x;
    if (a.residual) b.residual = static_cast<const T *>(a.residual) + r0 * a.ld_residual;
    if (a.sum) b.sum = static_cast<T *>(a.sum) + r0 * a.ld_sum;
    b.out = static_cast<TO *>(a.out) + r0 * a.ld_out;
    if (a.out_scale) b.out_scale = a.out_scale + r0;
    hipLaunchKernelGGL((RowKernel<T, TO, NORM, VE, TPR, NV>), dim3(CeilDiv(b.rows, RPB)), dim3(BLOCK), 0, st, b);
    KAMD_HIP(hipGetLastError());
  }
  return KAMD_OK;
}

// Threads per row and elements per thread: the pair that holds the row (piece by piece) with the least left over, for what is
// left over is loaded and computed for nothing; of equals, the first.  Waves of their own with 24 and more elements
// per lane count for 1.4 times their size.  Few rows are given the threads that shorten the way through one.  (us, MI355X)
//   norm 12000 x 1536 bf16  64 x 24  24.7   256 x 8 26.2   512 x 8  44         norm 16384 x 4096 bf16  512 x 8  92  256 x 16  95  64 x 64  108
//   norm 12000 x 1536 f32   64 x 24  28.2   256 x 8 26.4                       norm 16384 x 8192 bf16  1024 x 8 181  512 x 16 186  1024 x 16 250
//   codes of 40000 x (3 x 768) f32  64 x 40  43   256 x 16  64                 norm 1 x 1536 bf16  256 x 8  2.4   64 x 32  3.1
//   codes of 20000 x 4096 bf16  256 x 16  38.5   512 x 8  44.3  (the codes' kernels take the smaller workgroup of equals)
// Every piece of a splice is rounded up to a pass of the row's threads, which splices of many pieces pay for (us, and the time
// of their bytes):  40000 x (5 x 768) f32  80 (56),  bf16  474 (43);  40000 x (5 x 40) bf16  28 (2.3),  x (7 x 40)  624 (2.9).  From 7
// pieces of 16-bit rows on, from 5 on below 1024 rows or over 512 columns, no pair holds the row: 1024 threads read it twice.
// Norm to codes of 16385 .. 32768 f32 columns: 1024 threads x 32 elements spill 3 registers;  4096 x 32768  172 us (135).
template <typename T, typename TO, bool NORM>
static int RunRows(const RowArgs &a, hipStream_t st) {
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  constexpr bool I8 = sizeof(TO) == 1;
  static_assert(KAMD_MAX_OFFSETS <= 8, "pieces");
  if (a.part_dim < VE) return LaunchRows<T, TO, NORM, 1, 64, 8>(a, st);          // at most 7 columns, in at most 8 pieces
  typedef int (*Launch)(RowArgs, hipStream_t);
  struct Shape { int tpr, ept; Launch go; };
#define KAMD_SHAPE(TPR, EPT) {TPR, EPT, LaunchRows<T, TO, NORM, VE, TPR, (EPT) / VE>}
  static const Shape shapes[] = {KAMD_SHAPE(64, 8), KAMD_SHAPE(64, 16), KAMD_SHAPE(64, 24), KAMD_SHAPE(64, 32), KAMD_SHAPE(64, NORM ? 32 : 40),
                                 KAMD_SHAPE(64, NORM ? 32 : 48), KAMD_SHAPE(256, 8), KAMD_SHAPE(512, I8 ? 16 : 8), KAMD_SHAPE(256, 16), KAMD_SHAPE(256, 24),
                                 KAMD_SHAPE(1024, I8 ? 16 : 8), KAMD_SHAPE(512, 16), KAMD_SHAPE(512, 24), KAMD_SHAPE(1024, 16), KAMD_SHAPE(1024, 32)};
#undef KAMD_SHAPE
  const Shape *best = NULL;
  double least = 0.0;
  for (const Shape &s : shapes) {
    const int64_t need = static_cast<int64_t>(CeilDiv(a.part_dim, s.tpr * VE)) * VE * (NORM ? 1 : a.n_parts);
    if (need > s.ept || (a.rows < 1024 && s.tpr == 64 && s.ept > 16)) continue;
    const double size = static_cast<double>(s.tpr) * s.ept * (s.tpr == 64 && s.ept >= 24 ? 1.4 : 1.0);
    if (!best || size < least) { best = &s; least = size; }
  }
  return best ? best->go(a, st) : LaunchRows<T, TO, NORM, VE, 1024, 0>(a, st);
}

}  // namespace kamd
using kamd::SetError;

extern "C" {

int kamd_rms_norm_device(const void *d_x, int64_t ld_x, const void *d_residual, int64_t ld_residual, int type, const float *d_gain, float eps,
                         int64_t rows, int dim, void *d_sum, int64_t ld_sum, void *d_out, int64_t ld_out, int out_type, float *d_out_scale,
                         void *stream) {
  if (type != KAMD_F32 && type != KAMD_BF16 && type != KAMD_F16) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: unknown input type %d", type);
  if (out_type != type && out_type != KAMD_I8) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: the output has the input's type or 8 bits (type %d, output %d)", type, out_type);
  if (rows < 0 || dim <= 0 || dim > kamd::kMaxDim) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: bad sizes (%lld rows, dim %d)", static_cast<long long>(rows), dim);
  if (!(eps >= FLT_MIN) || !std::isfinite(eps)) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: eps must be a normal positive number, got %g", static_cast<double>(eps));
  if (ld_x < dim || ld_out < dim || (d_residual && ld_residual < dim) || (d_sum && ld_sum < dim))
    return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: leading dimension smaller than the matrix");
  if (rows == 0) return KAMD_OK;
  if (!d_x || !d_out) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: null argument");
  if (out_type == KAMD_I8 && !d_out_scale) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: 8-bit output needs d_out_scale");
  const int size = type == KAMD_F32 ? 4 : 2, out_size = out_type == KAMD_I8 ? 1 : size;
  const kamd::MemoryRows x = kamd::RowsOf(d_x, ld_x, dim, size, rows), residual = kamd::RowsOf(d_residual, ld_residual, dim, size, rows),
                         sum = kamd::RowsOf(d_sum, ld_sum, dim, size, rows), out = kamd::RowsOf(d_out, ld_out, dim, out_size, rows),
                         scale = kamd::RowsOf(out_type == KAMD_I8 ? d_out_scale : NULL, rows, rows, 4, 1), gain = kamd::RowsOf(d_gain, dim, dim, 4, 1);
  auto apart = [](const kamd::MemoryRows &a, const kamd::MemoryRows &b) { return kamd::SameRows(a, b) || !kamd::RowsMeet(a, b); };
  bool fine = apart(sum, x) && apart(sum, residual) && apart(out, x) && apart(out, residual) && apart(out, sum) && !RowsMeet(sum, gain) && !RowsMeet(out, gain);
  for (const kamd::MemoryRows &m : {x, residual, sum, out, gain}) fine = fine && !RowsMeet(scale, m);
  if (!fine) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: an output overlaps another argument (it may lie exactly on a matrix of its own type)");
  if (!kamd::RequireDevice()) return KAMD_ERR_HIP;
  kamd::RowArgs a = {};
  a.x = d_x; a.residual = d_residual; a.sum = d_sum; a.out = d_out; a.out_scale = out_type == KAMD_I8 ? d_out_scale : NULL; a.gain = d_gain;
  a.ld_x = ld_x; a.ld_residual = ld_residual; a.ld_sum = ld_sum; a.ld_out = ld_out;
  a.rows = rows; a.eps = eps; a.part_dim = dim; a.n_parts = 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool i8 = out_type == KAMD_I8;
  if (type == KAMD_F32) return i8 ? kamd::RunRows<float, int8_t, true>(a, st) : kamd::RunRows<float, float, true>(a, st);
  if (type == KAMD_BF16) return i8 ? kamd::RunRows<__bf16, int8_t, true>(a, st) : kamd::RunRows<__bf16, __bf16, true>(a, st);
  return i8 ? kamd::RunRows<_Float16, int8_t, true>(a, st) : kamd::RunRows<_Float16, _Float16, true>(a, st);
}

int kamd_quantize_rows_device(const void *d_x, int64_t ld_x, int type, int64_t in_rows, int dim, const int32_t *offsets, int n_offsets,
                              int8_t *d_q, int64_t ld_q, float *d_scale, void *stream) {
  if (type != KAMD_F32 && type != KAMD_BF16 && type != KAMD_F16) return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: unknown input type %d", type);
  if (in_rows < 0 || dim <= 0 || n_offsets < 1 || n_offsets > KAMD_MAX_OFFSETS || !offsets)
    return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: bad sizes (%lld rows, dim %d, %d offsets)", static_cast<long long>(in_rows), dim, n_offsets);
  if (static_cast<int64_t>(dim) * n_offsets > kamd::kMaxDim) return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: the spliced row is too long");
  int64_t lo = offsets[0], hi = offsets[0];
  for (int i = 1; i < n_offsets; i++) { lo = offsets[i] < lo ? offsets[i] : lo; hi = offsets[i] > hi ? offsets[i] : hi; }
  if (hi - lo > INT32_MAX) return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: offsets too far apart");
  if (ld_x < dim || ld_q < static_cast<int64_t>(dim) * n_offsets)
    return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: leading dimension smaller than the matrix");
  if (in_rows <= hi - lo) return KAMD_OK;                        // no row has all its context
  if (!d_x || !d_q || !d_scale) return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: null argument");
  const int64_t n = static_cast<int64_t>(dim) * n_offsets, rows = in_rows - (hi - lo);
  const kamd::MemoryRows x = kamd::RowsOf(d_x, ld_x, dim, type == KAMD_F32 ? 4 : 2, in_rows), q = kamd::RowsOf(d_q, ld_q, n, 1, rows),
                         scale = kamd::RowsOf(d_scale, rows, rows, 4, 1);
  if (RowsMeet(q, x) || RowsMeet(scale, x) || RowsMeet(scale, q)) return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: an output overlaps another argument");
  if (!kamd::RequireDevice()) return KAMD_ERR_HIP;
  kamd::RowArgs a = {};
  a.x = d_x; a.ld_x = ld_x; a.out = d_q; a.ld_out = ld_q; a.out_scale = d_scale;
  a.rows = rows; a.part_dim = dim; a.n_parts = n_offsets;
  for (int i = 0; i < n_offsets; i++) a.part_at[i] = (offsets[i] - lo) * ld_x;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (type == KAMD_F32) return kamd::RunRows<float, int8_t, false>(a, st);
  if (type == KAMD_BF16) return kamd::RunRows<__bf16, int8_t, false>(a, st);
  return kamd::RunRows<_Float16, int8_t, false>(a, st);
}

}  // extern "C"
