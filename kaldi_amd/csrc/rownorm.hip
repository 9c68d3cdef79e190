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
// What bounds it: the bytes.  Each row is read once and stays in registers (up to 32 elements per thread) between the
// reduction and the output; only rows longer than 32768 elements are read twice.
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
  int dim;                        // columns of the output row = n_parts * part_dim
  int part_dim;                   // columns of x
  int part_shift[KAMD_MAX_OFFSETS];   // part p of output row r comes from row r + part_shift[p] of x
};

// The widest access is used whatever the address: rows of odd length start anywhere, and MI355X's global loads and stores
// need no more than the element's own alignment.
template <typename V, typename T>
__device__ inline V LoadAny(const T *p) { V v; __builtin_memcpy(&v, p, sizeof(V)); return v; }
template <typename V, typename T>
__device__ inline void StoreAny(T *p, V v) { __builtin_memcpy(p, &v, sizeof(V)); }

template <typename TO> __device__ inline TO RoundTo(float v) { return static_cast<TO>(v); }

// T: the input's type; TO: the output's (T or int8_t); NORM: false = coding alone; TPR: threads per row; EPT: elements per
// thread held in registers, 0 = none (the row is read twice).
template <typename T, typename TO, bool NORM, int TPR, int EPT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void RowKernel(RowArgs a) {
  constexpr bool I8 = sizeof(TO) == 1;
  constexpr int VE = 16 / static_cast<int>(sizeof(T));          // elements of one 16-byte access
  constexpr int BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR, NW = TPR / 64;
  typedef T TV __attribute__((ext_vector_type(VE)));
  typedef TO OV __attribute__((ext_vector_type(VE)));
  const int t = RPB == 1 ? threadIdx.x : threadIdx.x & (TPR - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + (RPB == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR));
  if (row >= a.rows) return;                                     // (a whole wave; a whole workgroup where there is a barrier)
  const T *x = static_cast<const T *>(a.x) + row * a.ld_x;
  const T *res = NORM && a.residual ? static_cast<const T *>(a.residual) + row * a.ld_residual : NULL;
  T *sum = NORM && a.sum ? static_cast<T *>(a.sum) + row * a.ld_sum : NULL;
  TO *out = static_cast<TO *>(a.out) + row * a.ld_out;
  const int dim = a.dim;

  auto source = [&](int k) -> const T * {                        // element k of the row (k < dim)
    if constexpr (NORM) return x + k;
    const int p = k / a.part_dim;
    return x + a.part_shift[p] * a.ld_x + (k - p * a.part_dim);
  };
  // VE elements from k on, zeros from `dim` on: h of the norm, or the spliced row
  auto load_raw = [&](int k, TV *xv, TV *rv) {
    TV xz = {}, rz = {};
    *xv = xz; *rv = rz;
    const bool whole = NORM || k % a.part_dim + VE <= a.part_dim;         // does not straddle two parts
    if (k + VE <= dim && whole) {
      *xv = LoadAny<TV>(source(k));
      if (res) *rv = LoadAny<TV>(res + k);
    } else {
#pragma unroll
      for (int j = 0; j < VE; j++)
        if (k + j < dim) {
          (*xv)[j] = *source(k + j);
          if (res) (*rv)[j] = res[k + j];
        }
    }
  };
  auto store_sum = [&](int k, const float *h) {
    if (k + VE <= dim) {
      TV v;
#pragma unroll
      for (int j = 0; j < VE; j++) v[j] = RoundTo<T>(h[j]);
      StoreAny(sum + k, v);
    } else {
      for (int j = 0; j < VE; j++)
        if (k + j < dim) sum[k + j] = RoundTo<T>(h[j]);
    }
  };
  auto gains = [&](int k, float *g) {
#pragma unroll
    for (int j = 0; j < VE; j++) g[j] = 1.0f;
    if (!NORM || !a.gain) return;
    if (k + VE <= dim) {
      typedef float GV __attribute__((ext_vector_type(VE)));
      const GV v = LoadAny<GV>(a.gain + k);
#pragma unroll
      for (int j = 0; j < VE; j++) g[j] = v[j];
    } else {
      for (int j = 0; j < VE; j++)
        if (k + j < dim) g[j] = a.gain[k + j];
    }
  };

  double ss = 0.0;
  uint32_t most = 0;                                             // bits of max |t|: ordered like the values, NaN on top
  auto take = [&](const float *h, float *v, const float *g) {    // into the row's statistics; v = what the output is made of
#pragma unroll
    for (int j = 0; j < VE; j++) {
      if (NORM) ss += static_cast<double>(h[j]) * static_cast<double>(h[j]);
      v[j] = NORM && I8 ? h[j] * g[j] : h[j];
      if (I8) { const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu; most = b > most ? b : most; }
    }
  };

  constexpr int NV = EPT / VE;
  float v[NV > 0 ? NV : 1][VE];
  if constexpr (EPT > 0) {
    TV xr[NV], rr[NV];
#pragma unroll
    for (int c = 0; c < NV; c++)
      if (c * TPR * VE < dim) load_raw((c * TPR + t) * VE, &xr[c], &rr[c]);
#pragma unroll
    for (int c = 0; c < NV; c++) {
      const int k = (c * TPR + t) * VE;
      if (c * TPR * VE < dim) {
        float h[VE], g[VE];
#pragma unroll
        for (int j = 0; j < VE; j++) h[j] = res ? static_cast<float>(xr[c][j]) + static_cast<float>(rr[c][j]) : static_cast<float>(xr[c][j]);
        if (sum) store_sum(k, h);
        if (I8) gains(k, g);
        take(h, v[c], g);
      }
    }
  } else {
    for (int k = t * VE; k < dim; k += TPR * VE) {
      TV xr, rr;
      load_raw(k, &xr, &rr);
      float h[VE], g[VE];
#pragma unroll
      for (int j = 0; j < VE; j++) h[j] = res ? static_cast<float>(xr[j]) + static_cast<float>(rr[j]) : static_cast<float>(xr[j]);
      if (I8) gains(k, g);
      take(h, v[0], g);
    }
  }

  // over the wave, then over the row's waves (the same order for every thread: one value)
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) {
    if (NORM) ss += __shfl_xor(ss, s);
    if (I8) { const uint32_t o = __shfl_xor(most, s); most = o > most ? o : most; }
  }
  if constexpr (NW > 1) {
    __shared__ double part_ss[NW];
    __shared__ uint32_t part_most[NW];
    if ((t & 63) == 0) { part_ss[t >> 6] = ss; part_most[t >> 6] = most; }
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      if (NORM) ss += part_ss[w];
      if (I8) most = part_most[w] > most ? part_most[w] : most;
    }
  }
  const double r = NORM ? 1.0 / sqrt(ss / dim + static_cast<double>(a.eps)) : 1.0;
  const float rf = static_cast<float>(r);
  // A row that holds an infinity or a NaN has no codes: zeros under a NaN scale.  Rows below 2^-100 are lifted first (an exact
  // product), so that 127 / a stays finite down to the smallest denormal.
  const bool bad = I8 && most >= 0x7f800000u;
  const float top = __uint_as_float(most), lift = top < 7.8886090522101181e-31f ? 1.2676506002282294e+30f : 1.0f;
  const float to_code = I8 && !bad && most != 0 ? 127.0f / (top * lift) : 0.0f;
  if (I8 && t == 0) a.out_scale[row] = bad ? __uint_as_float(0x7fc00000u) : static_cast<float>(static_cast<double>(top) * r / 127.0);

  auto give = [&](int k, const float *w) {
    float g[VE];
    if (!I8) gains(k, g);
    OV o;
#pragma unroll
    for (int j = 0; j < VE; j++) {
      if constexpr (I8) o[j] = static_cast<TO>(bad ? 0 : static_cast<int>(rintf(w[j] * lift * to_code)));
      else o[j] = RoundTo<TO>(w[j] * rf * g[j]);
    }
    if (k + VE <= dim) StoreAny(out + k, o);
    else
#pragma unroll
      for (int j = 0; j < VE; j++)
        if (k + j < dim) out[k + j] = o[j];
  };
  if constexpr (EPT > 0) {
#pragma unroll
    for (int c = 0; c < NV; c++)
      if (c * TPR * VE < dim) {
        const int k = (c * TPR + t) * VE;
        if (k < dim) give(k, v[c]);
      }
  } else {
    for (int k = t * VE; k < dim; k += TPR * VE) {               // (the sum is stored here, after its parts have been read for the last time)
      TV xr, rr;
      load_raw(k, &xr, &rr);
      float h[VE], g[VE];
#pragma unroll
      for (int j = 0; j < VE; j++) h[j] = res ? static_cast<float>(xr[j]) + static_cast<float>(rr[j]) : static_cast<float>(xr[j]);
      if (sum) store_sum(k, h);
      if (NORM && I8) {
        gains(k, g);
#pragma unroll
        for (int j = 0; j < VE; j++) h[j] *= g[j];
      }
      give(k, h);
    }
  }
}

// At most this many workgroups per launch (rows beyond go to a launch of their own).
constexpr int64_t kMaxGroups = 1 << 22;

template <typename T, typename TO, bool NORM, int TPR, int EPT>
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
    hipLaunchKernelGGL((RowKernel<T, TO, NORM, TPR, EPT>), dim3(CeilDiv(b.rows, RPB)), dim3(BLOCK), 0, st, b);
    KAMD_HIP(hipGetLastError());
  }
  return KAMD_OK;
}

// A wave per row while the row fits into 32 elements per lane, then a workgroup of 256, then of 1024.
template <typename T, typename TO, bool NORM>
static int RunRows(const RowArgs &a, hipStream_t st) {
  if (a.dim <= 64 * 8) return LaunchRows<T, TO, NORM, 64, 8>(a, st);
  if (a.dim <= 64 * 16) return LaunchRows<T, TO, NORM, 64, 16>(a, st);
  if (a.dim <= 64 * 32) return LaunchRows<T, TO, NORM, 64, 32>(a, st);
  if (a.dim <= 256 * 16) return LaunchRows<T, TO, NORM, 256, 16>(a, st);
  if (a.dim <= 256 * 32) return LaunchRows<T, TO, NORM, 256, 32>(a, st);
  if (a.dim <= 1024 * 16) return LaunchRows<T, TO, NORM, 1024, 16>(a, st);
  if (a.dim <= 1024 * 32) return LaunchRows<T, TO, NORM, 1024, 32>(a, st);
  return LaunchRows<T, TO, NORM, 1024, 0>(a, st);
}

}  // namespace kamd
using kamd::SetError;

extern "C" {

int kamd_rms_norm_device(const void *d_x, int64_t ld_x, const void *d_residual, int64_t ld_residual, int type, const float *d_gain, float eps,
                         int64_t rows, int dim, void *d_sum, int64_t ld_sum, void *d_out, int64_t ld_out, int out_type, float *d_out_scale,
                         void *stream) {
  if (type != KAMD_F32 && type != KAMD_BF16 && type != KAMD_F16) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: unknown input type %d", type);
  if (out_type != type && out_type != KAMD_I8) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: the output has the input's type or 8 bits (type %d, output %d)", type, out_type);
  if (rows < 0 || dim <= 0) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: bad sizes (%lld rows, dim %d)", static_cast<long long>(rows), dim);
  if (!(eps >= FLT_MIN) || !std::isfinite(eps)) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: eps must be a normal positive number, got %g", static_cast<double>(eps));
  if (ld_x < dim || ld_out < dim || (d_residual && ld_residual < dim) || (d_sum && ld_sum < dim))
    return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: leading dimension smaller than the matrix");
  if (rows == 0) return KAMD_OK;
  if (!d_x || !d_out) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: null argument");
  if (out_type == KAMD_I8 && !d_out_scale) return SetError(KAMD_ERR_ARG, "kamd_rms_norm_device: 8-bit output needs d_out_scale");
  if (!kamd::RequireDevice()) return KAMD_ERR_HIP;
  kamd::RowArgs a = {};
  a.x = d_x; a.residual = d_residual; a.sum = d_sum; a.out = d_out; a.out_scale = out_type == KAMD_I8 ? d_out_scale : NULL; a.gain = d_gain;
  a.ld_x = ld_x; a.ld_residual = ld_residual; a.ld_sum = ld_sum; a.ld_out = ld_out;
  a.rows = rows; a.eps = eps; a.dim = dim; a.part_dim = dim;
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
  if (static_cast<int64_t>(dim) * n_offsets > INT32_MAX) return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: the spliced row is too long");
  int64_t lo = offsets[0], hi = offsets[0];
  for (int i = 1; i < n_offsets; i++) { lo = offsets[i] < lo ? offsets[i] : lo; hi = offsets[i] > hi ? offsets[i] : hi; }
  if (hi - lo > INT32_MAX) return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: offsets too far apart");
  if (ld_x < dim || ld_q < static_cast<int64_t>(dim) * n_offsets)
    return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: leading dimension smaller than the matrix");
  if (in_rows <= hi - lo) return KAMD_OK;                        // no row has all its context
  if (!d_x || !d_q || !d_scale) return SetError(KAMD_ERR_ARG, "kamd_quantize_rows_device: null argument");
  if (!kamd::RequireDevice()) return KAMD_ERR_HIP;
  kamd::RowArgs a = {};
  a.x = d_x; a.ld_x = ld_x; a.out = d_q; a.ld_out = ld_q; a.out_scale = d_scale;
  a.rows = in_rows - (hi - lo); a.dim = dim * n_offsets; a.part_dim = dim;
  for (int i = 0; i < n_offsets; i++) a.part_shift[i] = static_cast<int>(offsets[i] - lo);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (type == KAMD_F32) return kamd::RunRows<float, int8_t, false>(a, st);
  if (type == KAMD_BF16) return kamd::RunRows<__bf16, int8_t, false>(a, st);
  return kamd::RunRows<_Float16, int8_t, false>(a, st);
}

}  // extern "C"
