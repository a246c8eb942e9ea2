// Layer norm over the last axis, forward and backward, for gfx950 (MI355X).
//
//   forward   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), y = (x - m) r w + b
//   backward  h = (x - m) r, g = dy w:   dx = r (g - mean(g) - h mean(g h)),   dw = sum_rows dy h,   db = sum_rows dy
//
// Both are bound by HBM: every row is read once into registers, the mean and the variance are taken from there in two passes (the
// variance from centred values: no cancellation), and written once.  All sums are fp32; the only rounding to fewer bits is the
// store.  Small rows share a wave (lanes = a power of two that covers the row in K pieces per lane, reductions by shuffles); long
// ones take a workgroup (reductions through LDS).  The weight's and the bias's gradients are kept per lane in registers over
// all rows a workgroup walks, written as one partial row per workgroup and added up by a second launch in a fixed order
// (no atomics: the result does not depend on scheduling).
//
// Forward 262144 x 1024 bf16: 219 us, 4.9 TB/s (a large streaming copy reaches 6.4, torch's copy 5.4; without the next row in flight 268 us); 65536 x 211 fp32: 21 us;
// one row: 2 us, a launch's latency (4 with the parameters read element by element).  Forward + backward 65536 x 512 bf16: 29 + 35 us,
// and 4 for the partial rows' sum.
#include "oige_elem.hpp"

namespace oige {

constexpr int LN_THREADS = 256;
constexpr int LN_MAX_THREADS = 1024;
constexpr int LN_MAX_WIDTH = 16384;
constexpr int LN_LDS_COLS = 1024;  // most columns of a row in one wave: 64 lanes x 16 elements

// x + x of another lane, the lane found by the data path itself (no LDS round trip).
template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
// Sum over `lanes` (a power of two) neighbours, in all of them: pairs and fours by permutation, then mirrored halves of 8 and 16
// (their lanes hold equal sums by then), then two exchanges across 16 and 32 lanes.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  if (lanes > 1) v = add_dpp<0xB1>(v);    // quad_perm 1 0 3 2
  if (lanes > 2) v = add_dpp<0x4E>(v);    // quad_perm 2 3 0 1
  if (lanes > 4) v = add_dpp<0x141>(v);   // row_half_mirror
  if (lanes > 8) v = add_dpp<0x140>(v);   // row_mirror
  if (lanes > 16) v += __shfl_xor(v, 16, WAVE);
  if (lanes > 32) v += __shfl_xor(v, 32, WAVE);
  return v;
}

// Sum over the lanes that share a row: `lanes` neighbours of a wave, or the workgroup.
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, int lanes, float* lds) {
  v = lanes_sum(v, BLOCK ? WAVE : lanes);
  if (BLOCK) {
    const int w = threadIdx.x >> 6, waves = blockDim.x >> 6;
    __syncthreads();  // the last sum's readers are done
    if (lane_id() == 0) lds[w] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < waves; ++i) v += lds[i];
  }
  return v;
}

template <bool BLOCK>
__device__ __forceinline__ float2 row_sum2(float2 v, int lanes, float* lds) {
  v.x = lanes_sum(v.x, BLOCK ? WAVE : lanes);
  v.y = lanes_sum(v.y, BLOCK ? WAVE : lanes);
  if (BLOCK) {
    const int w = threadIdx.x >> 6, waves = blockDim.x >> 6;
    __syncthreads();
    if (lane_id() == 0) {
      lds[2 * w] = v.x;
      lds[2 * w + 1] = v.y;
    }
    __syncthreads();
    v = make_float2(0.f, 0.f);
    for (int i = 0; i < waves; ++i) {
      v.x += lds[2 * i];
      v.y += lds[2 * i + 1];
    }
  }
  return v;
}

// Whether element e of the run from `off` counts: rows are read by accesses of VEC elements on any boundary, a run across the end starts
// earlier and holds some elements a second time.  Those are computed and stored twice, to the same bits, and left out of the sums.
template <int VEC, int MODE>
__device__ __forceinline__ bool ln_once(int off, int e, int width) {
  return MODE == ELEMS_LOOSE ? run_start<VEC, MODE>(off, width) + e >= off : off + e < width;
}

// A run of the weight or the bias: of the rows' type or fp32, `none` everywhere where there is none.
template <typename T, int VEC, int MODE>
__device__ __forceinline__ void ln_param(float (&w)[VEC], const void* p, int dtype, int off, int width, float none) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = none;
  } else if (dtype == OIGE_F32) {
    load_run<float, VEC, MODE>(w, static_cast<const float*>(p), off, width);
  } else {
    load_run<T, VEC, MODE>(w, static_cast<const T*>(p), off, width);
  }
}

template <typename T, int VEC, int K, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? LN_MAX_THREADS : LN_THREADS) void layer_norm_forward_kernel(const oige_layer_norm_io a, int lanes) {
  constexpr int MODE = VEC == 1 ? ELEMS_SINGLE : ELEMS_LOOSE;
  __shared__ float lds[2 * LN_MAX_THREADS / WAVE];
  const int l = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & (lanes - 1));
  const int rows_per_block = BLOCK ? 1 : LN_THREADS / lanes;
  const int sub = BLOCK ? 0 : (int)threadIdx.x / lanes;
  const int width = a.width;
  const float inv = 1.f / (float)width;
  float w[K][VEC], b[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    ln_param<T, VEC, MODE>(w[k], a.weight, a.weight_dtype, (k * lanes + l) * VEC, width, 1.f);
    ln_param<T, VEC, MODE>(b[k], a.bias, a.weight_dtype, (k * lanes + l) * VEC, width, 0.f);
  }
  const auto once = [&](int k, int e) { return ln_once<VEC, MODE>((k * lanes + l) * VEC, e, width); };
  // the next row is on its way while this one is summed
  const int64_t first = (int64_t)blockIdx.x * rows_per_block + sub, step = (int64_t)gridDim.x * rows_per_block;
  Run<T, VEC, MODE> run[K];
  if (first < a.rows) {
#pragma unroll
    for (int k = 0; k < K; ++k) run[k].issue(static_cast<const T*>(a.x) + first * a.x_row_stride, (k * lanes + l) * VEC, width);
  }
  for (int64_t row = first; row < a.rows; row += step) {
    float x[K][VEC];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) run[k].take(x[k], (k * lanes + l) * VEC, width);
    const T* next = static_cast<const T*>(a.x) + (row + step < a.rows ? row + step : row) * a.x_row_stride;
#pragma unroll
    for (int k = 0; k < K; ++k) run[k].issue(next, (k * lanes + l) * VEC, width);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += once(k, e) ? x[k][e] : 0.f;
    const float mean = row_sum<BLOCK>(s, lanes, lds) * inv;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        x[k][e] -= mean;
        q = once(k, e) ? fmaf(x[k][e], x[k][e], q) : q;
      }
    const float rstd = 1.f / sqrtf(row_sum<BLOCK>(q, lanes, lds) * inv + a.eps);
    T* yr = static_cast<T*>(a.y) + row * (int64_t)width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = fmaf(x[k][e] * rstd, w[k][e], b[k][e]);
      store_run<T, VEC, MODE>(y, yr, (k * lanes + l) * VEC, width);
    }
    if (a.mean && l == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T, int VEC, int K, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? LN_MAX_THREADS : LN_THREADS) void layer_norm_backward_kernel(const oige_layer_norm_io a, int lanes) {
  constexpr int MODE = VEC == 1 ? ELEMS_SINGLE : ELEMS_LOOSE;
  __shared__ float lds[2 * LN_MAX_THREADS / WAVE];
  __shared__ float cols[BLOCK ? 1 : LN_THREADS / WAVE * LN_LDS_COLS];
  const int l = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & (lanes - 1));
  const int rows_per_block = BLOCK ? 1 : LN_THREADS / lanes;
  const int sub = BLOCK ? 0 : (int)threadIdx.x / lanes;
  const int width = a.width;
  const float inv = 1.f / (float)width;
  float w[K][VEC], dw[K][VEC], db[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    ln_param<T, VEC, MODE>(w[k], a.weight, a.weight_dtype, (k * lanes + l) * VEC, width, 1.f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[k][e] = db[k][e] = 0.f;
  }
  const auto once = [&](int k, int e) { return ln_once<VEC, MODE>((k * lanes + l) * VEC, e, width); };
  const int64_t first = (int64_t)blockIdx.x * rows_per_block + sub, step = (int64_t)gridDim.x * rows_per_block;
  Run<T, VEC, MODE> x_run[K], g_run[K];
  float next_mean = 0.f, next_rstd = 0.f;
  const auto issue = [&](int64_t row) {  // one row ahead, as above
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x_run[k].issue(static_cast<const T*>(a.x) + row * a.x_row_stride, (k * lanes + l) * VEC, width);
      g_run[k].issue(static_cast<const T*>(a.dy) + row * a.dy_row_stride, (k * lanes + l) * VEC, width);
    }
    next_mean = a.mean[row];
    next_rstd = a.rstd[row];
  };
  if (first < a.rows) issue(first);
  for (int64_t row = first; row < a.rows; row += step) {
    float x[K][VEC], g[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x_run[k].take(x[k], (k * lanes + l) * VEC, width);
      g_run[k].take(g[k], (k * lanes + l) * VEC, width);
    }
    const float mean = next_mean, rstd = next_rstd;
    issue(row + step < a.rows ? row + step : row);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        x[k][e] = (x[k][e] - mean) * rstd;
        dw[k][e] = fmaf(g[k][e], x[k][e], dw[k][e]);
        db[k][e] += g[k][e];
        g[k][e] *= w[k][e];
        s.x = once(k, e) ? s.x + g[k][e] : s.x;
        s.y = once(k, e) ? fmaf(g[k][e], x[k][e], s.y) : s.y;
      }
    s = row_sum2<BLOCK>(s, lanes, lds);
    const float mg = s.x * inv, mgx = s.y * inv;
    if (a.dx) {
      T* dxr = static_cast<T*>(a.dx) + row * (int64_t)width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float d[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[e] = rstd * (g[k][e] - fmaf(x[k][e], mgx, mg));
        store_run<T, VEC, MODE>(d, dxr, (k * lanes + l) * VEC, width);
      }
    }
  }
  if (!a.workspace) return;
  float* part = a.workspace + (int64_t)blockIdx.x * 2 * width;
  if (BLOCK) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int col = run_start<VEC, MODE>((k * lanes + l) * VEC, width) + e;
        if (col < width) {
          part[col] = dw[k][e];
          part[width + col] = db[k][e];
        }
      }
    return;
  }
  const int wv = threadIdx.x >> 6;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();  // the last table's readers are done
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float v = which ? db[k][e] : dw[k][e];
        for (int off = lanes; off < WAVE; off <<= 1) v += __shfl_xor(v, off, WAVE);  // the rows that shared this wave
        const int col = run_start<VEC, MODE>((k * lanes + l) * VEC, width) + e;
        if (col < width && lane_id() < lanes) cols[wv * LN_LDS_COLS + col] = v;
      }
    __syncthreads();
    for (int col = threadIdx.x; col < width; col += LN_THREADS) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < LN_THREADS / WAVE; ++i) v += cols[i * LN_LDS_COLS + col];
      part[which * width + col] = v;
    }
  }
}

// dweight / dbias = the column sums of the partial rows: 32 columns x 32 row slices per workgroup, every slice's rows and then
// the slices in a fixed order.
constexpr int LN_FOLD = 32;
__global__ __launch_bounds__(LN_FOLD * LN_FOLD) void layer_norm_fold_kernel(const oige_layer_norm_io a, int parts) {
  __shared__ float lds[LN_FOLD][LN_FOLD + 1];
  const int c = threadIdx.x % LN_FOLD, s = threadIdx.x / LN_FOLD;
  const int64_t col = (int64_t)blockIdx.x * LN_FOLD + c, cols = 2 * (int64_t)a.width;
  float v = 0.f;
  if (col < cols) {
    constexpr int U = 8;  // partial rows in flight
    for (int i0 = s; i0 < parts; i0 += U * LN_FOLD) {
      float p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * LN_FOLD;
        p[u] = a.workspace[(i < parts ? i : s) * cols + col];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) v += i0 + u * LN_FOLD < parts ? p[u] : 0.f;
    }
  }
  lds[s][c] = v;
  __syncthreads();
  if (s == 0 && col < cols) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < LN_FOLD; ++i) v += lds[i][c];
    void* out = col < a.width ? a.dweight : a.dbias;
    if (out) store_elem(out, col < a.width ? col : col - a.width, v, a.weight_dtype);
  }
}

// How a row is laid over lanes: `vec` elements per access (16 bytes, on any boundary), K accesses per lane,
// `lanes` of a wave -- or of a workgroup of 256 to 1024, where 64 lanes would hold more than 16 elements each (16384 x 2048 bf16: 44 us forward with 32 in a wave's lanes, 33 in a workgroup's).  A workgroup's lanes hold at most 16 of them, in the backward
// pass, which keeps five such rows, 8 (8192 x 8192 fp32: 347 us with 16, 173 with 8), as long as 1024 lanes are enough.
struct LnShape {
  int lanes, k;
  bool block;
};
static LnShape layer_norm_shape(int width, int vec, bool backward) {
  const int slots = (width + vec - 1) / vec;
  const int kmax = vec == 8 ? 2 : 4;
  LnShape s{1, 1, false};
  if (slots <= WAVE * kmax) {
    while (s.lanes < slots && s.lanes < WAVE) s.lanes *= 2;
    while (s.lanes * s.k < slots) s.k *= 2;
    return s;
  }
  s.block = true;
  s.lanes = LN_THREADS;
  const int each = (backward ? 8 : 16) / vec;
  while (s.lanes < LN_MAX_THREADS && s.lanes * each < slots) s.lanes *= 2;
  while (s.lanes * s.k < slots) s.k *= 2;
  return s;
}

// Workgroups walk rows, so that weights stay in registers and the next row is on its way behind this one's sums.  Forward: 4 per CU
// (262144 x 1024 bf16: 219 us; when it took 225, 238 with 8 per CU and 635 with a workgroup for every 4 rows).  Backward: 4 per CU, one partial row of
// the parameters' gradients each (65536 x 512 bf16: 35 us; when it took 37, 40 with 2 and 43 with 8).
constexpr int64_t LN_MAX_BLOCKS = 1024, LN_MAX_PARTS = 1024;

static int64_t layer_norm_blocks(int64_t rows, const LnShape& s, int64_t most) {
  const int64_t per = s.block ? 1 : LN_THREADS / s.lanes;
  const int64_t b = (rows + per - 1) / per;
  return b < most ? b : most;
}

template <typename T, int VEC, int K, bool BLOCK, bool BACKWARD>
static int layer_norm_launch(const oige_layer_norm_io& io, const LnShape& s, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks), threads(BLOCK ? s.lanes : LN_THREADS);
  if (BACKWARD) hipLaunchKernelGGL((layer_norm_backward_kernel<T, VEC, K, BLOCK>), grid, threads, 0, stream, io, s.lanes);
  else hipLaunchKernelGGL((layer_norm_forward_kernel<T, VEC, K, BLOCK>), grid, threads, 0, stream, io, s.lanes);
  return check_launch(BACKWARD ? "layer_norm_backward_kernel" : "layer_norm_forward_kernel");
}

template <typename T, int VEC, bool BACKWARD>
static int layer_norm_pick(const oige_layer_norm_io& io, const LnShape& s, int64_t blocks, hipStream_t stream) {
#define LN_CASE(K, BLOCK, OFFERED) \
  if constexpr (OFFERED) {           \
    if (s.k == K && s.block == BLOCK) return layer_norm_launch<T, VEC, K, BLOCK, BACKWARD>(io, s, blocks, stream); \
  }
  LN_CASE(1, false, true)
  LN_CASE(2, false, VEC > 1)
  LN_CASE(4, false, VEC == 4)
  LN_CASE(1, true, VEC > 1)
  LN_CASE(2, true, VEC > 1)
  LN_CASE(4, true, VEC == 4)
#undef LN_CASE
  return fail(OIGE_EINVAL, "layer_norm: no variant for %d lanes x %d accesses", s.lanes, s.k);
}

static int layer_norm_check(const oige_layer_norm_io* io, const char* what) {
  OIGE_REQUIRE(io != nullptr, "%s: null io", what);
  OIGE_REQUIRE(elem_bytes(io->dtype) && elem_bytes(io->weight_dtype), "%s: dtype must be OIGE_F32, OIGE_F16 or OIGE_BF16", what);
  OIGE_REQUIRE(io->weight_dtype == io->dtype || io->weight_dtype == OIGE_F32, "%s: weight and bias have the activations' type or fp32", what);
  OIGE_REQUIRE(io->rows >= 0 && io->width >= 1 && io->width <= LN_MAX_WIDTH, "%s: rows %lld, width %d (1 .. %d)", what,
               (long long)io->rows, io->width, LN_MAX_WIDTH);
  OIGE_REQUIRE(io->rows == 0 || io->x, "%s: null x", what);
  OIGE_REQUIRE(io->eps >= 0.f, "%s: eps must not be negative", what);
  return OIGE_OK;
}

// Elements of an access: 16 bytes, single ones in rows that are shorter.
static int layer_norm_vec(const oige_layer_norm_io& io) {
  const int v = 16 / elem_bytes(io.dtype);
  return io.width >= v ? v : 1;
}

template <bool BACKWARD>
static int layer_norm_dispatch(const oige_layer_norm_io& io, const LnShape& s, int64_t blocks, hipStream_t stream) {
  const bool wide = layer_norm_vec(io) > 1;
  if (io.dtype == OIGE_F32)
    return wide ? layer_norm_pick<float, 4, BACKWARD>(io, s, blocks, stream) : layer_norm_pick<float, 1, BACKWARD>(io, s, blocks, stream);
  if (io.dtype == OIGE_F16)
    return wide ? layer_norm_pick<_Float16, 8, BACKWARD>(io, s, blocks, stream) : layer_norm_pick<_Float16, 1, BACKWARD>(io, s, blocks, stream);
  return wide ? layer_norm_pick<__bf16, 8, BACKWARD>(io, s, blocks, stream) : layer_norm_pick<__bf16, 1, BACKWARD>(io, s, blocks, stream);
}

}  // namespace oige

using namespace oige;

extern "C" {

int oige_layer_norm_forward(const oige_layer_norm_io* io, oige_stream_t stream) {
  const int rc = layer_norm_check(io, "layer_norm_forward");
  if (rc) return rc;
  if (io->rows == 0) return OIGE_OK;
  OIGE_REQUIRE(io->y, "layer_norm_forward: null y");
  OIGE_REQUIRE((io->mean == nullptr) == (io->rstd == nullptr), "layer_norm_forward: mean and rstd are kept together or not at all");
  const LnShape s = layer_norm_shape(io->width, layer_norm_vec(*io), false);
  return layer_norm_dispatch<false>(*io, s, layer_norm_blocks(io->rows, s, LN_MAX_BLOCKS), (hipStream_t)stream);
}

int64_t oige_layer_norm_workspace_floats(int64_t rows, int32_t width) {
  if (rows < 1 || width < 1 || width > LN_MAX_WIDTH)
    return fail(OIGE_EINVAL, "layer_norm_workspace: rows %lld, width %d (1 .. %d)", (long long)rows, width, LN_MAX_WIDTH);
  return (rows < LN_MAX_PARTS ? rows : LN_MAX_PARTS) * 2 * (int64_t)width;
}

int oige_layer_norm_backward(const oige_layer_norm_io* io, oige_stream_t stream) {
  const int rc = layer_norm_check(io, "layer_norm_backward");
  if (rc) return rc;
  const bool params = io->dweight || io->dbias;
  if (io->rows == 0 && !params) return OIGE_OK;  // (no rows have no dx: its pointer may be NULL)
  OIGE_REQUIRE(io->rows == 0 || (io->dy && io->mean && io->rstd), "layer_norm_backward: null dy, mean or rstd");
  OIGE_REQUIRE(io->dx || params, "layer_norm_backward: no gradient asked for");
  OIGE_REQUIRE(!params || io->rows == 0 || io->workspace, "layer_norm_backward: the weight's gradient needs a workspace");
  OIGE_REQUIRE(!params || io->rows == 0 || io->workspace_floats >= oige_layer_norm_workspace_floats(io->rows, io->width),
               "layer_norm_backward: workspace of %lld floats is too small", (long long)io->workspace_floats);
  oige_layer_norm_io a = *io;
  if (!params) a.workspace = nullptr;
  int64_t blocks = 0;
  if (a.rows > 0) {
    const LnShape s = layer_norm_shape(a.width, layer_norm_vec(a), true);
    blocks = layer_norm_blocks(a.rows, s, LN_MAX_PARTS);
    const int rc2 = layer_norm_dispatch<true>(a, s, blocks, (hipStream_t)stream);
    if (rc2) return rc2;
  }
  if (!params) return OIGE_OK;
  hipLaunchKernelGGL(layer_norm_fold_kernel, dim3((unsigned)((2 * (int64_t)a.width + LN_FOLD - 1) / LN_FOLD)), dim3(LN_FOLD * LN_FOLD), 0,
                     (hipStream_t)stream, a, (int)blocks);  // no rows: zeroes
  return check_launch("layer_norm_fold_kernel");
}

}  // extern "C"
