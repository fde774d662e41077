// The matrix product with bias, activation and residual, and its gradients:
//
//   z = lhs * rhs + bias,  out = residual + scale * act(z)
//   dz = scale * dy * act'(z),  d_lhs = dz * rhs^T (times act_in'(z_in)),  d_rhs = lhs^T * dz,  d_bias = sum of dz's rows
//
// General form, in two steps: the product in fp32, in scratch, and one pass over it for the rest.
#include "activation.cuh"
#include "column_sums.cuh"
#include "tc_gemm.cuh"

#include <algorithm>
#include <cstring>

namespace pdnn {
namespace {

// Scratch from the stream-ordered allocator, released when it goes out of scope.
struct Scratch {
  void* p = nullptr;
  cudaStream_t s;
  explicit Scratch(cudaStream_t stream) : s(stream) {}
  Scratch(const Scratch&) = delete;
  bool get(size_t bytes) {
    if (bytes == 0) return true;
    if (cudaMallocAsync(&p, bytes, s) != cudaSuccess) {
      cudaGetLastError();
      p = nullptr;
      return false;
    }
    return true;
  }
  ~Scratch() {
    if (p != nullptr) cudaFreeAsync(p, s);
  }
};

size_t round_up(size_t v, size_t unit) { return (v + unit - 1) / unit * unit; }

template <typename F>
int dispatch(int dtype, F&& f) {
  switch (dtype) {
    case PDNN_F32: return f(float{});
    case PDNN_F16: return f(__half{});
    case PDNN_BF16: return f(__nv_bfloat16{});
  }
  return fail(PDNN_INVALID_PARAMETER, "matmul_fused: unknown dtype %d", dtype);
}

// A matrix in memory: `rows` rows of `cols` elements, `pitch` elements apart.
struct Matrix {
  const void* p;
  long long pitch;
  int rows, cols;
};

// rows x cols of the source, zeros up to to_rows x to_cols.
template <typename W>
__global__ void __launch_bounds__(256) pad_matrix_kernel(const W* from, long long pitch, int rows, int cols, W* to, size_t items,
                                                         int to_cols) {
  overlap_wait();
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (size_t)gridDim.x * 256) {
    const size_t r = i / to_cols;
    const int c = (int)(i - r * to_cols);
    to[i] = r < (size_t)rows && c < cols ? from[(long long)r * pitch + c] : W(0);
  }
}

int pad_matrix(int dtype, const Matrix& a, void* to, int to_rows, int to_cols, cudaStream_t s) {
  const size_t items = (size_t)to_rows * to_cols;
  const unsigned grid = grid_for(items, 256, device_sm_count());
  if (dtype == PDNN_F32)
    launch_overlapped(pad_matrix_kernel<unsigned>, grid, 256, s, static_cast<const unsigned*>(a.p), a.pitch, a.rows, a.cols,
                      static_cast<unsigned*>(to), items, to_cols);
  else
    launch_overlapped(pad_matrix_kernel<unsigned short>, grid, 256, s, static_cast<const unsigned short*>(a.p), a.pitch, a.rows,
                      a.cols, static_cast<unsigned short*>(to), items, to_cols);
  return check_launch("matmul_fused: padding");
}

// What is made of a product.
struct Finish {
  const void* bias;
  const void* aux;     // forward: the residual; gradient: what the slope is taken of
  void* pre;           // forward: z
  void* out;
  long long aux_pitch, pre_pitch, out_pitch;
  int rows, cols, act, gradient;
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(256) finish_product_kernel(const float* z, long long z_pitch, const Finish f) {
  overlap_wait();
  const size_t items = (size_t)f.rows * f.cols;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (size_t)gridDim.x * 256) {
    const long long r = (long long)(i / f.cols);
    const int c = (int)(i - (size_t)r * f.cols);
    float v = z[r * z_pitch + c];
    if (f.bias != nullptr) v += to_f32(static_cast<const T*>(f.bias)[c]);
    if (f.pre != nullptr) static_cast<T*>(f.pre)[r * f.pre_pitch + c] = from_f32<T>(v);
    if (f.gradient) {
      if (f.aux != nullptr) v *= activation_slope(f.act, to_f32(static_cast<const T*>(f.aux)[r * f.aux_pitch + c]));
    } else {
      v = f.scale * activate(f.act, v);
      if (f.aux != nullptr) v += to_f32(static_cast<const T*>(f.aux)[r * f.aux_pitch + c]);
    }
    static_cast<T*>(f.out)[r * f.out_pitch + c] = from_f32<T>(v);
  }
}

// op(a) [m][k] times op(b) [k][n], ta / tb: stored the other way round, with f's finish.
int product(int dtype, int ta, int tb, const Matrix& a, const Matrix& b, int m, int k, int n, const Finish& f, cudaStream_t s) {
  const size_t es = dtype_size(dtype), unit = 16 / es;
  // The engine takes dense operands whose rows are whole 16-byte packets.
  const int pm = ta ? (int)round_up(m, unit) : m, pn = (int)round_up(n, unit);
  const int pk = !ta || tb ? (int)round_up(k, unit) : k;
  struct {
    const Matrix* m;
    int rows, cols;
    const void* p;
    size_t bytes;
  } op[2] = {{&a, ta ? pk : pm, ta ? pm : pk, a.p, 0}, {&b, tb ? pn : pk, tb ? pk : pn, b.p, 0}};
  size_t need = round_up((size_t)pm * pn * sizeof(float), 256);
  for (auto& o : op) {
    if (o.m->rows != o.rows || o.m->cols != o.cols || (o.m->pitch != o.m->cols && o.m->rows > 1) || !aligned16(o.p))
      o.bytes = round_up((size_t)o.rows * o.cols * es, 256);
    need += o.bytes;
  }
  Scratch scratch(s);
  if (!scratch.get(need)) return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused: cannot allocate %zu bytes of scratch", need);
  char* at = static_cast<char*>(scratch.p);
  float* z = reinterpret_cast<float*>(at);
  at += round_up((size_t)pm * pn * sizeof(float), 256);
  for (auto& o : op) {
    if (o.bytes == 0) continue;
    const int st = pad_matrix(dtype, *o.m, at, o.rows, o.cols, s);
    if (st != PDNN_OK) return st;
    o.p = at;
    at += o.bytes;
  }
  int st;
  if (tc_matmul_supported(dtype, ta, tb, op[0].p, op[1].p, z, 1, pm, pk, pn))
    st = tc_matmul(dtype, ta, tb, op[0].p, op[1].p, z, 1, pm, pk, pn, 0.f, s, /*out_f32=*/true);
  else
    st = simt_matmul(dtype, ta, tb, op[0].p, op[1].p, z, 1, pm, pk, pn, 0.f, s, /*out_f32=*/true);
  if (st != PDNN_OK) return st;
  const unsigned grid = grid_for((size_t)f.rows * f.cols, 256, device_sm_count());
  return dispatch(dtype, [&](auto type) {
    launch_overlapped(finish_product_kernel<decltype(type)>, grid, 256, s, z, (long long)pn, f);
    return check_launch("matmul_fused: epilogue");
  });
}

// ---- dz and the bias gradient -----------------------------------------------------------------------
// A block takes 32 pieces of V columns and a slice of the rows, eight of them at a time; its column sums are one line of
// `partial`.
constexpr int kSlopeLanes = 8;

struct SlopeArgs {
  const void *dy, *pre;
  void* dz;        // may be null: the sums alone
  float* partial;  // [slices][n]; may be null
  long long dy_pitch, pre_pitch, dz_pitch;
  int m, n, act, rows_per_slice;
  float scale;
};

template <typename T, int V>
__global__ void __launch_bounds__(32 * kSlopeLanes) activation_slope_kernel(const SlopeArgs a) {
  overlap_wait();
  __shared__ float red[kSlopeLanes][32 * V + 1];
  const int tx = (int)threadIdx.x & 31, ty = (int)threadIdx.x >> 5;
  const int col = ((int)blockIdx.x * 32 + tx) * V;
  const int first = (int)blockIdx.y * a.rows_per_slice, last = min(first + a.rows_per_slice, a.m);
  float sum[V] = {};
  if (col < a.n) {
#pragma unroll 2
    for (int r = first + ty; r < last; r += kSlopeLanes) {
      const T* dy = static_cast<const T*>(a.dy) + (long long)r * a.dy_pitch + col;
      const T* pre = static_cast<const T*>(a.pre) + (long long)r * a.pre_pitch + col;
      float v[V];
      if constexpr (V == 1) {
        v[0] = a.scale * to_f32(*dy) * (a.pre != nullptr ? activation_slope(a.act, to_f32(*pre)) : 1.f);
        if (a.dz != nullptr) static_cast<T*>(a.dz)[(long long)r * a.dz_pitch + col] = from_f32<T>(v[0]);
      } else {
        const Vec16<T> d = load16(dy);
        Vec16<T> z = d, o;
        if (a.pre != nullptr) z = load16(pre);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[i] = a.scale * to_f32(d.get(i)) * (a.pre != nullptr ? activation_slope(a.act, to_f32(z.get(i))) : 1.f);
          o.set(i, from_f32<T>(v[i]));
        }
        if (a.dz != nullptr) store16(static_cast<T*>(a.dz) + (long long)r * a.dz_pitch + col, o);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += v[i];
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < V; ++i) red[ty][tx * V + i] = sum[i];
  __syncthreads();
  for (int c = (int)threadIdx.x; c < 32 * V; c += 32 * kSlopeLanes) {
    const int at = (int)blockIdx.x * 32 * V + c;
    if (at >= a.n) continue;
    float v = 0.f;
#pragma unroll
    for (int y = 0; y < kSlopeLanes; ++y) v += red[y][c];
    a.partial[(size_t)blockIdx.y * a.n + at] = v;
  }
}

// dz of m x n into dz (null: not wanted), and the sums of its columns into bias_grad (null: not wanted).
int slope_and_sums(int dtype, const Matrix& dy, const void* pre, long long pre_pitch, int act, float scale, void* dz,
                   long long dz_pitch, void* bias_grad, cudaStream_t s) {
  const int sms = device_sm_count(), m = dy.rows, n = dy.cols;
  return dispatch(dtype, [&](auto type) {
    using T = decltype(type);
    constexpr int N = Vec16<T>::N;
    const bool packets = n % N == 0 && dy.pitch % N == 0 && aligned16(dy.p) &&
                         (pre == nullptr || (pre_pitch % N == 0 && aligned16(pre))) &&
                         (dz == nullptr || (dz_pitch % N == 0 && aligned16(dz)));
    const int width = 32 * (packets ? N : 1), tiles = (n + width - 1) / width;
    // slices of at least four rows to a thread, about four blocks to an SM
    int slices = std::max(1, std::min(4 * sms / tiles, (m + 4 * kSlopeLanes - 1) / (4 * kSlopeLanes)));
    slices = std::min(slices, 65535);
    SlopeArgs a = {};
    a.dy = dy.p;
    a.pre = pre;
    a.dz = dz;
    a.dy_pitch = dy.pitch;
    a.pre_pitch = pre_pitch;
    a.dz_pitch = dz_pitch;
    a.m = m;
    a.n = n;
    a.act = act;
    a.scale = scale;
    a.rows_per_slice = (m + slices - 1) / slices;
    slices = (m + a.rows_per_slice - 1) / a.rows_per_slice;
    Scratch scratch(s);
    if (bias_grad != nullptr) {
      if (!scratch.get((size_t)slices * n * sizeof(float))) return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused gradient: cannot allocate scratch");
      a.partial = static_cast<float*>(scratch.p);
    }
    const dim3 grid((unsigned)tiles, (unsigned)slices);
    if (packets)
      launch_overlapped(activation_slope_kernel<T, N>, grid, 32 * kSlopeLanes, s, a);
    else
      launch_overlapped(activation_slope_kernel<T, 1>, grid, 32 * kSlopeLanes, s, a);
    int st = check_launch("matmul_fused gradient: slope");
    if (st != PDNN_OK || bias_grad == nullptr) return st;
    launch_column_sums(a.partial, slices, (size_t)n, sms, s, StoreSum<T>{static_cast<T*>(bias_grad), false});
    return check_launch("matmul_fused gradient: bias");
  });
}

}  // namespace

int launch_matmul_fused(int dtype, const void* lhs, const void* rhs, void* out, const PdnnMatmulParams& p,
                        const PdnnMatmulEpilogue& e, cudaStream_t s) {
  Finish f = {};
  f.bias = e.bias;
  f.aux = e.residual;
  f.aux_pitch = e.residual_pitch;
  f.pre = e.pre_activation;
  f.pre_pitch = e.pre_activation_pitch;
  f.out = out;
  f.out_pitch = p.output_pitch;
  f.rows = p.m;
  f.cols = p.n;
  f.act = e.activation;
  f.scale = e.scale;
  const Matrix a{lhs, p.lhs_pitch, p.m, p.k}, b{rhs, p.rhs_pitch, p.transpose_rhs ? p.n : p.k, p.transpose_rhs ? p.k : p.n};
  return product(dtype, 0, p.transpose_rhs, a, b, p.m, p.k, p.n, f, s);
}

int launch_matmul_fused_gradient(int dtype, const void* grad, const void* lhs, const void* rhs, const PdnnMatmulParams& p,
                                 const PdnnMatmulGradient& g, cudaStream_t s) {
  const size_t es = dtype_size(dtype);
  const int w_rows = p.transpose_rhs ? p.n : p.k, w_cols = p.transpose_rhs ? p.k : p.n;
  if (p.m == 0) {  // sums over no rows
    if ((g.rhs_grad != nullptr && cudaMemset2DAsync(g.rhs_grad, g.rhs_grad_pitch * es, 0, w_cols * es, w_rows, s) != cudaSuccess) ||
        (g.bias_grad != nullptr && cudaMemsetAsync(g.bias_grad, 0, p.n * es, s) != cudaSuccess))
      return check_launch("matmul_fused gradient");
    return PDNN_OK;
  }
  Matrix dz{grad, p.output_pitch, p.m, p.n};
  const bool own = (g.activation != PDNN_ACT_NONE || g.scale != 1.f) && (g.lhs_grad != nullptr || g.rhs_grad != nullptr);
  Scratch scratch(s);
  if (own || g.bias_grad != nullptr) {
    const long long pitch = (long long)round_up(p.n, 16 / es);
    if (own && !scratch.get((size_t)p.m * pitch * es)) return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused gradient: cannot allocate scratch");
    const int st = slope_and_sums(dtype, dz, g.activation != PDNN_ACT_NONE ? g.pre_activation : nullptr, g.pre_activation_pitch,
                                  g.activation, g.scale, scratch.p, pitch, g.bias_grad, s);
    if (st != PDNN_OK) return st;
    if (own) {
      dz.p = scratch.p;
      dz.pitch = pitch;
    }
  }
  if (g.lhs_grad != nullptr) {
    Finish f = {};
    f.out = g.lhs_grad;
    f.out_pitch = g.lhs_grad_pitch;
    f.rows = p.m;
    f.cols = p.k;
    f.act = g.input_activation;
    f.gradient = 1;
    f.aux = g.input_activation != PDNN_ACT_NONE ? g.input_pre_activation : nullptr;
    f.aux_pitch = g.input_pre_activation_pitch;
    const int st = product(dtype, 0, !p.transpose_rhs, dz, Matrix{rhs, p.rhs_pitch, w_rows, w_cols}, p.m, p.n, p.k, f, s);
    if (st != PDNN_OK) return st;
  }
  if (g.rhs_grad != nullptr) {
    Finish f = {};
    f.out = g.rhs_grad;
    f.out_pitch = g.rhs_grad_pitch;
    f.rows = w_rows;
    f.cols = w_cols;
    f.gradient = 1;
    const Matrix x{lhs, p.lhs_pitch, p.m, p.k};
    const int st = p.transpose_rhs ? product(dtype, 1, 0, dz, x, p.n, p.m, p.k, f, s) : product(dtype, 1, 0, x, dz, p.k, p.m, p.n, f, s);
    if (st != PDNN_OK) return st;
  }
  return PDNN_OK;
}

}  // namespace pdnn
