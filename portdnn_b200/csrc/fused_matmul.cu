// The matrix product with bias, activation and residual, and its gradients:
//
//   z = lhs * rhs + bias,  out = residual + scale * act(z)
//   dz = scale * dy * act'(z),  d_lhs = dz * rhs^T (times act_in'(z_in)),  d_rhs = lhs^T * dz,  d_bias = sum of dz's rows
//
// Each product with its end is one launch of fused_gemm.cu's.  What is left here is dz - the elementwise slope, one pass that
// takes the bias gradient's sums on its way - and copies of 16-bit operands that TMA cannot read in place.
#include "activation.cuh"
#include "column_sums.cuh"
#include "fused_gemm.cuh"

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

// The 16-bit elements of a matrix in rows of to_cols, zeros behind the matrix' own.
__global__ void __launch_bounds__(256) pad_matrix_kernel(const unsigned short* from, long long pitch, int cols, unsigned short* to,
                                                         size_t items, int to_cols) {
  overlap_wait();
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (size_t)gridDim.x * 256) {
    const size_t r = i / to_cols;
    const int c = (int)(i - r * to_cols);
    to[i] = c < cols ? from[(long long)r * pitch + c] : (unsigned short)0;
  }
}

// op(a) times op(b) with f's finish; ta, tb: stored the other way round.
int product(int dtype, int ta, int tb, const Matrix& a, const Matrix& b, int k, const Finish& f, cudaStream_t s) {
  Matrix in[2] = {a, b};
  size_t bytes[2] = {0, 0};
  const size_t es = dtype_size(dtype);
  for (int i = 0; i < 2; ++i)
    if (!fused_gemm_operand_ok(dtype, in[i])) bytes[i] = round_up((size_t)in[i].rows * round_up(in[i].cols, 16 / es) * es, 256);
  Scratch scratch(s);
  if (!scratch.get(bytes[0] + bytes[1]))
    return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused: cannot allocate %zu bytes of scratch", bytes[0] + bytes[1]);
  for (int i = 0; i < 2; ++i) {
    if (bytes[i] == 0) continue;
    char* to = static_cast<char*>(scratch.p) + (i == 0 ? 0 : bytes[0]);
    const int pitch = (int)round_up(in[i].cols, 16 / es);
    const size_t items = (size_t)in[i].rows * pitch;
    launch_overlapped(pad_matrix_kernel, grid_for(items, 256, device_sm_count()), 256, s, static_cast<const unsigned short*>(in[i].p),
                      in[i].pitch, in[i].cols, reinterpret_cast<unsigned short*>(to), items, pitch);
    const int st = check_launch("matmul_fused: padding");
    if (st != PDNN_OK) return st;
    in[i].p = to;
    in[i].pitch = pitch;
  }
  return fused_gemm(dtype, ta, tb, in[0], in[1], k, f, s);
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
  if (col < a.n)
    with_activation(a.pre != nullptr ? a.act : PDNN_ACT_NONE, [&](auto act) {
      constexpr int ACT = decltype(act)::value, kAhead = V == 1 ? 8 : 4;  // rows of a thread whose loads are in flight together
      for (int r0 = first + ty; r0 < last; r0 += kAhead * kSlopeLanes) {
        Piece<T, V> d[kAhead], z[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int r = r0 + u * kSlopeLanes;
          if (r >= last) continue;
          d[u].load(static_cast<const T*>(a.dy) + (long long)r * a.dy_pitch + col);
          if (ACT != PDNN_ACT_NONE) z[u].load(static_cast<const T*>(a.pre) + (long long)r * a.pre_pitch + col);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int r = r0 + u * kSlopeLanes;
          if (r >= last) continue;
          float dz[V];
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            constexpr int kNext = V > 1 ? 1 : 0;
            float2 v = make_float2(a.scale * d[u].get(i), a.scale * d[u].get(i + kNext));
            if (ACT != PDNN_ACT_NONE) v = mul2(v, slope_of<ACT, T>(make_float2(z[u].get(i), z[u].get(i + kNext))));
            dz[i + kNext] = v.y;
            dz[i] = v.x;
          }
#pragma unroll
          for (int i = 0; i < V; ++i) sum[i] += dz[i];
          Piece<T, V> o;
          o.round(dz);
          if (a.dz != nullptr) o.store(static_cast<T*>(a.dz) + (long long)r * a.dz_pitch + col);
        }
      }
    });
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
  return product(dtype, 0, p.transpose_rhs, a, b, p.k, f, s);
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
  // (without an activation dz is dy, and the scale goes into the products' ends)
  const bool own = g.activation != PDNN_ACT_NONE && (g.lhs_grad != nullptr || g.rhs_grad != nullptr);
  const float end_scale = g.activation != PDNN_ACT_NONE ? 1.f : g.scale;
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
    f.scale = end_scale;
    f.gradient = 1;
    f.aux = g.input_activation != PDNN_ACT_NONE ? g.input_pre_activation : nullptr;
    f.aux_pitch = g.input_pre_activation_pitch;
    const int st = product(dtype, 0, !p.transpose_rhs, dz, Matrix{rhs, p.rhs_pitch, w_rows, w_cols}, p.n, f, s);
    if (st != PDNN_OK) return st;
  }
  if (g.rhs_grad != nullptr) {
    Finish f = {};
    f.out = g.rhs_grad;
    f.out_pitch = g.rhs_grad_pitch;
    f.rows = w_rows;
    f.cols = w_cols;
    f.act = PDNN_ACT_NONE;
    f.scale = end_scale;
    f.gradient = 1;
    const Matrix x{lhs, p.lhs_pitch, p.m, p.k};
    const int st = p.transpose_rhs ? product(dtype, 1, 0, dz, x, p.m, f, s) : product(dtype, 1, 0, x, dz, p.m, f, s);
    if (st != PDNN_OK) return st;
  }
  return PDNN_OK;
}

}  // namespace pdnn
