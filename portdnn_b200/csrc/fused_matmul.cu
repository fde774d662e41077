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
#include "umma.cuh"

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

// op(a) times op(b) with f's finish; ta, tb: stored the other way round.  alone: nothing but the product was launched.
// beside: as fused_gemm's (not where copies come first).
int product(int dtype, int ta, int tb, const Matrix& a, const Matrix& b, int k, const Finish& f, cudaStream_t s, bool beside = false,
            bool* alone = nullptr) {
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
  const bool copied = bytes[0] + bytes[1] > 0 || dtype == PDNN_F32;
  if (alone != nullptr) *alone = !copied;
  return fused_gemm(dtype, ta, tb, in[0], in[1], k, f, beside && !copied, s);
}

// ---- dz and the bias gradient -----------------------------------------------------------------------
// Bound by memory: dy and z are read once and dz written once.  A block takes CL pieces of V columns, its other threads lie along
// the rows; the blocks of a cluster share the rows of their columns and add their sums in the order of their ranks, so
// that the bias gradient needs neither scratch nor a second launch.  Large tensors are cut into more slices of rows than a
// cluster has blocks, and wider ones (512 bytes of a row to a warp): there every slice leaves a line of sums for
// column_sums.cuh (8192x8192 bf16 gelu, sums alone, cluster of eight / slices 76 / 64 us; 512x512 with both products 13.4 / 15.2).
constexpr int kSlopeThreads = 256;
constexpr long long kSlicedElements = 8ll << 20;

struct SlopeArgs {
  const void *dy, *pre;
  void *dz, *bias_grad;  // either may be null
  float* partial;        // [slices][n], in the place of bias_grad
  long long dy_pitch, pre_pitch, dz_pitch;
  int m, n, act, rows_per_rank;
  float scale;
};

template <typename T, int V, int CL>
__global__ void __launch_bounds__(kSlopeThreads, 4) activation_slope_kernel(const SlopeArgs a) {
  overlap_wait();
  constexpr int RL = kSlopeThreads / CL, kCols = CL * V;
  __shared__ float red[RL][kCols + 1];
  __shared__ float sums[kCols];
  uint32_t ranks, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int tx = (int)threadIdx.x % CL, ty = (int)threadIdx.x / CL, col0 = (int)(blockIdx.x / ranks) * kCols, col = col0 + tx * V;
  const int slice = (int)blockIdx.y + (int)rank;  // (slices or ranks: the other is 0)
  const int first = min(slice * a.rows_per_rank, a.m), last = min(first + a.rows_per_rank, a.m);
  float sum[V] = {};
  if (col < a.n)
    with_activation(a.pre != nullptr ? a.act : PDNN_ACT_NONE, [&](auto act) {
      constexpr int ACT = decltype(act)::value, kAhead = V == 1 ? 8 : 4;  // rows of a thread whose loads are in flight together
      for (int r0 = first + ty; r0 < last; r0 += kAhead * RL) {
        Piece<T, V> d[kAhead], z[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int r = r0 + u * RL;
          if (r >= last) continue;
          d[u].load(static_cast<const T*>(a.dy) + (long long)r * a.dy_pitch + col);
          if (ACT != PDNN_ACT_NONE) z[u].load(static_cast<const T*>(a.pre) + (long long)r * a.pre_pitch + col);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int r = r0 + u * RL;
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
  if (a.bias_grad == nullptr && a.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < V; ++i) red[ty][tx * V + i] = sum[i];
  __syncthreads();
  for (int c = (int)threadIdx.x; c < kCols; c += kSlopeThreads) {
    float v = 0.f;
#pragma unroll
    for (int y = 0; y < RL; ++y) v += red[y][c];
    if (a.partial != nullptr && col0 + c < a.n) a.partial[(size_t)slice * a.n + col0 + c] = v;
    sums[c] = v;
  }
  if (a.partial != nullptr) return;
  __syncthreads();
  umma::cluster_sync_all();
  for (int c = (int)(rank * kSlopeThreads + threadIdx.x); c < kCols && col0 + c < a.n; c += (int)ranks * kSlopeThreads) {
    const uint32_t at = umma::smem_u32(&sums[c]);
    float v = 0.f;
    for (uint32_t r = 0; r < ranks; ++r) {
      float s;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s) : "r"(umma::cluster_map_shared(at, r)) : "memory");
      v += s;
    }
    static_cast<T*>(a.bias_grad)[col0 + c] = from_f32<T>(v);
  }
  __syncwarp();
  umma::cluster_sync_all();  // nobody leaves while its sums are read
}

template <typename T, int V, int CL>
int launch_slope(const SlopeArgs& args, cudaStream_t s) {
  constexpr int RL = kSlopeThreads / CL, kCols = CL * V;
  SlopeArgs a = args;
  int ranks = 1;  // four rows to a thread, or as many blocks as a cluster has
  while (ranks < 8 && a.m > ranks * RL * 4) ranks *= 2;
  a.rows_per_rank = (a.m + ranks - 1) / ranks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.n + kCols - 1) / kCols * ranks));
  cfg.blockDim = dim3(kSlopeThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, activation_slope_kernel<T, V, CL>, a);  // (check_launch reads the error)
  return check_launch("matmul_fused gradient: slope");
}

// dz of m x n into dz (null: not wanted), and the sums of its columns into bias_grad (null: not wanted).
int slope_and_sums(int dtype, const Matrix& dy, const void* pre, long long pre_pitch, int act, float scale, void* dz,
                   long long dz_pitch, void* bias_grad, cudaStream_t s) {
  const int sms = device_sm_count();
  return dispatch(dtype, [&](auto type) {
    using T = decltype(type);
    constexpr int N = Vec16<T>::N;
    SlopeArgs a = {};
    a.dy = dy.p;
    a.pre = pre;
    a.dz = dz;
    a.bias_grad = bias_grad;
    a.dy_pitch = dy.pitch;
    a.pre_pitch = pre_pitch;
    a.dz_pitch = dz_pitch;
    a.m = dy.rows;
    a.n = dy.cols;
    a.act = act;
    a.scale = scale;
    const bool packets = a.n % N == 0 && dy.pitch % N == 0 && aligned16(dy.p) &&
                         (pre == nullptr || (pre_pitch % N == 0 && aligned16(pre))) &&
                         (dz == nullptr || (dz_pitch % N == 0 && aligned16(dz)));
    if ((long long)a.m * a.n >= kSlicedElements && a.n >= 32 * N && packets) {
      const int tiles = (a.n + 32 * N - 1) / (32 * N);
      const int slices = std::max(1, std::min(4 * sms / tiles, a.m / 32));  // about four blocks to an SM
      a.rows_per_rank = (a.m + slices - 1) / slices;
      const int lines = (a.m + a.rows_per_rank - 1) / a.rows_per_rank;
      Scratch scratch(s);
      if (bias_grad != nullptr) {
        if (!scratch.get((size_t)lines * a.n * sizeof(float)))
          return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused gradient: cannot allocate scratch");
        a.partial = static_cast<float*>(scratch.p);
        a.bias_grad = nullptr;
      }
      launch_overlapped(activation_slope_kernel<T, N, 32>, dim3((unsigned)tiles, (unsigned)lines), kSlopeThreads, s, a);
      const int st = check_launch("matmul_fused gradient: slope");
      if (st != PDNN_OK || bias_grad == nullptr) return st;
      launch_column_sums(a.partial, lines, (size_t)a.n, sms, s, StoreSum<T>{static_cast<T*>(bias_grad), false});
      return check_launch("matmul_fused gradient: bias");
    }
    if (!packets) return launch_slope<T, 1, 32>(a, s);
    // the width whose blocks (eight to a strip) come out most evenly on the SMs, the widest of equals (8192x8192 gelu, sums alone: 16
    // pieces, 3.5 blocks to an SM, 84 us; eight, 6.9, 76)
    auto evenness = [&](int pieces) {
      const int blocks = (a.n + pieces * N - 1) / (pieces * N) * 8;
      return (double)blocks / ((blocks + sms - 1) / sms * sms);
    };
    const double wide = evenness(16), middle = evenness(8), narrow = evenness(4);
    if (wide >= middle && wide >= narrow) return launch_slope<T, N, 16>(a, s);
    return middle >= narrow ? launch_slope<T, N, 8>(a, s) : launch_slope<T, N, 4>(a, s);
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
  bool alone = false;  // the launch ahead of the next product is a product, too
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
    const int st = product(dtype, 0, !p.transpose_rhs, dz, Matrix{rhs, p.rhs_pitch, w_rows, w_cols}, p.n, f, s, false, &alone);
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
    const int st = p.transpose_rhs ? product(dtype, 1, 0, dz, x, p.m, f, s, alone) : product(dtype, 1, 0, x, dz, p.m, f, s, alone);
    if (st != PDNN_OK) return st;
  }
  return PDNN_OK;
}

}  // namespace pdnn
