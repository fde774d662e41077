// The product of a few fp32 rows (tokens being served) with a weight matrix, and the end of the layer.
//
// Bound by memory: each weight is read once and meets at most eight rows.  The tensor cores would need the weights cut into
// parts first (fused_gemm.cu), which reads and writes several times their bytes; fp32 multiply-adds on the CUDA cores keep up
// with the memory.  A block takes a strip of columns; up to eight blocks of a cluster share K and add their sums in the
// order of their ranks.  Weights in rows of K: four of them to a warp, lanes along K, whose sums meet in shuffles.  Weights
// in columns of K: a packet of neighbouring columns to a lane, warps along K, whose sums meet in shared memory.
// One row of 4096 x 4096: 59 us on parts, 14.9 (rows of
// K) and 17.1 (columns) here, of which 10.3 are the weights' bytes.
#include "fused_gemm.cuh"

#include "activation.cuh"
#include "tc_gemm.cuh"
#include "umma.cuh"

#include <algorithm>

namespace pdnn {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kChunk = 1024, kFeatures = 4;

struct RowsArgs {
  const float *x, *w;
  long long x_pitch, w_pitch;
  int k, k_per_rank, n;
  Finish f;
};

template <int V>
__device__ __forceinline__ void load_floats(const float* p, float (&v)[V]) {
  if constexpr (V == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  } else {
    v[0] = *p;
  }
}

// M: rows (those behind the last are zeros).  V: elements to a load of the weights.
template <int M, int V, bool K_ROWS>
__global__ void __launch_bounds__(kThreads) rows_product_kernel(const RowsArgs a) {
  overlap_wait();
  constexpr int kCols = K_ROWS ? kWarps * kFeatures : 32 * V;  // columns of a block
  __shared__ __align__(16) float xs[M][kChunk];
  __shared__ float sums[M][kCols];
  const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t ranks, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int col0 = (int)(blockIdx.x / ranks) * kCols, row0 = (int)blockIdx.y * M, rows = min(M, a.f.rows - row0);
  const int k0 = (int)rank * a.k_per_rank, k1 = min(k0 + a.k_per_rank, a.k);
  constexpr int kMine = K_ROWS ? kFeatures : V;  // columns of a thread
  float acc[M][kMine] = {};
  for (int c0 = k0; c0 < k1; c0 += kChunk) {
    const int len = min(kChunk, k1 - c0);
    __syncthreads();
    for (int i = tid; i < M * kChunk; i += kThreads) {
      const int r = i / kChunk, c = i % kChunk;
      xs[r][c] = r < rows && c < len ? a.x[(long long)(row0 + r) * a.x_pitch + c0 + c] : 0.f;
    }
    __syncthreads();
    if constexpr (K_ROWS) {
      const float* w[kFeatures];
#pragma unroll
      for (int j = 0; j < kFeatures; ++j) w[j] = a.w + (long long)min(col0 + warp * kFeatures + j, a.n - 1) * a.w_pitch + c0;
#pragma unroll 2
      for (int i = lane * V; i < len; i += 32 * V) {  // (V = 4: the chunk is whole packets but for the matrix' last ones)
        float v[kFeatures][V];
        const bool whole = i + V <= len;
#pragma unroll
        for (int j = 0; j < kFeatures; ++j) {
          if (whole) {
            load_floats<V>(w[j] + i, v[j]);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[j][e] = i + e < len ? w[j][i + e] : 0.f;
          }
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
          float x[V];
          load_floats<V>(&xs[m][i], x);
#pragma unroll
          for (int j = 0; j < kFeatures; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[m][j] += x[e] * v[j][e];
        }
      }
    } else {
      const int col = col0 + lane * V;
      if (col < a.n) {
        const bool whole = col + V <= a.n;
#pragma unroll 1
        for (int i = warp * 4; i < len; i += kWarps * 4) {
          float v[4][V];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float* w = a.w + (long long)(c0 + i + u) * a.w_pitch + col;
            if (i + u < len && whole) {
              load_floats<V>(w, v[u]);
            } else {
#pragma unroll
              for (int e = 0; e < V; ++e) v[u][e] = i + u < len && col + e < a.n ? w[e] : 0.f;
            }
          }
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const float4 x = *reinterpret_cast<const float4*>(&xs[m][i]);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[m][e] += x.x * v[0][e] + x.y * v[1][e] + x.z * v[2][e] + x.w * v[3][e];
          }
        }
      }
    }
  }
  // the block's sums
  if constexpr (K_ROWS) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < kFeatures; ++j) {
        float v = acc[m][j];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        if (lane == 0) sums[m][warp * kFeatures + j] = v;
      }
  } else {
    __syncthreads();
    float* part = &xs[0][0];  // [warp][M][kCols], in the rows' place
    static_assert(kWarps * kCols <= kChunk, "the partial sums take the rows' place");
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int e = 0; e < V; ++e) part[(warp * M + m) * kCols + lane * V + e] = acc[m][e];
    __syncthreads();
    for (int i = tid; i < M * kCols; i += kThreads) {
      float v = 0.f;
#pragma unroll
      for (int p = 0; p < kWarps; ++p) v += part[p * M * kCols + i];
      sums[i / kCols][i % kCols] = v;
    }
  }
  __syncthreads();
  umma::cluster_sync_all();
  const Finish& f = a.f;
  for (int i = (int)rank * kThreads + tid; i < rows * kCols; i += (int)ranks * kThreads) {
    const int r = i / kCols, c = i % kCols, col = col0 + c;
    if (col >= a.n) continue;
    const uint32_t at = umma::smem_u32(&sums[r][c]);
    float v = 0.f;
    for (uint32_t p = 0; p < ranks; ++p) {
      float s;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s) : "r"(umma::cluster_map_shared(at, p)) : "memory");
      v += s;
    }
    const long long row = row0 + r;
    if (f.bias != nullptr) v += static_cast<const float*>(f.bias)[col];
    if (f.pre != nullptr) static_cast<float*>(f.pre)[row * f.pre_pitch + col] = v;
    const float x = f.aux != nullptr ? static_cast<const float*>(f.aux)[row * f.aux_pitch + col] : 0.f;
    if (f.gradient)
      v = f.scale * (f.aux != nullptr ? v * activation_slope(f.act, x) : v);
    else
      v = f.scale * activate(f.act, v) + x;
    static_cast<float*>(f.out)[row * f.out_pitch + col] = v;
  }
  __syncwarp();
  umma::cluster_sync_all();  // nobody leaves while its sums are read
}

template <int M, int V, bool K_ROWS>
int launch(const RowsArgs& a, int sms, cudaStream_t s) {
  constexpr int kCols = K_ROWS ? kWarps * kFeatures : 32 * V;
  const int strips = (a.n + kCols - 1) / kCols, groups = (a.f.rows + M - 1) / M;
  int ranks = 1;  // blocks for two to an SM, with a quarter of a chunk to each
  while (ranks < 8 && (long long)strips * groups * ranks < 2ll * sms && a.k >= ranks * 2 * (kChunk / 4)) ranks *= 2;
  RowsArgs args = a;
  args.k_per_rank = ((a.k + ranks - 1) / ranks + 3) / 4 * 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(strips * ranks), (unsigned)groups);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, rows_product_kernel<M, V, K_ROWS>, args);  // (check_launch reads the error)
  tc_set_last_kernel("rows_product_kernel");
  return check_launch("matmul_fused (rows)");
}

}  // namespace

int fused_rows(bool k_rows, const Matrix& x, const Matrix& w, int k, const Finish& f, cudaStream_t s) {
  const int sms = device_sm_count();
  RowsArgs a = {};
  a.x = static_cast<const float*>(x.p);
  a.w = static_cast<const float*>(w.p);
  a.x_pitch = x.pitch;
  a.w_pitch = w.pitch;
  a.k = k;
  a.n = f.cols;
  a.f = f;
  // (columns of K: strips of 32 columns, not 128, where eight blocks to a strip would leave SMs idle.  One row of 8192 x 1024: 25.8 us in
  // strips of 128)
  const bool packets = aligned16(w.p) && w.pitch % 4 == 0 && (k_rows || (f.cols + 127) / 128 * 8 * ((f.rows + 7) / 8) >= sms);
  auto run = [&](auto m) {
    constexpr int M = decltype(m)::value;
    if (k_rows) return packets ? launch<M, 4, true>(a, sms, s) : launch<M, 1, true>(a, sms, s);
    return packets ? launch<M, 4, false>(a, sms, s) : launch<M, 1, false>(a, sms, s);
  };
  if (f.rows == 1) return run(std::integral_constant<int, 1>{});
  if (f.rows <= 2) return run(std::integral_constant<int, 2>{});
  if (f.rows <= 4) return run(std::integral_constant<int, 4>{});
  return run(std::integral_constant<int, 8>{});
}

}  // namespace pdnn
