// Clipped policy loss over the logits of a model's answers, with an estimate of the divergence from a reference
// policy, forward and gradient in one call.  For token i with target t, logits x, temperature tau:
//
//   lp    = x_t / tau - log sum_j exp(x_j / tau)             log-probability of the token now
//   ratio = exp(lp - old),  q = exp(ref - lp)
//   loss  = -min(ratio * A, clip(ratio, 1 - low, 1 + high) * A) + kl * (q - 1 - (ref - lp))
//   slope = d loss / d lp = -(ratio * A where that is the smaller one, else 0) + kl * (1 - q)
//   grad_j = grad_scale * w / tau * slope * ([j = t] - p_j),   p_j = exp(x_j / tau) / sum
//
// Bound by memory: the logits are read once and the gradient written once.  The loss of a token depends on its whole
// row, so that a block walks the row twice: once for the maximum and the sum - together, the sum scaled down whenever
// the maximum rises - and once for the gradient.  The rows that the device works on at a time stay in the 126 MB L2
// cache, from where the second walk reads them.  Few rows are split among the CTAs of a cluster, which exchange
// maxima and sums through distributed shared memory and add them in the order of their ranks.
#include "common.cuh"
#include "umma.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace pdnn {
namespace {

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;  // (log2 e, ln 2)

struct LossArgs {
  const void *logits, *targets;
  const float *advantages, *old_logp, *ref_logp, *weights;
  float *token_loss, *logp;
  void* grad;
  int rows, vocab, wide_targets;
  long long pitch, grad_pitch;
  float c, inv_temperature, clip_low, clip_high, kl, grad_scale;  // c = log2(e) / temperature
};

// Sums of 2^(x c - shift): the shift is the largest x so far times c, rounded, and cancels from every result, so that its
// rounding does no harm.  Of values that are all minus infinity the sum is 0 and the shift minus infinity.
struct alignas(8) Partial {
  float shift, sum;
};
__device__ __forceinline__ float scale_to(float from, float to) { return from == to ? 1.f : exp2_approx(from - to); }  // (both may be infinite)
__device__ __forceinline__ Partial merge(Partial a, Partial b) {
  const float shift = fmaxf(a.shift, b.shift);
  return Partial{shift, a.sum * scale_to(a.shift, shift) + b.sum * scale_to(b.shift, shift)};
}

// The largest entry (NaN passed over).
__device__ __forceinline__ float packet_max(const Vec16<float>& p) {
  return fmaxf(fmaxf(p.get(0), p.get(1)), fmaxf(p.get(2), p.get(3)));
}
__device__ __forceinline__ float packet_max(const Vec16<__half>& p) {
  const __half2* h = reinterpret_cast<const __half2*>(&p.raw);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float packet_max(const Vec16<__nv_bfloat16>& p) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&p.raw);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

template <typename T>
__device__ __forceinline__ void store_streaming(T* p, const Vec16<T>& v) {
  __stcs(reinterpret_cast<uint4*>(p), v.raw);
}

// One row to a cluster of CTAs (most often to a CTA).  An element costs an exponential in either walk, and as little else as
// possible: product and shift are one multiply-add, the gradient's factor is added to the exponent and its sign put
// on afterwards, and the chosen token's entry is written over at the end.
template <typename T>
__global__ void __launch_bounds__(512, 3) policy_loss_kernel(const LossArgs a) {
  overlap_wait();
  constexpr int N = Vec16<T>::N, kUnroll = 4;
  __shared__ Partial warp_part[16];
  __shared__ Partial cta_part;
  __shared__ float shared_slope;
  const int threads = (int)blockDim.x, tid = (int)threadIdx.x;
  uint32_t ranks, rank;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int row = (int)(blockIdx.x / ranks);
  const T* x = static_cast<const T*>(a.logits) + (size_t)row * a.pitch;
  T* g = a.grad != nullptr ? static_cast<T*>(a.grad) + (size_t)row * a.grad_pitch : nullptr;
  // this CTA's share of the row: [begin, body) and [tail, end) are what lies in front of the first 16-byte boundary and behind
  // the last; where logits and gradient lie on different ones there are no packets
  const int share = ((a.vocab + (int)ranks - 1) / (int)ranks + N - 1) / N * N;
  const int begin = min((int)rank * share, a.vocab), end = min(begin + share, a.vocab);
  const int head = (int)((16 - (reinterpret_cast<uintptr_t>(x + begin) & 15)) & 15) / (int)sizeof(T);
  const bool packets = g == nullptr || ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
  const int body = packets ? min(begin + head, end) : end, tail = packets ? body + (end - body) / N * N : end;
  const int kStep = threads * N;
  // f(whole, j): the packets at j, j + kStep, .. of the body, kUnroll of them, or as many as there are where it is not whole;
  // single(j): an element around it
  auto walk = [&](auto&& f, auto&& single) {
    int j = body + tid * N;
    for (; j + (kUnroll - 1) * kStep < tail; j += kUnroll * kStep) f(std::true_type{}, j);
    if (j < tail) f(std::false_type{}, j);
    for (j = begin + tid; j < body; j += threads) single(j);
    for (j = tail + tid; j < end; j += threads) single(j);
  };
  const long long t = a.wide_targets ? static_cast<const long long*>(a.targets)[row] : (long long)static_cast<const int*>(a.targets)[row];
  const float weight = a.weights != nullptr ? a.weights[row] : 1.f;
  // A row without weight or without a token counts for nothing, whatever stands in it: it is not read.
  const bool counts = weight != 0.f && t >= 0 && t < a.vocab;
  if (!counts) {
    if (rank == 0 && tid == 0) {
      a.token_loss[row] = 0.f;
      a.logp[row] = 0.f;
    }
    if (g != nullptr) {
      Vec16<T> zero;
      zero.raw = make_uint4(0u, 0u, 0u, 0u);
      walk([&](auto whole, int j) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (whole || j + u * kStep < tail) store_streaming(g + j + u * kStep, zero);
      }, [&](int j) { g[j] = from_f32<T>(0.f); });
    }
    return;  // (all CTAs of the cluster alike)
  }

  // (read ahead of every write: the gradient may take the place of the logits; and ahead of the row, whose end all wait for)
  float chosen = 0.f, adv = 0.f, old = 0.f, ref = 0.f;
  if (tid == 0) {
    chosen = to_f32(x[t]);
    adv = a.advantages[row];
    if (a.old_logp != nullptr) old = a.old_logp[row];
    if (a.ref_logp != nullptr) ref = a.ref_logp[row];
  }
  Partial part{-INFINITY, 0.f};
  // Makes room for a value: false where there is nothing but minus infinity so far (or NaN, which no maximum sees).
  auto rise = [&](float top) {
    const float shift = top * a.c;
    if (shift > part.shift) {
      part.sum *= exp2_approx(part.shift - shift);  // (from minus infinity: 0 times 0)
      part.shift = shift;
    }
    return part.shift != -INFINITY;
  };
  auto take = [&](float v) {
    if (rise(v))
      part.sum += exp2_approx(fmaf(v, a.c, -part.shift));
    else if (v != v)
      part.sum = v;
  };
  auto take_packet = [&](const Vec16<T>& p) {
    float2 v[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = make_float2(to_f32(p.get(2 * i)), to_f32(p.get(2 * i + 1)));
    if (rise(packet_max(p))) {
      float2 sum = both(0.f);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 e = fma2(v[i], both(a.c), both(-part.shift));
        sum = add2(sum, make_float2(exp2_approx(e.x), exp2_approx(e.y)));
      }
      part.sum += sum.x + sum.y;
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (v[i].x != v[i].x) part.sum = v[i].x;
        if (v[i].y != v[i].y) part.sum = v[i].y;
      }
    }
  };
  walk([&](auto whole, int j) {
    Vec16<T> p[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (whole || j + u * kStep < tail) p[u] = load16(x + j + u * kStep);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (whole || j + u * kStep < tail) take_packet(p[u]);
  }, [&](int j) {
    take(to_f32(x[j]));
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Partial other{__shfl_xor_sync(0xFFFFFFFFu, part.shift, o), __shfl_xor_sync(0xFFFFFFFFu, part.sum, o)};
    part = merge(part, other);
  }
  if ((tid & 31) == 0) warp_part[tid >> 5] = part;
  __syncthreads();
  // (each warp merges the warps' sums, of which there are a power of two)
  part = warp_part[(tid & 31) & (threads / 32 - 1)];
  for (int o = threads / 64; o > 0; o >>= 1) {
    const Partial other{__shfl_xor_sync(0xFFFFFFFFu, part.shift, o), __shfl_xor_sync(0xFFFFFFFFu, part.sum, o)};
    part = merge(part, other);
  }
  if (ranks > 1) {
    if (tid == 0) cta_part = part;
    __syncwarp();
    umma::cluster_sync_all();
    const uint32_t mine = umma::smem_u32(&cta_part);
    for (uint32_t r = 0; r < ranks; ++r) {
      Partial other;
      const uint32_t at = umma::cluster_map_shared(mine, r);
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(other.shift), "=f"(other.sum) : "r"(at) : "memory");
      part = r == 0 ? other : merge(part, other);
    }
    umma::cluster_sync_all();  // nobody leaves while its sums are read
  }
  float chosen_grad = 0.f;
  if (tid == 0) {
    float slope = 0.f, loss = 0.f, lp = 0.f;
    if (!(part.shift == -INFINITY && part.sum == 0.f)) {  // (a row of nothing but minus infinity counts for nothing)
      lp = (fmaf(chosen, a.c, -part.shift) - log2f(part.sum)) * kLn2;
      const float ratio = a.old_logp != nullptr ? expf(lp - old) : 1.f;
      const float open = ratio * adv, clipped = fminf(fmaxf(ratio, 1.f - a.clip_low), 1.f + a.clip_high) * adv;
      loss = -fminf(open, clipped);
      slope = open <= clipped ? -open : 0.f;
      if (open != open) loss = slope = open;
      if (a.ref_logp != nullptr) {
        const float d = ref - lp, q = expf(d);
        loss += a.kl * (q - d - 1.f);
        slope += a.kl * (1.f - q);
      }
      loss *= weight;
      slope *= weight * a.grad_scale * a.inv_temperature;
      chosen_grad = slope - slope * (exp2_approx(fmaf(chosen, a.c, -part.shift)) / part.sum);
    }
    shared_slope = slope;
    if (rank == 0) {
      a.token_loss[row] = loss;
      a.logp[row] = lp;
    }
  }
  if (g == nullptr) return;
  __syncthreads();
  // -slope * p_j = -sign(slope) * 2^(x_j c - shift + log2(|slope| / sum)), but for a slope of 0 (NaN stays NaN)
  const float slope = shared_slope;
  const float lift = log2f(fabsf(slope) / part.sum) - part.shift;
  const bool none = slope == 0.f;
  const uint32_t sign = slope > 0.f ? 0x80008000u : 0u;
  auto packet = [&](const Vec16<T>& p) {
    Vec16<T> o;
    if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 e = fma2(make_float2(to_f32(p.get(2 * i)), to_f32(p.get(2 * i + 1))), both(a.c), both(lift));
        w[i] = pair_word<T>(exp2_approx(e.x), exp2_approx(e.y)) ^ sign;
      }
      o.raw = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float e = exp2_approx(fmaf(to_f32(p.get(i)), a.c, lift));
        o.set(i, from_f32<T>(slope > 0.f ? -e : e));
      }
    }
    return o;
  };
  auto alone = [&](int j) {
    const float e = exp2_approx(fmaf(to_f32(x[j]), a.c, lift));
    g[j] = from_f32<T>(none ? 0.f : slope > 0.f ? -e : e);
  };
  walk([&](auto whole, int j) {
    Vec16<T> p[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (whole || j + u * kStep < tail) p[u] = load16(x + j + u * kStep);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (whole || j + u * kStep < tail) {
        Vec16<T> o = packet(p[u]);
        if (none) o.raw = make_uint4(0u, 0u, 0u, 0u);
        store_streaming(g + j + u * kStep, o);
      }
  }, alone);
  __syncthreads();
  if (tid == 0 && t >= begin && t < end) g[t] = from_f32<T>(chosen_grad);
}

// The sum of the tokens' losses, in one order.
__global__ void __launch_bounds__(1024) loss_sum_kernel(const float* token_loss, int rows, float* loss) {
  overlap_wait();
  __shared__ float warp_sums[32];
  float sum = 0.f;
  for (int i = (int)threadIdx.x; i < rows; i += 1024) sum += token_loss[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = warp_sums[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (threadIdx.x == 0) *loss = sum;
  }
}

template <typename T>
void launch_rows(const LossArgs& a, int cluster, int threads, cudaStream_t s) {
  const dim3 grid((unsigned)a.rows * (unsigned)cluster);
  if (cluster == 1) {
    launch_overlapped(policy_loss_kernel<T>, grid, (unsigned)threads, s, a);
    return;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, policy_loss_kernel<T>, a);  // (the caller's check_launch() reads the error)
}

}  // namespace

int launch_policy_loss(int dtype, const PdnnPolicyLossParams& p, const PdnnPolicyLossTensors& t, cudaStream_t s) {
  const char* what = "policy loss";
  if (dtype < PDNN_F32 || dtype > PDNN_BF16) return fail(PDNN_INVALID_PARAMETER, "%s: unknown dtype %d", what, dtype);
  if (p.rows < 0 || p.vocab <= 0) return fail(PDNN_INVALID_PARAMETER, "%s: %d rows of %d logits", what, p.rows, p.vocab);
  if (p.vocab > 1 << 30) return fail(PDNN_INDEX_EXCEEDED, "%s: rows of more than 2^30 logits", what);
  if (p.logits_pitch < p.vocab || (t.grad != nullptr && p.grad_pitch < p.vocab))
    return fail(PDNN_INVALID_PARAMETER, "%s: a row's pitch is shorter than the row", what);
  if (p.target_bytes != 4 && p.target_bytes != 8)
    return fail(PDNN_INVALID_PARAMETER, "%s: targets are whole numbers of 4 or 8 bytes", what);
  if (!(p.temperature > 0.f) || std::isinf(p.temperature))
    return fail(PDNN_INVALID_PARAMETER, "%s: the temperature must be positive", what);
  if (!(p.clip_low >= 0.f) || !(p.clip_high >= 0.f))
    return fail(PDNN_INVALID_PARAMETER, "%s: clipping bounds must not be negative", what);
  if (t.loss == nullptr) return fail(PDNN_INVALID_PARAMETER, "%s: null tensor", what);
  if (p.rows > 0 && (t.logits == nullptr || t.targets == nullptr || t.advantages == nullptr || t.token_loss == nullptr || t.logp == nullptr))
    return fail(PDNN_INVALID_PARAMETER, "%s: null tensor", what);
  {
    const long long es = (long long)dtype_size(dtype);
    const Extent in{t.logits, p.rows, p.vocab * es, p.logits_pitch * es}, out{t.grad, p.rows, p.vocab * es, p.grad_pitch * es};
    if (overlap(in, out) && !same_place(in, out)) return fail(PDNN_INVALID_PARAMETER, "%s: the gradient lies across the logits", what);
  }
  const int sms = device_sm_count();
  if (sms <= 0) return fail(PDNN_ALLOCATION_PROBLEM, "%s: no sm_100 CUDA device", what);
  if (p.rows > 0) {
    const long long es = (long long)dtype_size(dtype);
    LossArgs a = {};
    a.logits = t.logits;
    a.targets = t.targets;
    a.advantages = t.advantages;
    a.old_logp = t.old_logp;
    a.ref_logp = t.ref_logp;
    a.weights = t.weights;
    a.token_loss = t.token_loss;
    a.logp = t.logp;
    a.grad = t.grad;
    a.rows = p.rows;
    a.vocab = p.vocab;
    a.wide_targets = p.target_bytes == 8;
    a.pitch = p.logits_pitch;
    a.grad_pitch = p.grad_pitch;
    a.inv_temperature = 1.f / p.temperature;
    a.c = kLog2e / p.temperature;
    a.clip_low = p.clip_low;
    a.clip_high = p.clip_high;
    a.kl = p.kl;
    a.grad_scale = p.grad_scale;
    // A packet to a thread and walk, at most 512 threads; rows in shares of at least a walk of 128 threads while the device
    // has room for more blocks.
    const long long packets = ((long long)p.vocab * es + 15) / 16;
    int cluster = 1;
    while (cluster < 8 && (long long)p.rows * cluster * 2 <= 2ll * sms && packets / (cluster * 2) >= 128) cluster *= 2;
    // (rows enough for many blocks to an SM: four packets to a thread, so that a row's chain of latencies overlaps others)
    const int to_thread = (long long)p.rows * cluster >= 8ll * sms ? 4 : 2;
    int threads = to_thread == 4 ? 64 : 128;
    while (threads < 512 && packets / cluster > to_thread * threads) threads *= 2;
    if (dtype == PDNN_F32) launch_rows<float>(a, cluster, threads, s);
    if (dtype == PDNN_F16) launch_rows<__half>(a, cluster, threads, s);
    if (dtype == PDNN_BF16) launch_rows<__nv_bfloat16>(a, cluster, threads, s);
    const int st = check_launch(what);
    if (st != PDNN_OK) return st;
  }
  launch_overlapped(loss_sum_kernel, 1, 1024, s, t.token_loss, p.rows, t.loss);
  return check_launch("policy loss sum");
}

}  // namespace pdnn
