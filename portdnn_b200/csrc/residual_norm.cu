// The norms around a block of a network, its gate and its residual sum, in one pass forward and one back:
//
//   n   = norm_post(branch)                    the block's output, normalised (or as it is)
//   sum = residual + scale * act(gate) * n     the residual stream behind the block
//   out = norm_pre(sum)                        what the next block reads
//
// norm(v) = (v - mean) * r * gamma + beta with r = 1 / sqrt(mean((v - mean)^2) + epsilon), mean = 0 and no beta for the
// root-mean-square form.  With hat = (v - mean) * r and u = gradient * gamma the way back through a norm is
//   dv = r * (u - hat * mean(u * hat) - mean(u)),   the last term for layer norms only.
//
// Bound by memory: forward reads two tensors and writes two, backward reads four and writes two, each once.  A
// team of threads keeps a row in registers (a packet or two to a thread), so that statistics over the row - taken
// about the mean, in fp32 - cost no second read, and has the next three rows on their way.  Teams keep to
// whole stretches of rows: what depends on the column alone stays in registers, multiplied out (scale * act(gate) * gamma
// is one number), and the sums over rows of the backward pass are the thread's own until its stretch ends.  Both of
// the gradients behind the post norm's result come of one sum over the group's rows, P = sum ds * hat: gamma's is
// scale * act(gate) * P, the gate's scale * act'(gate) * gamma * P.  A block leaves one line of partial sums, which a second
// launch adds in a fixed order.
#include "activation.cuh"
#include "common.cuh"
#include "umma.cuh"

#include <algorithm>
#include <cstring>
#include <initializer_list>
#include <mutex>
#include <type_traits>

namespace pdnn {
namespace {

// Rows on their way: a thread asks for its own pieces of the rows to come, kAhead of them, with cp.async into slots of shared
// memory that nobody else touches, so that no barrier is needed and no registers wait.  (Packets; smaller pieces are
// requested into registers one row ahead: four bytes to a copy are too few, 1999x1003 f32 gradient 23.4 us so, 21.9 in registers.)
template <typename T, int V>
constexpr bool in_slots() { return V * sizeof(T) == 16; }

__device__ __forceinline__ void async_copy(void* slot, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(slot)), "l"(from) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// TENSORS tensors' pieces of a thread, NP of each, AHEAD rows.
template <typename T, int V, int NP, int TENSORS, int AHEAD, int THREADS>
struct Incoming {
  static constexpr bool kSlots = in_slots<T, V>();
  static constexpr int kBytes = V * (int)sizeof(T), kRow = TENSORS * NP * THREADS * kBytes;
  static constexpr int kFit = 200 * 1024 / kRow, kDepth = !kSlots || kFit < 1 ? 1 : kFit < AHEAD ? kFit : AHEAD;
  static constexpr int kSharedBytes = kSlots ? kDepth * kRow : 0;
  Piece<T, V> held[kSlots ? 1 : TENSORS][NP];
  char* mine;  // [depth][tensor][piece][thread]
  int slot = 0;

  __device__ __forceinline__ Incoming(char* shared) : mine(shared + (int)threadIdx.x * kBytes) {
    Piece<T, V> zero;
    zero.clear();
    if constexpr (kSlots) {  // (what is never asked for is zero)
      for (int i = 0; i < kDepth * TENSORS * NP; ++i) zero.store(reinterpret_cast<T*>(mine + i * THREADS * kBytes));
    } else {
#pragma unroll
      for (int i = 0; i < TENSORS; ++i)
#pragma unroll
        for (int p = 0; p < NP; ++p) held[i][p] = zero;
    }
  }
  // Asks for a row's pieces (null tensors stay zero) into the slot of `row` steps from now; one group a row, asked for or not.
  __device__ __forceinline__ void request(const T* const (&from)[TENSORS], size_t base, bool wanted, const bool (&live)[NP],
                                          const int (&at)[NP], int into) {
    if (wanted) {
#pragma unroll
      for (int i = 0; i < TENSORS; ++i)
#pragma unroll
        for (int p = 0; p < NP; ++p)
          if (live[p] && from[i] != nullptr) {
            if constexpr (kSlots)
              async_copy(mine + ((into * TENSORS + i) * NP + p) * THREADS * kBytes, from[i] + base + at[p]);
            else
              held[i][p].load(from[i] + base + at[p]);
          }
    }
    if constexpr (kSlots) async_commit();
  }
  // The oldest row's pieces.
  __device__ __forceinline__ void take(Piece<T, V> (&to)[TENSORS][NP]) {
    if constexpr (kSlots) {
      async_wait<kDepth - 1>();
#pragma unroll
      for (int i = 0; i < TENSORS; ++i)
#pragma unroll
        for (int p = 0; p < NP; ++p) to[i][p].load(reinterpret_cast<const T*>(mine + ((slot * TENSORS + i) * NP + p) * THREADS * kBytes));
    } else {
#pragma unroll
      for (int i = 0; i < TENSORS; ++i)
#pragma unroll
        for (int p = 0; p < NP; ++p) to[i][p] = held[i][p];
    }
  }
  // The slot just taken from is the next one to be filled.
  __device__ __forceinline__ int freed() {
    const int s = slot;
    slot = slot + 1 == kDepth ? 0 : slot + 1;
    return s;
  }
};

// o = a * b + c and o = a * b, two entries to an instruction where there are pairs.
template <int V>
__device__ __forceinline__ void fma_all(float (&o)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V == 1) {
    o[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = fma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), make_float2(c[i], c[i + 1]));
      o[i] = r.x;
      o[i + 1] = r.y;
    }
  }
}
template <int V>
__device__ __forceinline__ void mul_all(float (&o)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    o[0] = a[0] * b[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = mul2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
      o[i] = r.x;
      o[i + 1] = r.y;
    }
  }
}
// The same with one factor for all, and o = (a + c) * b with c and b for all.
template <int V>
__device__ __forceinline__ void mul_by(float (&o)[V], const float (&a)[V], float b) {
  if constexpr (V == 1) {
    o[0] = a[0] * b;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = mul2(make_float2(a[i], a[i + 1]), both(b));
      o[i] = r.x;
      o[i + 1] = r.y;
    }
  }
}
template <int V>
__device__ __forceinline__ void add_mul(float (&o)[V], const float (&a)[V], float c, float b) {
  if constexpr (V == 1) {
    o[0] = (a[0] + c) * b;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = mul2(add2(make_float2(a[i], a[i + 1]), both(c)), both(b));
      o[i] = r.x;
      o[i + 1] = r.y;
    }
  }
}
// The sum of all products a * b.
template <int V, int NP>
__device__ __forceinline__ float dot(const float (&a)[NP][V], const float (&b)[NP][V]) {
  if constexpr (V == 1) {
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < NP; ++p) s = fmaf(a[p][0], b[p][0], s);
    return s;
  } else {
    float2 s = both(0.f);
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int i = 0; i < V; i += 2) s = fma2(make_float2(a[p][i], a[p][i + 1]), make_float2(b[p][i], b[p][i + 1]), s);
    return s.x + s.y;
  }
}
template <int V, int NP>
__device__ __forceinline__ float total(const float (&a)[NP][V]) {
  float s = 0.f;
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < V; ++i) s += a[p][i];
  return s;
}

struct NormArgs {
  const void *branch, *residual, *post_gamma, *post_beta, *gate, *pre_gamma, *pre_beta;
  void *sum, *out;
  float* statistics;  // [4][rows]: mean and r behind the block, mean and r before the next; may be null
  int rows, channels, post_norm, pre_norm, gate_groups, gate_activation, rows_per_group;
  float scale, epsilon, inv_channels;
  // backward
  const void *sum_grad, *out_grad;
  void *branch_grad, *residual_grad, *gate_grad;
  // Partial sums: a line of `line` floats to a block, the parameter vectors' behind one another, the gate's too (vector
  // gate_vector) where there is one group; with more groups (gate_vector -1) the gate's are [parts][groups][channels].
  float *partial, *gate_partial, *row_sums;
  size_t line;
  int parts;    // stretches of rows that a group is cut into
  int vectors;  // parameter vectors with a gradient
  int gate_vector;
  int slot[4];                    // where in a line of `partial` post gamma, post beta, pre gamma, pre beta are; -1: nowhere
};

// Sums over a team of one value or two.  Teams of a warp need no barrier; others use two sets of slots in turn, so that one
// barrier a reduction is enough: whoever is about to write a set has passed the barrier behind everybody's last read of it.
// (Each warp adds the warps' sums up in shuffles: a thread that reads all sixteen of 512 threads has as much to do with them as with
// its eight elements.)
template <int TEAM>
struct TeamSum {
  float2* slots;  // the team's, [2][TEAM / 32]; twice as many for three values
  int turn = 0;
  template <int COUNT>
  __device__ __forceinline__ float2 sum(float a, float b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
      if (COUNT == 2) b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    if constexpr (TEAM > 32) {
      constexpr int W = TEAM / 32;
      float2* mine = slots + turn * W;
      turn ^= 1;
      const int warp = (int)(threadIdx.x >> 5) & (W - 1);
      if ((threadIdx.x & 31) == 0) {
        if (COUNT == 2) mine[warp] = make_float2(a, b);
        else mine[warp].x = a;
      }
      if (TEAM >= 256)
        __syncthreads();
      else  // (a block has several teams)
        umma::named_barrier_sync(1 + threadIdx.x / TEAM, TEAM);
      const int from = (int)threadIdx.x & (W - 1);
      a = mine[from].x;
      if (COUNT == 2) b = mine[from].y;
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
        if (COUNT == 2) b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
      }
    }
    return make_float2(a, b);
  }
  // Three values at once (one barrier, and twelve shuffles where one after another takes 27): two steps leave a lane with one of them.
  __device__ __forceinline__ float3 three(float a, float b, float c) {
    const int lane = (int)threadIdx.x & 31;
    const bool odd = (lane & 1) != 0, upper = (lane & 2) != 0;
    float x = odd ? b : a, y = odd ? 0.f : c;
    x += __shfl_xor_sync(0xFFFFFFFFu, odd ? a : b, 1);
    y += __shfl_xor_sync(0xFFFFFFFFu, odd ? c : 0.f, 1);
    float v = upper ? y : x;  // lanes 0 to 3 of a group of four: a, b, c, nothing
    v += __shfl_xor_sync(0xFFFFFFFFu, upper ? x : y, 2);
#pragma unroll
    for (int o = 4; o < 32; o *= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if constexpr (TEAM > 32) {
      constexpr int W = TEAM / 32;
      float* mine = reinterpret_cast<float*>(slots) + turn * (4 * W);
      turn ^= 1;
      if (lane < 4) mine[((int)(threadIdx.x >> 5) & (W - 1)) * 4 + lane] = v;
      if (TEAM >= 256)
        __syncthreads();
      else  // (a block has several teams)
        umma::named_barrier_sync(1 + threadIdx.x / TEAM, TEAM);
      v = mine[lane & (4 * W - 1)];
#pragma unroll
      for (int w = 32; w < 4 * W; w += 32) v += mine[w + lane];
#pragma unroll
      for (int o = 4; o < (W < 8 ? 4 * W : 32); o *= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    }
    return make_float3(__shfl_sync(0xFFFFFFFFu, v, 0), __shfl_sync(0xFFFFFFFFu, v, 1), __shfl_sync(0xFFFFFFFFu, v, 2));
  }
  __device__ __forceinline__ float one(float a) { return sum<1>(a, 0.f).x; }
  __device__ __forceinline__ float2 two(float a, float b) { return sum<2>(a, b); }
};

constexpr int block_of(int team) { return team < 256 ? 256 : team; }

// Mean and r of a row that a team holds; entries behind the row's end are zero and `live` says which are not.
template <int V, int NP, bool LAYER, typename Sum>
__device__ __forceinline__ void row_statistics(int kind, const float (&v)[NP][V], const bool (&live)[NP], float inv_channels,
                                               float epsilon, Sum& team_sum, float& mean, float& r) {
  mean = 0.f;
  r = 1.f;
  if (kind == PDNN_NORM_NONE) return;
  if (LAYER && kind == PDNN_NORM_LAYER) mean = team_sum.one(total<V, NP>(v)) * inv_channels;
  float squares;
  if constexpr (LAYER) {
    float d[NP][V];
#pragma unroll
    for (int p = 0; p < NP; ++p) add_mul<V>(d[p], v[p], live[p] ? -mean : 0.f, 1.f);  // (entries that are not live are zero)
    squares = dot<V, NP>(d, d);
  } else {
    squares = dot<V, NP>(v, v);
  }
  r = 1.f / sqrtf(team_sum.one(squares) * inv_channels + epsilon);
}

// Blocks to an SM that the kernels' registers are cut for, by the elements that a thread keeps of a tensor: forward 1024 threads of
// 64 registers, half as many with more than eight elements (layer norms: four); backward 512 threads of 128.
constexpr int forward_blocks(int team, int elements, bool layer) {
  const int threads = elements > 8 || (layer && elements > 4) ? 512 : 1024;
  return threads < block_of(team) ? 1 : threads / block_of(team);
}
constexpr int gradient_blocks(int team) { return team > 512 ? 1 : 512 / block_of(team); }

// LAYER: at least one of the norms is a layer norm, or there is a beta.
template <typename T, int V, int TEAM, int NP>
using ForwardRows = Incoming<T, V, NP, 2, 3, block_of(TEAM)>;
template <typename T, int V, int TEAM, int NP, bool LAYER>
__global__ void __launch_bounds__(block_of(TEAM), forward_blocks(TEAM, V * NP, LAYER)) residual_norm_kernel(const NormArgs a) {
  overlap_wait();
  extern __shared__ __align__(16) char rows_shared[];
  constexpr int kBlock = block_of(TEAM), kTeams = kBlock / TEAM;
  __shared__ float2 slots[2 * kBlock / 32];
  TeamSum<TEAM> team_sum{slots + (int)threadIdx.x / TEAM * (2 * TEAM / 32)};
  const int t = (int)threadIdx.x % TEAM;
  const long long team = (long long)blockIdx.x * kTeams + (int)threadIdx.x / TEAM, teams = (long long)gridDim.x * kTeams;
  const int first = (int)((long long)a.rows * team / teams), last = (int)((long long)a.rows * (team + 1) / teams);
  bool live[NP];
  int at[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    at[p] = (t + p * TEAM) * V;
    live[p] = at[p] < a.channels;
  }
  // by column: scale * act(gate) * gamma and * beta of the norm behind the block; gamma and beta of the one before the next
  float slope[NP][V], offset[NP][LAYER ? V : 1], pre_gamma[NP][V], pre_beta[NP][LAYER ? V : 1];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    Piece<T, V> g, b;
    if (live[p] && a.pre_gamma != nullptr) g.load(static_cast<const T*>(a.pre_gamma) + at[p]);
    if (LAYER && live[p] && a.pre_beta != nullptr) b.load(static_cast<const T*>(a.pre_beta) + at[p]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      pre_gamma[p][i] = a.pre_gamma == nullptr ? 1.f : live[p] ? g.get(i) : 0.f;
      if constexpr (LAYER) pre_beta[p][i] = a.pre_beta == nullptr || !live[p] ? 0.f : b.get(i);
    }
  }
  int group = -1;
  auto enter_group = [&](int to) {
    group = to;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      Piece<T, V> k, g, b;
      if (live[p] && a.gate != nullptr) k.load(static_cast<const T*>(a.gate) + (size_t)group * a.channels + at[p]);
      if (live[p] && a.post_gamma != nullptr) g.load(static_cast<const T*>(a.post_gamma) + at[p]);
      if (LAYER && live[p] && a.post_beta != nullptr) b.load(static_cast<const T*>(a.post_beta) + at[p]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v = a.scale;
        if (live[p] && a.gate != nullptr) v *= activate(a.gate_activation, k.get(i));
        if constexpr (LAYER) offset[p][i] = live[p] && a.post_beta != nullptr ? v * b.get(i) : 0.f;
        if (live[p] && a.post_gamma != nullptr) v *= g.get(i);
        slope[p][i] = live[p] ? v : 0.f;
      }
    }
  };

  using Rows = ForwardRows<T, V, TEAM, NP>;
  Rows incoming(rows_shared);
  const T* const from[2] = {static_cast<const T*>(a.branch), static_cast<const T*>(a.residual)};
  auto request = [&](int row, int into) { incoming.request(from, (size_t)row * a.channels, row < last, live, at, into); };
#pragma unroll
  for (int d = 0; d < Rows::kDepth; ++d) request(first + d, d);
  int group_ends = first;  // the first row of the next group
#pragma unroll 1
  for (int row = first; row < last; ++row) {
    if (row == group_ends) {
      enter_group(row / a.rows_per_group);
      group_ends = (group + 1) * a.rows_per_group;
    }
    float v[NP][V], x[NP][V];
    {
      Piece<T, V> in[2][NP];
      incoming.take(in);
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[p][i] = in[0][p].get(i);
          x[p][i] = in[1][p].get(i);
        }
    }
    if (!Rows::kSlots) request(row + Rows::kDepth, incoming.freed());
    float mean1, r1, mean2, r2;
    row_statistics<V, NP, LAYER>(a.post_norm, v, live, a.inv_channels, a.epsilon, team_sum, mean1, r1);
    if (Rows::kSlots) request(row + Rows::kDepth, incoming.freed());  // (what was in the slot has been used)
    const size_t base = (size_t)row * a.channels;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      if constexpr (LAYER) {
        add_mul<V>(v[p], v[p], -mean1, r1);  // (the slope of entries that are not live is zero)
        fma_all<V>(v[p], v[p], slope[p], offset[p]);
#pragma unroll
        for (int i = 0; i < V; ++i) v[p][i] += x[p][i];
      } else {
        mul_by<V>(v[p], v[p], r1);
        fma_all<V>(v[p], v[p], slope[p], x[p]);
      }
      if (live[p] && a.sum != nullptr) {
        Piece<T, V> s;
        s.round(v[p]);
        s.store(static_cast<T*>(a.sum) + base + at[p]);
      }
    }
    // (the statistics and the result are of the sum in 32 bits: the stored one is rounded once, and so is the result)
    row_statistics<V, NP, LAYER>(a.pre_norm, v, live, a.inv_channels, a.epsilon, team_sum, mean2, r2);
#pragma unroll
    for (int p = 0; p < NP; ++p)
      if (live[p] && a.out != nullptr) {
        Piece<T, V> o;
        if constexpr (LAYER) {
          add_mul<V>(v[p], v[p], -mean2, r2);
          fma_all<V>(v[p], v[p], pre_gamma[p], pre_beta[p]);
        } else {
          mul_by<V>(v[p], v[p], r2);
          mul_all<V>(v[p], v[p], pre_gamma[p]);
        }
        o.round(v[p]);
        o.store(static_cast<T*>(a.out) + base + at[p]);
      }
    if (t == 0 && a.statistics != nullptr) {
      a.statistics[row] = mean1;
      a.statistics[(size_t)a.rows + row] = r1;
      a.statistics[2 * (size_t)a.rows + row] = mean2;
      a.statistics[3 * (size_t)a.rows + row] = r2;
    }
  }
}

// What a thread that keeps no row does with V of its columns.
template <typename T, int V>
struct LongRow {
  const NormArgs& a;
  static __device__ __forceinline__ void load(const T* p, size_t at, float missing, float (&to)[V]) {
    Piece<T, V> v;
    if (p != nullptr) v.load(p + at);
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = p != nullptr ? v.get(i) : missing;
  }
  // scale * act(gate) of a group's columns
  __device__ __forceinline__ void gate(int group, int c, float (&raw)[V], float (&factor)[V]) const {
    load(a.gate != nullptr ? static_cast<const T*>(a.gate) + (size_t)group * a.channels : nullptr, c, 0.f, raw);
#pragma unroll
    for (int i = 0; i < V; ++i) factor[i] = a.scale;
    if (a.gate != nullptr)
      with_activation(a.gate_activation, [&](auto act) {  // (one way through the switch for all)
#pragma unroll
        for (int i = 0; i < V; ++i) factor[i] *= activate(decltype(act)::value, raw[i]);
      });
  }
  // the result's gradient g, u and hat of the norm before the next block
  __device__ __forceinline__ void before(size_t at, float mean, float r, const float (&gamma)[V], float (&g)[V], float (&u)[V], float (&hat)[V]) const {
    load(static_cast<const T*>(a.out_grad), at, 0.f, g);
    load(static_cast<const T*>(a.residual), at, 0.f, hat);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      u[i] = g[i] * gamma[i];
      hat[i] = (hat[i] - mean) * r;
    }
  }
  // the sum's gradient and hat of the norm behind the block
  __device__ __forceinline__ void behind(size_t at, float mean, float r, float r2, float a1, float a2, const float (&u)[V], const float (&hat)[V],
                                         float (&ds)[V], float (&f)[V]) const {
    load(static_cast<const T*>(a.sum_grad), at, 0.f, ds);
    load(static_cast<const T*>(a.branch), at, 0.f, f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      ds[i] += r2 * (u[i] - hat[i] * a1 - a2);
      f[i] = (f[i] - mean) * r;
    }
  }
};

constexpr int kLongThreads = 512;
constexpr int long_blocks(int v) { return v == 1 ? 4 : 3; }
// Rows that no team can keep: a block walks the row once for each sum and once more for the results (1000x20000 bf16 83 us, 1.9 TB/s:
// bound by the latency of its walks).
template <typename T, int V>
__global__ void __launch_bounds__(kLongThreads, long_blocks(V)) residual_norm_long_kernel(const NormArgs a) {
  overlap_wait();
  __shared__ float2 slots[2 * kLongThreads / 32];
  TeamSum<kLongThreads> team_sum{slots};
  const LongRow<T, V> long_row{a};
  const T *branch = static_cast<const T*>(a.branch), *residual = static_cast<const T*>(a.residual);
  for (int row = (int)blockIdx.x; row < a.rows; row += (int)gridDim.x) {
    const size_t base = (size_t)row * a.channels;
    float mean[2] = {0.f, 0.f}, r[2] = {1.f, 1.f};
    auto at_sum = [&](int c, float (&v)[V]) {  // V entries of the sum, in 32 bits
      float f[V], k[V], gamma[V], beta[V];
      long_row.load(branch, base + c, 0.f, f);
      long_row.load(residual, base + c, 0.f, v);
      long_row.gate(row / a.rows_per_group, c, gamma, k);
      long_row.load(static_cast<const T*>(a.post_gamma), c, 1.f, gamma);
      long_row.load(static_cast<const T*>(a.post_beta), c, 0.f, beta);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += k[i] * ((f[i] - mean[0]) * r[0] * gamma[i] + beta[i]);
    };
    for (int which = 0; which < 2; ++which) {
      const int kind = which == 0 ? a.post_norm : a.pre_norm;
      auto sum_of = [&](auto&& term) {
        float total = 0.f;
        for (int c = (int)threadIdx.x * V; c < a.channels; c += kLongThreads * V) {
          float v[V];
          if (which == 0)
            long_row.load(branch, base + c, 0.f, v);
          else
            at_sum(c, v);
#pragma unroll
          for (int i = 0; i < V; ++i) total += term(v[i]);
        }
        return team_sum.one(total) * a.inv_channels;
      };
      if (kind == PDNN_NORM_NONE) continue;
      float m = 0.f;
      if (kind == PDNN_NORM_LAYER) m = sum_of([](float v) { return v; });
      const float q = 1.f / sqrtf(sum_of([m](float v) { return (v - m) * (v - m); }) + a.epsilon);
      mean[which] = m;
      r[which] = q;
    }
    __syncthreads();  // (the results may take the place of the inputs)
    for (int c = (int)threadIdx.x * V; c < a.channels; c += kLongThreads * V) {
      float v[V];
      at_sum(c, v);
      Piece<T, V> s, o;
      float w[V], gamma[V], beta[V];
      long_row.load(static_cast<const T*>(a.pre_gamma), c, 1.f, gamma);
      long_row.load(static_cast<const T*>(a.pre_beta), c, 0.f, beta);
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = (v[i] - mean[1]) * r[1] * gamma[i] + beta[i];
      s.round(v);
      o.round(w);
      if (a.sum != nullptr) s.store(static_cast<T*>(a.sum) + base + c);
      if (a.out != nullptr) o.store(static_cast<T*>(a.out) + base + c);
    }
    if (threadIdx.x == 0 && a.statistics != nullptr)
      for (int i = 0; i < 2; ++i) {
        a.statistics[(size_t)(2 * i) * a.rows + row] = mean[i];
        a.statistics[(size_t)(2 * i + 1) * a.rows + row] = r[i];
      }
  }
}

// The stretch of rows that is unit `unit`: part `unit % parts` of group `unit / parts`.
__device__ __forceinline__ void unit_rows(const NormArgs& a, long long unit, int& group, int& part, int& first, int& last) {
  group = (int)(unit / a.parts);
  part = (int)(unit % a.parts);
  first = group * a.rows_per_group + (int)((long long)a.rows_per_group * part / a.parts);
  last = group * a.rows_per_group + (int)((long long)a.rows_per_group * (part + 1) / a.parts);
}

// LAYER: at least one of the norms is a layer norm, or there is a beta: gradients of beta, and sums of u.
// (One row at a time: with two, whose reductions lie side by side, the registers for them are missing - 8192x2048 bf16 48.7 -> 51.3
// us, 16384x1024 48 -> 70.  Bound by issue slots
// and a row's reductions: 16384x4096 bf16 5.9 TB/s, 8192x2048 with eight gates 48 us, 4.2 TB/s.  One reduction of three sums for two of one:
// 16384x4096 145.9 -> 137.6 us, 16384x1024 48.1 -> 45.5, 20000x512 34.5 -> 32.6, but 20000x100 19.5 -> 20.9.)
template <typename T, int V, int TEAM, int NP>
using BackwardRows = Incoming<T, V, NP, 4, 3, block_of(TEAM)>;
template <typename T, int V, int TEAM, int NP, bool LAYER>
__global__ void __launch_bounds__(block_of(TEAM), gradient_blocks(TEAM)) residual_norm_grad_kernel(const NormArgs a) {
  overlap_wait();
  extern __shared__ __align__(16) char rows_shared[];
  constexpr int kBlock = block_of(TEAM), kTeams = kBlock / TEAM, VL = LAYER ? V : 1;
  using Rows = BackwardRows<T, V, TEAM, NP>;
  __shared__ float2 slots[4 * kBlock / 32];
  TeamSum<TEAM> team_sum{slots + (int)threadIdx.x / TEAM * (4 * TEAM / 32)};
  const int t = (int)threadIdx.x % TEAM;
  const long long team = (long long)blockIdx.x * kTeams + (int)threadIdx.x / TEAM, teams = (long long)gridDim.x * kTeams;
  const int groups = a.rows / a.rows_per_group;
  const long long units = (long long)groups * a.parts;
  bool live[NP];
  int at[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    at[p] = (t + p * TEAM) * V;
    live[p] = at[p] < a.channels;
  }
  float pre_gamma[NP][V];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    Piece<T, V> g;
    if (live[p] && a.pre_gamma != nullptr) g.load(static_cast<const T*>(a.pre_gamma) + at[p]);
#pragma unroll
    for (int i = 0; i < V; ++i) pre_gamma[p][i] = a.pre_gamma == nullptr ? 1.f : live[p] ? g.get(i) : 0.f;
  }
  float d_pre_gamma[NP][V] = {}, d_pre_beta[NP][VL] = {};
  // the team's line of partial sums; the teams of a block leave theirs in shared memory, where the block adds them up
  float* line = a.partial == nullptr ? nullptr
                : kTeams > 1         ? reinterpret_cast<float*>(rows_shared + Rows::kSharedBytes) + ((int)threadIdx.x / TEAM) * a.line
                                     : a.partial + (size_t)team * a.line;
  if (kTeams > 1 && line != nullptr) {
    for (int c = t; c < (int)a.line; c += TEAM) line[c] = 0.f;
    __syncthreads();  // (other threads write what a stretch leaves)
  }
  Rows incoming(rows_shared);
  const T* const from[4] = {static_cast<const T*>(a.branch), static_cast<const T*>(a.residual), static_cast<const T*>(a.sum_grad),
                            static_cast<const T*>(a.out_grad)};

#pragma unroll 1
  for (long long unit = team; unit < units; unit += teams) {
    int group, part, first, last;
    unit_rows(a, unit, group, part, first, last);
    // by column: scale * act(gate) * gamma, what takes the sum's gradient to u; sums over the stretch's rows of ds * hat and ds
    float slope[NP][V], p_sum[NP][V] = {}, q_sum[NP][VL] = {};
    auto column = [&](int p, float (&gate)[V], float (&gamma)[V]) {
      Piece<T, V> k, g;
      if (live[p] && a.gate != nullptr) k.load(static_cast<const T*>(a.gate) + (size_t)group * a.channels + at[p]);
      if (live[p] && a.post_gamma != nullptr) g.load(static_cast<const T*>(a.post_gamma) + at[p]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        gate[i] = live[p] && a.gate != nullptr ? k.get(i) : 1.f;
        gamma[i] = live[p] && a.post_gamma != nullptr ? g.get(i) : 1.f;
      }
    };
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float gate[V], gamma[V];
      column(p, gate, gamma);
#pragma unroll
      for (int i = 0; i < V; ++i)
        slope[p][i] = live[p] ? a.scale * (a.gate != nullptr ? activate(a.gate_activation, gate[i]) : 1.f) * gamma[i] : 0.f;
    }
    float next_stats[4];
    auto request = [&](int row, int into) { incoming.request(from, (size_t)row * a.channels, row < last, live, at, into); };
    auto request_statistics = [&](int row) {
      if (row >= last) return;
#pragma unroll
      for (int i = 0; i < 4; ++i) next_stats[i] = a.statistics[(size_t)i * a.rows + row];
    };
    incoming.slot = 0;  // (every group of the stretch before has been waited for)
#pragma unroll
    for (int d = 0; d < Rows::kDepth; ++d) request(first + d, d);
    request_statistics(first);
#pragma unroll 1
    for (int row = first; row < last; ++row) {
      const float mean1 = next_stats[0], r1 = next_stats[1], mean2 = next_stats[2], r2 = next_stats[3];
      float u[NP][V], hat[NP][V], f[NP][V], ds[NP][V];
      float a1 = 0.f, a2 = 0.f;
      {
        Piece<T, V> in[4][NP];
        incoming.take(in);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          float g[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            f[p][i] = in[0][p].get(i);
            hat[p][i] = in[1][p].get(i);
            ds[p][i] = in[2][p].get(i);
            g[i] = in[3][p].get(i);
          }
          if constexpr (LAYER) {  // (u and the slope of entries that are not live are zero)
            add_mul<V>(hat[p], hat[p], -mean2, r2);
            add_mul<V>(f[p], f[p], -mean1, r1);
#pragma unroll
            for (int i = 0; i < V; ++i) d_pre_beta[p][i] += g[i];
          } else {
            mul_by<V>(hat[p], hat[p], r2);
            mul_by<V>(f[p], f[p], r1);
          }
          mul_all<V>(u[p], g, pre_gamma[p]);
          fma_all<V>(d_pre_gamma[p], g, hat[p], d_pre_gamma[p]);
        }
        a1 = dot<V, NP>(u, hat);
        if constexpr (LAYER) a2 = total<V, NP>(u);
      }
      float b1 = 0.f, b2 = 0.f;
      if constexpr (!LAYER) {
        // ds = ds0 - hat * r2 * a1 with ds0 = sum_grad + r2 * u, so b1 = mean(slope f ds) is mean(slope f ds0) - r2 * a1 * mean(slope
        // f hat): the row's three sums are taken at once.  (No more cancels than in ds itself.)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          float k[V];
#pragma unroll
          for (int i = 0; i < V; ++i) k[i] = r2;
          fma_all<V>(ds[p], u[p], k, ds[p]);
          mul_all<V>(u[p], slope[p], f[p]);
        }
        b1 = dot<V, NP>(u, ds);
        b2 = dot<V, NP>(u, hat);
      }
      if (!Rows::kSlots) request(row + Rows::kDepth, incoming.freed());
      request_statistics(row + 1);
      const size_t base = (size_t)row * a.channels;
      if constexpr (LAYER) {
        const float2 s = a.pre_norm != PDNN_NORM_NONE ? team_sum.two(a1, a2) : make_float2(0.f, 0.f);
        a1 = s.x * a.inv_channels;
        a2 = a.pre_norm == PDNN_NORM_LAYER ? s.y * a.inv_channels : 0.f;
      } else {
        float3 s = make_float3(0.f, 0.f, 0.f);
        if (a.pre_norm != PDNN_NORM_NONE || a.post_norm != PDNN_NORM_NONE) s = team_sum.three(a1, b1, b2);
        a1 = a.pre_norm != PDNN_NORM_NONE ? -r2 * (s.x * a.inv_channels) : 0.f;
        b1 = a.post_norm != PDNN_NORM_NONE ? fmaf(a1, s.z, s.y) * a.inv_channels : 0.f;
      }
      if (Rows::kSlots) request(row + Rows::kDepth, incoming.freed());  // (what was in the slot has been used)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        float k1[V], k2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          k1[i] = LAYER ? -a1 : a1;
          k2[i] = r2;
          if constexpr (LAYER) u[p][i] -= a2;
        }
        if constexpr (LAYER) {
          fma_all<V>(u[p], hat[p], k1, u[p]);
          fma_all<V>(ds[p], u[p], k2, ds[p]);
        } else {
          fma_all<V>(ds[p], hat[p], k1, ds[p]);
        }
        if (live[p] && a.residual_grad != nullptr) {
          Piece<T, V> o;
          o.round(ds[p]);
          o.store(static_cast<T*>(a.residual_grad) + base + at[p]);
        }
        fma_all<V>(p_sum[p], ds[p], f[p], p_sum[p]);
        mul_all<V>(u[p], ds[p], slope[p]);
        if constexpr (LAYER) {
#pragma unroll
          for (int i = 0; i < V; ++i) q_sum[p][i] += ds[p][i];
        }
      }
      if constexpr (LAYER) {
        float2 s = make_float2(0.f, 0.f);
        if (a.post_norm != PDNN_NORM_NONE) s = team_sum.two(dot<V, NP>(u, f), total<V, NP>(u));
        b1 = s.x * a.inv_channels;
        b2 = a.post_norm == PDNN_NORM_LAYER ? s.y * a.inv_channels : 0.f;
      }
#pragma unroll
      for (int p = 0; p < NP; ++p)
        if (live[p] && a.branch_grad != nullptr) {
          Piece<T, V> o;
          float k[V];
#pragma unroll
          for (int i = 0; i < V; ++i) k[i] = -b1;
          fma_all<V>(u[p], f[p], k, u[p]);
          if constexpr (LAYER) add_mul<V>(u[p], u[p], -b2, r1);
          else mul_by<V>(u[p], u[p], r1);
          o.round(u[p]);
          o.store(static_cast<T*>(a.branch_grad) + base + at[p]);
        }
    }
    // what the stretch's sums are worth
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float gate[V], gamma[V], d_gate[V];
      column(p, gate, gamma);
      Piece<T, V> b;
      if (LAYER && live[p] && a.post_beta != nullptr) b.load(static_cast<const T*>(a.post_beta) + at[p]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float k = a.scale * (a.gate != nullptr ? activate(a.gate_activation, gate[i]) : 1.f);
        // (the line takes the sums over a team's stretches, most often one: registers for them are needed elsewhere)
        if (live[p] && line != nullptr && a.slot[0] >= 0) {
          float* to = line + (size_t)a.slot[0] * a.channels + at[p] + i;
          *to = (unit == team ? 0.f : *to) + k * p_sum[p][i];
        }
        d_gate[i] = gamma[i] * p_sum[p][i];
        if constexpr (LAYER) {
          if (live[p] && line != nullptr && a.slot[1] >= 0) {
            float* to = line + (size_t)a.slot[1] * a.channels + at[p] + i;
            *to = (unit == team ? 0.f : *to) + k * q_sum[p][i];
          }
          if (live[p] && a.post_beta != nullptr) d_gate[i] += b.get(i) * q_sum[p][i];
        }
        d_gate[i] *= a.scale;
      }
      if (a.gate_grad == nullptr || !live[p]) continue;
      if (a.parts == 1) {
        Piece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) d_gate[i] *= activation_slope(a.gate_activation, gate[i]);
        o.round(d_gate);
        o.store(static_cast<T*>(a.gate_grad) + (size_t)group * a.channels + at[p]);
      } else {
        float* to = a.gate_vector >= 0 ? line + (size_t)a.gate_vector * a.channels + at[p]
                                       : a.gate_partial + ((size_t)part * groups + group) * a.channels + at[p];
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] = d_gate[i];
      }
    }
  }
  if (line == nullptr) return;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    if (!live[p]) continue;
    for (int which = 0; which < 2; ++which)  // a team without rows
      if (team >= units && a.slot[which] >= 0)
        for (int i = 0; i < V; ++i) line[(size_t)a.slot[which] * a.channels + at[p] + i] = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (a.slot[2] >= 0) line[(size_t)a.slot[2] * a.channels + at[p] + i] = d_pre_gamma[p][i];
      if constexpr (LAYER) {
        if (a.slot[3] >= 0) line[(size_t)a.slot[3] * a.channels + at[p] + i] = d_pre_beta[p][i];
      }
    }
  }
  if constexpr (kTeams > 1) {
    __syncthreads();
    const float* lines = reinterpret_cast<const float*>(rows_shared + Rows::kSharedBytes);
    for (int c = (int)threadIdx.x; c < (int)a.line; c += kBlock) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kTeams; ++w) sum += lines[w * a.line + c];
      a.partial[(size_t)blockIdx.x * a.line + c] = sum;
    }
  }
}

// Rows that no team can keep, in two launches: a block to a row for the four sums over it (row_sums, [4][rows]), then a thread to V
// columns, which walks down a stretch of rows with the parameters and their sums in registers.  Two reads of everything, the second
// one from L2 in part (us, a block to a row for it all, its sums over rows in memory / so: 1000x20000
// bf16 468 / 135, 1000x16384 f32 249 / 155, 1000x20001 bf16, by element, 549 / 373).
template <typename T, int V>
__global__ void __launch_bounds__(kLongThreads, 2) residual_norm_grad_rows_kernel(const NormArgs a) {
  overlap_wait();
  __shared__ float2 slots[2 * kLongThreads / 32];
  TeamSum<kLongThreads> team_sum{slots};
  const LongRow<T, V> long_row{a};
  for (int row = (int)blockIdx.x; row < a.rows; row += (int)gridDim.x) {
    const size_t base = (size_t)row * a.channels;
    float st[4];
    for (int i = 0; i < 4; ++i) st[i] = a.statistics[(size_t)i * a.rows + row];
    float2 s[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    for (int which = 0; which < 2; ++which) {
      const int kind = which == 0 ? a.pre_norm : a.post_norm;
      if (kind == PDNN_NORM_NONE) continue;
      float p = 0.f, q = 0.f;
      for (int c = (int)threadIdx.x * V; c < a.channels; c += kLongThreads * V) {
        float gamma[V], g[V], u[V], hat[V], f[V];
        long_row.load(static_cast<const T*>(a.pre_gamma), c, 1.f, gamma);
        long_row.before(base + c, st[2], st[3], gamma, g, u, hat);
        if (which == 0) {
#pragma unroll
          for (int i = 0; i < V; ++i) p += u[i] * hat[i], q += u[i];
        } else {
          long_row.behind(base + c, st[0], st[1], st[3], s[0].x, s[0].y, u, hat, g, f);
          float raw[V];
          long_row.gate(row / a.rows_per_group, c, raw, hat);
          long_row.load(static_cast<const T*>(a.post_gamma), c, 1.f, gamma);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float v = g[i] * hat[i] * gamma[i];
            p += v * f[i];
            q += v;
          }
        }
      }
      s[which] = team_sum.two(p, q);
      s[which].x *= a.inv_channels;
      s[which].y = kind == PDNN_NORM_LAYER ? s[which].y * a.inv_channels : 0.f;
    }
    if (threadIdx.x == 0) {
      a.row_sums[row] = s[0].x;
      a.row_sums[(size_t)a.rows + row] = s[0].y;
      a.row_sums[2 * (size_t)a.rows + row] = s[1].x;
      a.row_sums[3 * (size_t)a.rows + row] = s[1].y;
    }
  }
}

constexpr int kColumnThreads = 128;
template <typename T, int V>
__global__ void __launch_bounds__(kColumnThreads, 4) residual_norm_grad_columns_kernel(const NormArgs a) {
  overlap_wait();
  const int c = ((int)blockIdx.x * kColumnThreads + (int)threadIdx.x) * V, groups = a.rows / a.rows_per_group;
  if (c >= a.channels) return;
  const LongRow<T, V> long_row{a};
  float pre_gamma[V], gamma[V], sums[4][V] = {};  // (of the gradients of post gamma, post beta, pre gamma, pre beta)
  long_row.load(static_cast<const T*>(a.pre_gamma), c, 1.f, pre_gamma);
  long_row.load(static_cast<const T*>(a.post_gamma), c, 1.f, gamma);
  float* line = a.partial != nullptr ? a.partial + (size_t)blockIdx.y * a.line + c : nullptr;
  for (long long unit = blockIdx.y; unit < (long long)groups * a.parts; unit += gridDim.y) {
    int group, part, first, last;
    unit_rows(a, unit, group, part, first, last);
    float raw[V], factor[V], p_sum[V] = {}, q_sum[V] = {};
    long_row.gate(group, c, raw, factor);
#pragma unroll 2
    for (int row = first; row < last; ++row) {
      float st[4], by[4], g[V], u[V], hat[V], ds[V], f[V];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st[i] = a.statistics[(size_t)i * a.rows + row];
        by[i] = a.row_sums[(size_t)i * a.rows + row];
      }
      const size_t at = (size_t)row * a.channels + c;
      long_row.before(at, st[2], st[3], pre_gamma, g, u, hat);
      long_row.behind(at, st[0], st[1], st[3], by[0], by[1], u, hat, ds, f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sums[2][i] += g[i] * hat[i];
        sums[3][i] += g[i];
        p_sum[i] += ds[i] * f[i];
        q_sum[i] += ds[i];
        u[i] = st[1] * (ds[i] * factor[i] * gamma[i] - f[i] * by[2] - by[3]);
      }
      Piece<T, V> o;
      if (a.residual_grad != nullptr) {
        o.round(ds);
        o.store(static_cast<T*>(a.residual_grad) + at);
      }
      if (a.branch_grad != nullptr) {
        o.round(u);
        o.store(static_cast<T*>(a.branch_grad) + at);
      }
    }
    float beta[V];
    long_row.load(static_cast<const T*>(a.post_beta), c, 0.f, beta);
    float* gate_line = a.gate_vector >= 0        ? line + (size_t)a.gate_vector * a.channels
                       : a.gate_partial != nullptr ? a.gate_partial + ((size_t)part * groups + group) * a.channels + c : nullptr;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sums[0][i] += factor[i] * p_sum[i];
      sums[1][i] += factor[i] * q_sum[i];
      if (gate_line != nullptr) gate_line[i] = a.scale * (gamma[i] * p_sum[i] + beta[i] * q_sum[i]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (a.slot[k] >= 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) line[(size_t)a.slot[k] * a.channels + i] = sums[k][i];
    }
}

// ---- the second stage: the blocks' lines, and the gate's parts, added up in a fixed order, both in one launch --------------
template <typename T>
struct SumArgs {
  const float *lines, *gates;  // [blocks][line], [parts][gate_entries]
  size_t line, gate_entries;
  int blocks, parts, channels, gate_vector, activation;
  T* to[5];  // vectors of a line
  const T* gate;
  T* gate_grad;
};

// 32 columns to a block, sixteen threads to a column with LOADS loads in flight each (the matrices are in L2: bound by latency.
// 8192x2048 bf16, eight groups, whole gradient, sixteen / 32 threads: 48.4 / 50.9 us).  Twenty loads, so that two blocks' lines to an
// SM are one walk, where the columns are one wave of blocks, eight otherwise (whole gradients, eight / twenty: 1999x1003 f32 23.3 /
// 21.2 us, 16384x1024 bf16 45.2 / 43.1; 640 blocks, 8192x2048 with eight groups 47.9 / 49.5; few lines, 300x4096 20.8 / 21.5).
constexpr int kSumLanes = 16;
template <typename T, int LOADS>
__global__ void __launch_bounds__(32 * kSumLanes) residual_norm_sums_kernel(const SumArgs<T> a) {
  overlap_wait();
  __shared__ float red[kSumLanes][33];
  const unsigned line_tiles = (unsigned)((a.line + 31) / 32);
  const bool gates = blockIdx.x >= line_tiles;
  const float* m = gates ? a.gates : a.lines;
  const size_t n = gates ? a.gate_entries : a.line, first = (size_t)(gates ? blockIdx.x - line_tiles : blockIdx.x) * 32;
  const int rows = gates ? a.parts : a.blocks, tx = (int)threadIdx.x & 31, ty = (int)threadIdx.x >> 5;
  float sum = 0.f;
  if (first + tx < n)
    for (int r = ty; r < rows; r += kSumLanes * LOADS) {
      float v[LOADS];
#pragma unroll
      for (int u = 0; u < LOADS; ++u) v[u] = r + u * kSumLanes < rows ? m[(size_t)(r + u * kSumLanes) * n + first + tx] : 0.f;
#pragma unroll
      for (int u = 0; u < LOADS; ++u) sum += v[u];
    }
  red[ty][tx] = sum;
  __syncthreads();
  // kSumLanes neighbouring threads add the lanes of a column
  const int col = (int)threadIdx.x / kSumLanes;
  float v = red[(int)threadIdx.x % kSumLanes][col];
#pragma unroll
  for (int o = kSumLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  const size_t i = first + col;
  if ((int)threadIdx.x % kSumLanes != 0 || i >= n) return;
  if (gates) {
    a.gate_grad[i] = from_f32<T>(v * activation_slope(a.activation, to_f32(a.gate[i])));
    return;
  }
  const int which = (int)(i / a.channels), c = (int)(i - (size_t)which * a.channels);
  if (which == a.gate_vector) v *= activation_slope(a.activation, to_f32(a.gate[c]));
  T* p = a.to[0];
#pragma unroll
  for (int k = 1; k < 5; ++k)
    if (which == k) p = a.to[k];
  p[c] = from_f32<T>(v);
}

template <typename F>
int dispatch(int dtype, F&& f) {
  switch (dtype) {
    case PDNN_F32: return f(float{});
    case PDNN_F16: return f(__half{});
    case PDNN_BF16: return f(__nv_bfloat16{});
  }
  return fail(PDNN_INVALID_PARAMETER, "residual norm: unknown dtype %d", dtype);
}

template <int TEAM, int NP>
struct Shape {
  static constexpr int team = TEAM, np = NP;
};

// The smallest team that keeps a row of `pieces` packets (PACKETS) or smaller pieces; 0 where none does.  LONG: of packets of
// four or single elements a thread keeps more.  TWO: two packets to a thread, and registers for them, which pays for layer
// norms forward (us, one / two: 8192x4096 bf16 layer and rms norm 74.8 / 59.2, both rms 16384x4096 91.5 / 103.2).
template <bool PACKETS, bool LONG, bool TWO, typename F>
int with_shape(int pieces, F&& f) {
  if constexpr (PACKETS && TWO) {
    if (pieces <= 32) return f(Shape<32, 1>{});
    if (pieces <= 64) return f(Shape<32, 2>{});
    if (pieces <= 128) return f(Shape<64, 2>{});
    if (pieces <= 256) return f(Shape<128, 2>{});
    if (pieces <= 512) return f(Shape<256, 2>{});
    if (pieces <= 1024) return f(Shape<512, 2>{});
    if constexpr (LONG) {
      if (pieces <= 2048) return f(Shape<1024, 2>{});
    }
  } else if constexpr (PACKETS) {
    if (pieces <= 32) return f(Shape<32, 1>{});
    if (pieces <= 64) return f(Shape<64, 1>{});
    if (pieces <= 128) return f(Shape<128, 1>{});
    if (pieces <= 256) return f(Shape<256, 1>{});
    if (pieces <= 512) return f(Shape<512, 1>{});
    if (pieces <= 1024) return f(Shape<512, 2>{});
    if constexpr (LONG) {
      if (pieces <= 2048) return f(Shape<1024, 2>{});
    }
  } else {
    // (eight single elements to a thread: 1999x1003 f32 gradient 22 -> 32 us, half as many loads on their way)
    if (pieces <= 128) return f(Shape<32, 4>{});
    if (pieces <= 512) return f(Shape<128, 4>{});
    if (pieces <= 1024) return f(Shape<256, 4>{});
    if (pieces <= 2048) return f(Shape<512, 4>{});
    if constexpr (LONG) {
      if (pieces <= 4096) return f(Shape<512, 8>{});
    }
  }
  return 0;
}
template <typename T, bool TWO, typename F>
int with_pieces(int width, int channels, F&& f) {
  constexpr int N = Vec16<T>::N;
  if (width == N) return with_shape<true, N == 4, TWO>(channels / N, [&](auto shape) { return f(std::integral_constant<int, N>{}, shape); });
  if constexpr (N == 8) {
    if (width == 2) return with_shape<false, false, TWO>(channels / 2, [&](auto shape) { return f(std::integral_constant<int, 2>{}, shape); });
  }
  return with_shape<false, true, TWO>(channels, [&](auto shape) { return f(std::integral_constant<int, 1>{}, shape); });
}
// Elements to a load: a packet, a pair of 16-bit elements or one, by the channels and what all tensors' addresses are multiples of.
template <typename T>
int piece_width(int channels, std::initializer_list<const void*> list) {
  uintptr_t low = 0;
  for (const void* p : list) low |= reinterpret_cast<uintptr_t>(p);
  if (channels % Vec16<T>::N == 0 && low % 16 == 0) return Vec16<T>::N;
  return sizeof(T) == 2 && channels % 2 == 0 && channels <= 4096 && low % 4 == 0 ? 2 : 1;
}

constexpr int kMostShared = 224 * 1024;
// As launch_overlapped, with dynamic shared memory, much of it by opting in (once for a kernel and device).
void launch_rows(void (*kernel)(NormArgs), unsigned grid, unsigned block, int shared, const NormArgs& a, cudaStream_t s) {
  if (shared > 40 * 1024) {  // (the kernels' own few slots come on top)
    struct Entry {
      void (*kernel)(NormArgs);
      int device;
    };
    static std::mutex mu;
    static Entry known[256];
    static int count = 0;
    const int device = current_device();
    std::lock_guard<std::mutex> lock(mu);
    bool found = false;
    for (int i = 0; i < count; ++i) found = found || (known[i].kernel == kernel && known[i].device == device);
    if (!found) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) return;  // (check_launch reads the error)
      if (count < 256) known[count++] = Entry{kernel, device};
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = (size_t)shared;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;  // (a grid is one wave at most)
  cudaLaunchKernelEx(&cfg, kernel, a);  // (the caller's check_launch() reads the error)
}

int check_params(const char* what, int dtype, const PdnnResidualNormParams& p) {
  if (dtype < PDNN_F32 || dtype > PDNN_BF16) return fail(PDNN_INVALID_PARAMETER, "%s: unknown dtype %d", what, dtype);
  if (p.rows < 0 || p.channels <= 0) return fail(PDNN_INVALID_PARAMETER, "%s: %d rows of %d channels", what, p.rows, p.channels);
  if (p.rows > 0x7FFF0000 || p.channels > 0x7FFF0000)  // (kernels count a little past them)
    return fail(PDNN_INVALID_PARAMETER, "%s: %d rows of %d channels are too many", what, p.rows, p.channels);
  for (int kind : {p.post_norm, p.pre_norm})
    if (kind < PDNN_NORM_NONE || kind > PDNN_NORM_LAYER) return fail(PDNN_INVALID_PARAMETER, "%s: unknown norm %d", what, kind);
  if (p.gate_groups < 0 || (p.gate_groups > 0 && p.rows % p.gate_groups != 0))
    return fail(PDNN_INVALID_PARAMETER, "%s: %d rows do not make %d groups", what, p.rows, p.gate_groups);
  if (!known_activation(p.gate_activation))
    return fail(PDNN_INVALID_PARAMETER, "%s: unknown activation %d", what, p.gate_activation);
  if (!(p.epsilon >= 0.f)) return fail(PDNN_INVALID_PARAMETER, "%s: epsilon must not be negative", what);
  return PDNN_OK;
}

Extent whole(int dtype, const PdnnResidualNormParams& p, const void* t) {
  return Extent{t, p.rows > 0 ? 1 : 0, (long long)p.rows * p.channels * (long long)dtype_size(dtype), (long long)p.rows * p.channels * (long long)dtype_size(dtype)};
}
// Whether two tensors of all rows share bytes without being the same one.
bool partly(int dtype, const PdnnResidualNormParams& p, const void* a, const void* b) {
  return a != b && overlap(whole(dtype, p, a), whole(dtype, p, b));
}

// Whether a result of all rows lies on a vector that other rows still read.
bool on_vectors(int dtype, const PdnnResidualNormParams& p, const PdnnResidualNormTensors& t, const void* written) {
  const long long row = (long long)p.channels * (long long)dtype_size(dtype);
  const Extent result = whole(dtype, p, written);
  for (const void* v : {t.post_gamma, t.post_beta, t.pre_gamma, t.pre_beta})
    if (overlap(result, Extent{v, 1, row, row})) return true;
  return overlap(result, Extent{t.gate, 1, row * p.gate_groups, row * p.gate_groups});
}

NormArgs make_args(const PdnnResidualNormParams& p) {
  NormArgs a;
  std::memset(&a, 0, sizeof(a));
  a.rows = p.rows;
  a.channels = p.channels;
  a.post_norm = p.post_norm;
  a.pre_norm = p.pre_norm;
  a.gate_groups = p.gate_groups;
  a.gate_activation = p.gate_activation;
  a.rows_per_group = p.gate_groups > 0 ? std::max(p.rows / p.gate_groups, 1) : std::max(p.rows, 1);
  a.scale = p.scale;
  a.epsilon = p.epsilon;
  a.inv_channels = 1.f / (float)p.channels;
  return a;
}

}  // namespace

int launch_residual_norm(int dtype, const PdnnResidualNormParams& p, const PdnnResidualNormTensors& t, cudaStream_t s) {
  const char* what = "residual norm";
  int st = check_params(what, dtype, p);
  if (st != PDNN_OK) return st;
  if ((t.gate != nullptr) != (p.gate_groups > 0) && p.rows > 0)
    return fail(PDNN_INVALID_PARAMETER, "%s: a gate and its groups belong together", what);
  if (p.rows > 0 && (t.branch == nullptr || (t.sum == nullptr && t.output == nullptr)))
    return fail(PDNN_INVALID_PARAMETER, "%s: null tensor", what);
  for (const void* written : {(const void*)t.sum, (const void*)t.output})
    for (const void* read : {t.branch, t.residual})
      if (partly(dtype, p, written, read)) return fail(PDNN_INVALID_PARAMETER, "%s: a result lies across an input", what);
  if (on_vectors(dtype, p, t, t.sum) || on_vectors(dtype, p, t, t.output)) return fail(PDNN_INVALID_PARAMETER, "%s: a result lies on a vector", what);
  if (overlap(whole(dtype, p, t.sum), whole(dtype, p, t.output))) return fail(PDNN_INVALID_PARAMETER, "%s: the results lie on one another", what);
  const int sms = device_sm_count();
  if (sms <= 0) return fail(PDNN_ALLOCATION_PROBLEM, "%s: no sm_100 CUDA device", what);
  if (p.rows == 0) return PDNN_OK;
  NormArgs a = make_args(p);
  a.branch = t.branch;
  a.residual = t.residual;
  a.post_gamma = t.post_gamma;
  a.post_beta = t.post_beta;
  a.gate = t.gate;
  a.pre_gamma = t.pre_gamma;
  a.pre_beta = t.pre_beta;
  a.sum = t.sum;
  a.out = t.output;
  a.statistics = t.statistics;
  const bool layer = p.post_norm == PDNN_NORM_LAYER || p.pre_norm == PDNN_NORM_LAYER || t.post_beta != nullptr || t.pre_beta != nullptr;
  return dispatch(dtype, [&](auto type) {
    using T = decltype(type);
    const int width = piece_width<T>(p.channels, {t.branch, t.residual, t.post_gamma, t.post_beta, t.gate, t.pre_gamma, t.pre_beta,
                                                 t.sum, t.output});
    auto run = [&](auto layered, auto elements, auto shape) {
      constexpr bool LAYER = decltype(layered)::value;
      constexpr int V = decltype(elements)::value, TEAM = decltype(shape)::team, NP = decltype(shape)::np, kTeams = block_of(TEAM) / TEAM;
      // one wave, with a row or more to each team
      const long long wave = (long long)sms * forward_blocks(TEAM, V * NP, LAYER);
      const unsigned grid = (unsigned)std::min<long long>(wave, ((long long)p.rows + kTeams - 1) / kTeams);
      launch_rows(residual_norm_kernel<T, V, TEAM, NP, LAYER>, grid, block_of(TEAM), ForwardRows<T, V, TEAM, NP>::kSharedBytes, a, s);
      return 1;
    };
    const int known =
        layer ? with_pieces<T, true>(width, p.channels, [&](auto elements, auto shape) { return run(std::true_type{}, elements, shape); })
              : with_pieces<T, false>(width, p.channels, [&](auto elements, auto shape) { return run(std::false_type{}, elements, shape); });
    if (known == 0) {
      const unsigned grid = (unsigned)std::min(p.rows, long_blocks(width) * sms);
      if (width == Vec16<T>::N)
        launch_overlapped(residual_norm_long_kernel<T, Vec16<T>::N>, grid, kLongThreads, s, a);
      else
        launch_overlapped(residual_norm_long_kernel<T, 1>, grid, kLongThreads, s, a);
    }
    return check_launch(what);
  });
}

int launch_residual_norm_gradient(int dtype, const PdnnResidualNormParams& p, const PdnnResidualNormTensors& t,
                                  const PdnnResidualNormGradients& g, cudaStream_t s) {
  const char* what = "residual norm gradient";
  int st = check_params(what, dtype, p);
  if (st != PDNN_OK) return st;
  if ((t.gate != nullptr) != (p.gate_groups > 0) && p.rows > 0)
    return fail(PDNN_INVALID_PARAMETER, "%s: a gate and its groups belong together", what);
  if (p.rows > 0 && (t.branch == nullptr || t.sum == nullptr || t.statistics == nullptr || g.output_grad == nullptr))
    return fail(PDNN_INVALID_PARAMETER, "%s: null tensor", what);
  if (g.gate_grad != nullptr && p.gate_groups == 0) return fail(PDNN_INVALID_PARAMETER, "%s: there is no gate", what);
  for (const void* written : {(const void*)g.branch_grad, (const void*)g.residual_grad})
    for (const void* read : {t.branch, (const void*)t.sum, g.sum_grad, g.output_grad})
      if (partly(dtype, p, written, read)) return fail(PDNN_INVALID_PARAMETER, "%s: a result lies across an input", what);
  if (on_vectors(dtype, p, t, g.branch_grad) || on_vectors(dtype, p, t, g.residual_grad))
    return fail(PDNN_INVALID_PARAMETER, "%s: a result lies on a vector", what);
  if (overlap(whole(dtype, p, g.branch_grad), whole(dtype, p, g.residual_grad)))
    return fail(PDNN_INVALID_PARAMETER, "%s: the results lie on one another", what);
  const int sms = device_sm_count();
  if (sms <= 0) return fail(PDNN_ALLOCATION_PROBLEM, "%s: no sm_100 CUDA device", what);
  NormArgs a = make_args(p);
  void* const vectors[4] = {g.post_gamma_grad, g.post_beta_grad, g.pre_gamma_grad, g.pre_beta_grad};
  if (p.rows == 0) {  // sums over no rows
    const size_t bytes = (size_t)p.channels * dtype_size(dtype);
    for (void* v : vectors)
      if (v != nullptr && cudaMemsetAsync(v, 0, bytes, s) != cudaSuccess) return check_launch(what);
    if (g.gate_grad != nullptr && cudaMemsetAsync(g.gate_grad, 0, bytes * p.gate_groups, s) != cudaSuccess) return check_launch(what);
    return PDNN_OK;
  }
  a.branch = t.branch;
  a.residual = t.sum;
  a.post_gamma = t.post_gamma;
  a.post_beta = t.post_beta;
  a.gate = t.gate;
  a.pre_gamma = t.pre_gamma;
  a.pre_beta = t.pre_beta;
  a.statistics = t.statistics;
  a.sum_grad = g.sum_grad;
  a.out_grad = g.output_grad;
  a.branch_grad = g.branch_grad;
  a.residual_grad = g.residual_grad;
  a.gate_grad = g.gate_grad;
  for (int i = 0; i < 4; ++i) a.slot[i] = vectors[i] != nullptr ? a.vectors++ : -1;
  const bool layer = p.post_norm == PDNN_NORM_LAYER || p.pre_norm == PDNN_NORM_LAYER || g.post_beta_grad != nullptr ||
                     g.pre_beta_grad != nullptr || t.post_beta != nullptr;
  return dispatch(dtype, [&](auto type) {
    using T = decltype(type);
    const int width = piece_width<T>(p.channels, {t.branch, t.sum, t.post_gamma, t.post_beta, t.gate, t.pre_gamma, g.sum_grad,
                                                 g.output_grad, g.branch_grad, g.residual_grad, g.gate_grad});
    const int groups = p.rows / a.rows_per_group;
    // The cut of the groups for at most `wave` teams (of which a block has `to_block`), and scratch for what the blocks leave.
    // Returns the blocks, 0 where there is no scratch.
    void* scratch = nullptr;
    size_t more = 0;  // floats for the rows' sums
    long long blocks = 0;
    auto plan = [&](long long wave, int to_block, bool direct) {
      a.parts = (int)std::max<long long>(1, std::min<long long>(wave / groups, a.rows_per_group));
      blocks = (std::min<long long>(wave, (long long)groups * a.parts) + to_block - 1) / to_block;
      const bool gates = g.gate_grad != nullptr && !(direct && a.parts == 1);
      a.gate_vector = gates && groups == 1 ? a.vectors : -1;
      a.line = (size_t)(a.vectors + (a.gate_vector >= 0 ? 1 : 0)) * p.channels;
      const size_t lines = (size_t)blocks * a.line, apart = gates && groups > 1 ? (size_t)groups * a.parts * p.channels : 0;
      if (lines + apart + more > 0) {
        if (cudaMallocAsync(&scratch, (lines + apart + more) * sizeof(float), s) != cudaSuccess) {
          cudaGetLastError();
          scratch = nullptr;
          return 0u;
        }
        a.partial = lines > 0 ? static_cast<float*>(scratch) : nullptr;
        a.gate_partial = apart > 0 ? static_cast<float*>(scratch) + lines : nullptr;
        a.row_sums = static_cast<float*>(scratch) + lines + apart;
      }
      return (unsigned)blocks;
    };
    unsigned grid = 0;
    const int known = with_pieces<T, false>(width, p.channels, [&](auto elements, auto shape) {
      constexpr int V = decltype(elements)::value, TEAM = decltype(shape)::team, NP = decltype(shape)::np;
      constexpr int kThreads = block_of(TEAM), kTeams = kThreads / TEAM;
      const long long wave = std::min<long long>((long long)sms * gradient_blocks(TEAM) * kTeams, p.rows);
      grid = plan(wave, kTeams, true);
      if (grid == 0) return 1;
      const int shared = BackwardRows<T, V, TEAM, NP>::kSharedBytes + (kTeams > 1 ? (int)(kTeams * a.line * sizeof(float)) : 0);
      launch_rows(layer ? residual_norm_grad_kernel<T, V, TEAM, NP, true> : residual_norm_grad_kernel<T, V, TEAM, NP, false>, grid,
                  kThreads, shared, a, s);
      return 1;
    });
    if (known == 0) {
      auto run = [&](auto elements) {
        constexpr int V = decltype(elements)::value;
        const int tiles = (p.channels + kColumnThreads * V - 1) / (kColumnThreads * V);
        // (a wave of blocks; a grid's second dimension ends at 65535)
        more = 4 * (size_t)p.rows;
        grid = plan(std::min<long long>(p.rows, std::max(1, 4 * sms / tiles)), 1, false);
        if (grid == 0) return;
        launch_overlapped(residual_norm_grad_rows_kernel<T, V>, (unsigned)std::min(p.rows, 4 * sms), kLongThreads, s, a);
        launch_overlapped(residual_norm_grad_columns_kernel<T, V>, dim3((unsigned)tiles, grid), kColumnThreads, s, a);
      };
      if (width == Vec16<T>::N)
        run(std::integral_constant<int, Vec16<T>::N>{});
      else
        run(std::integral_constant<int, 1>{});
    }
    if (grid == 0) return fail(PDNN_ALLOCATION_PROBLEM, "%s: cannot allocate scratch", what);
    int status = check_launch(what);
    if (status == PDNN_OK && (a.partial != nullptr || a.gate_partial != nullptr)) {
      SumArgs<T> sums = {};
      sums.lines = a.partial;
      sums.gates = a.gate_partial;
      sums.line = a.partial != nullptr ? a.line : 0;
      sums.gate_entries = a.gate_partial != nullptr ? (size_t)groups * p.channels : 0;
      sums.blocks = (int)blocks;
      sums.parts = a.parts;
      sums.channels = p.channels;
      sums.gate_vector = a.gate_vector;
      sums.activation = p.gate_activation;
      for (int i = 0; i < 4; ++i)
        if (a.slot[i] >= 0) sums.to[a.slot[i]] = static_cast<T*>(vectors[i]);
      if (a.gate_vector >= 0) sums.to[a.gate_vector] = static_cast<T*>(g.gate_grad);
      sums.gate = static_cast<const T*>(t.gate);
      sums.gate_grad = static_cast<T*>(g.gate_grad);
      const size_t tiles = (sums.line + 31) / 32 + (sums.gate_entries + 31) / 32;
      if (blocks > kSumLanes * 8 && tiles <= 2 * (size_t)sms)
        launch_overlapped(residual_norm_sums_kernel<T, 20>, dim3((unsigned)tiles), 32 * kSumLanes, s, sums);
      else
        launch_overlapped(residual_norm_sums_kernel<T, 8>, dim3((unsigned)tiles), 32 * kSumLanes, s, sums);
      status = check_launch(what);
    }
    if (scratch != nullptr) cudaFreeAsync(scratch, s);
    return status;
  });
}

}  // namespace pdnn
