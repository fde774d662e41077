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
// about the mean, in fp32 - cost no second read, and requests the next row before it reduces this one.  Teams keep to
// whole stretches of rows: gamma, beta and the gate stay in registers, and the sums over rows of the backward pass are
// the thread's own until its stretch ends.  They end in one line of partial sums a team, which column_sums.cuh
// adds in a fixed order.
#include "activation.cuh"
#include "column_sums.cuh"

#include <algorithm>
#include <cstring>
#include <initializer_list>

namespace pdnn {
namespace {

// V elements as a thread keeps them: a 16-byte packet or a single element.
template <typename T, int V>
struct Piece {
  Vec16<T> raw;
  __device__ __forceinline__ void load(const T* p) { raw = load16(p); }
  __device__ __forceinline__ float get(int i) const { return to_f32(raw.get(i)); }
  __device__ __forceinline__ void set(int i, float v) { raw.set(i, from_f32<T>(v)); }
  __device__ __forceinline__ void store(T* p) const { store16(p, raw); }
};
template <typename T>
struct Piece<T, 1> {
  T raw;
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ float get(int) const { return to_f32(raw); }
  __device__ __forceinline__ void set(int, float v) { raw = from_f32<T>(v); }
  __device__ __forceinline__ void store(T* p) const { *p = raw; }
};

struct NormArgs {
  const void *branch, *residual, *post_gamma, *post_beta, *gate, *pre_gamma, *pre_beta;
  void *sum, *out;
  float* statistics;  // [4][rows]: mean and r behind the block, mean and r before the next; may be null
  int rows, channels, post_norm, pre_norm, gate_groups, gate_activation, rows_per_group;
  float scale, epsilon, inv_channels;
  // backward
  const void *sum_grad, *out_grad;
  void *branch_grad, *residual_grad, *gate_grad;
  float *partial, *gate_partial;  // [teams][vectors][channels], [parts][groups][channels]
  int parts, vectors;             // stretches of rows that a group is cut into; parameter vectors with a gradient
  int slot[4];                    // where in a line of `partial` post gamma, post beta, pre gamma, pre beta are; -1: nowhere
};

// Sums over a team.  Teams of a warp need no barrier; others use two sets of slots in turn, so that one barrier a
// reduction is enough: whoever is about to write a set has passed the barrier behind everybody's last read of it.
template <int TEAM>
struct TeamSum {
  float2* slots;  // [2][TEAM / 32]
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
      b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    if constexpr (TEAM > 32) {
      constexpr int W = TEAM / 32;
      float2* mine = slots + turn * W;
      turn ^= 1;
      if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = make_float2(a, b);
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 v = mine[w];
        a += v.x;
        b += v.y;
      }
    }
    return make_float2(a, b);
  }
};

constexpr int block_of(int team) { return team == 32 ? 256 : team; }

// Mean and r of a row that a team holds; entries behind the row's end are zero and `live` says which are not.
template <int V, int NP, typename Sum>
__device__ __forceinline__ void row_statistics(int kind, const float (&v)[NP][V], const bool (&live)[NP], float inv_channels,
                                               float epsilon, Sum& team_sum, float& mean, float& r) {
  mean = 0.f;
  r = 1.f;
  if (kind == PDNN_NORM_NONE) return;
  if (kind == PDNN_NORM_LAYER) {
    float total = 0.f;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) total += v[p][i];
    mean = team_sum(total, 0.f).x * inv_channels;
  }
  float squares = 0.f;
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = v[p][i] - mean;
      if (live[p]) squares += d * d;
    }
  r = 1.f / sqrtf(team_sum(squares, 0.f).x * inv_channels + epsilon);
}

template <typename T, int V, int NP>
__device__ __forceinline__ void load_vector(const void* from, float fill, const bool (&live)[NP], const int (&at)[NP],
                                            Piece<T, V> (&to)[NP]) {
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    if (from != nullptr && live[p]) {
      to[p].load(static_cast<const T*>(from) + at[p]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) to[p].set(i, fill);
    }
  }
}

template <typename T, int V, int TEAM, int NP>
__global__ void __launch_bounds__(block_of(TEAM)) residual_norm_kernel(const NormArgs a) {
  overlap_wait();
  constexpr int kBlock = block_of(TEAM), kTeams = kBlock / TEAM;
  __shared__ float2 slots[2 * (TEAM > 32 ? TEAM / 32 : 1)];
  TeamSum<TEAM> team_sum{slots};
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
  Piece<T, V> post_gamma[NP], post_beta[NP], pre_gamma[NP], pre_beta[NP];
  load_vector<T, V, NP>(a.post_gamma, 1.f, live, at, post_gamma);
  load_vector<T, V, NP>(a.post_beta, 0.f, live, at, post_beta);
  load_vector<T, V, NP>(a.pre_gamma, 1.f, live, at, pre_gamma);
  load_vector<T, V, NP>(a.pre_beta, 0.f, live, at, pre_beta);
  float gate[NP][V];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < V; ++i) gate[p][i] = a.scale;
  int group = -1;

  const T *branch = static_cast<const T*>(a.branch), *residual = static_cast<const T*>(a.residual);
  Piece<T, V> next_f[NP], next_x[NP];
  auto request = [&](int row) {
    const size_t base = (size_t)row * a.channels;
#pragma unroll
    for (int p = 0; p < NP; ++p)
      if (live[p]) {
        next_f[p].load(branch + base + at[p]);
        if (residual != nullptr) next_x[p].load(residual + base + at[p]);
      }
  };
  if (first < last) request(first);
  for (int row = first; row < last; ++row) {
    float v[NP][V], x[NP][V];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[p][i] = live[p] ? next_f[p].get(i) : 0.f;
        x[p][i] = live[p] && residual != nullptr ? next_x[p].get(i) : 0.f;
      }
    if (row + 1 < last) request(row + 1);
    if (a.gate != nullptr && row / a.rows_per_group != group) {
      group = row / a.rows_per_group;
#pragma unroll
      for (int p = 0; p < NP; ++p)
        if (live[p]) {
          Piece<T, V> g;
          g.load(static_cast<const T*>(a.gate) + (size_t)group * a.channels + at[p]);
#pragma unroll
          for (int i = 0; i < V; ++i) gate[p][i] = a.scale * activate(a.gate_activation, g.get(i));
        }
    }
    float mean1, r1, mean2, r2;
    row_statistics<V, NP>(a.post_norm, v, live, a.inv_channels, a.epsilon, team_sum, mean1, r1);
    const size_t base = (size_t)row * a.channels;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        v[p][i] = live[p] ? x[p][i] + gate[p][i] * ((v[p][i] - mean1) * r1 * post_gamma[p].get(i) + post_beta[p].get(i)) : 0.f;
      if (live[p] && a.sum != nullptr) {
        Piece<T, V> s;
#pragma unroll
        for (int i = 0; i < V; ++i) s.set(i, v[p][i]);
        s.store(static_cast<T*>(a.sum) + base + at[p]);
      }
    }
    // (the statistics and the result are of the sum in 32 bits: the stored one is rounded once, and so is the result)
    row_statistics<V, NP>(a.pre_norm, v, live, a.inv_channels, a.epsilon, team_sum, mean2, r2);
#pragma unroll
    for (int p = 0; p < NP; ++p)
      if (live[p] && a.out != nullptr) {
        Piece<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.set(i, (v[p][i] - mean2) * r2 * pre_gamma[p].get(i) + pre_beta[p].get(i));
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

// Rows that no team can keep: a block walks the row once for each sum and once more for the results.
template <typename T, int V>
__global__ void __launch_bounds__(1024) residual_norm_long_kernel(const NormArgs a) {
  overlap_wait();
  __shared__ float2 slots[64];
  TeamSum<1024> team_sum{slots};
  const T *branch = static_cast<const T*>(a.branch), *residual = static_cast<const T*>(a.residual);
  for (int row = (int)blockIdx.x; row < a.rows; row += (int)gridDim.x) {
    const size_t base = (size_t)row * a.channels;
    const T* gate = a.gate != nullptr ? static_cast<const T*>(a.gate) + (size_t)(row / a.rows_per_group) * a.channels : nullptr;
    float mean[2] = {0.f, 0.f}, r[2] = {1.f, 1.f};
    auto at_sum = [&](int c, float (&v)[V]) {  // V entries of the sum, in 32 bits
      Piece<T, V> f, x, g, pg, pb;
      f.load(branch + base + c);
      if (residual != nullptr) x.load(residual + base + c);
      if (gate != nullptr) g.load(gate + c);
      if (a.post_gamma != nullptr) pg.load(static_cast<const T*>(a.post_gamma) + c);
      if (a.post_beta != nullptr) pb.load(static_cast<const T*>(a.post_beta) + c);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float n = (f.get(i) - mean[0]) * r[0] * (a.post_gamma != nullptr ? pg.get(i) : 1.f) +
                        (a.post_beta != nullptr ? pb.get(i) : 0.f);
        const float k = gate != nullptr ? a.scale * activate(a.gate_activation, g.get(i)) : a.scale;
        v[i] = (residual != nullptr ? x.get(i) : 0.f) + k * n;
      }
    };
    for (int which = 0; which < 2; ++which) {
      const int kind = which == 0 ? a.post_norm : a.pre_norm;
      auto sum_of = [&](auto&& term) {
        float total = 0.f;
        for (int c = (int)threadIdx.x * V; c < a.channels; c += 1024 * V) {
          float v[V];
          if (which == 0) {
            Piece<T, V> f;
            f.load(branch + base + c);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = f.get(i);
          } else {
            at_sum(c, v);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) total += term(v[i]);
        }
        return team_sum(total, 0.f).x * a.inv_channels;
      };
      if (kind == PDNN_NORM_NONE) continue;
      float m = 0.f;
      if (kind == PDNN_NORM_LAYER) m = sum_of([](float v) { return v; });
      const float q = 1.f / sqrtf(sum_of([m](float v) { return (v - m) * (v - m); }) + a.epsilon);
      mean[which] = m;
      r[which] = q;
    }
    __syncthreads();  // (the results may take the place of the inputs)
    for (int c = (int)threadIdx.x * V; c < a.channels; c += 1024 * V) {
      float v[V];
      at_sum(c, v);
      Piece<T, V> s, o, pg, pb;
      if (a.pre_gamma != nullptr) pg.load(static_cast<const T*>(a.pre_gamma) + c);
      if (a.pre_beta != nullptr) pb.load(static_cast<const T*>(a.pre_beta) + c);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s.set(i, v[i]);
        o.set(i, (v[i] - mean[1]) * r[1] * (a.pre_gamma != nullptr ? pg.get(i) : 1.f) + (a.pre_beta != nullptr ? pb.get(i) : 0.f));
      }
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

// LAYER: at least one of the norms is a layer norm, so that there are gradients of beta and sums of u.
template <typename T, int V, int TEAM, int NP, bool LAYER>
__global__ void __launch_bounds__(block_of(TEAM)) residual_norm_grad_kernel(const NormArgs a) {
  overlap_wait();
  constexpr int kBlock = block_of(TEAM), kTeams = kBlock / TEAM;
  __shared__ float2 slots[2 * (TEAM > 32 ? TEAM / 32 : 1)];
  TeamSum<TEAM> team_sum{slots};
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
  Piece<T, V> post_gamma[NP], post_beta[NP], pre_gamma[NP];
  load_vector<T, V, NP>(a.post_gamma, 1.f, live, at, post_gamma);
  if constexpr (LAYER) load_vector<T, V, NP>(a.post_beta, 0.f, live, at, post_beta);
  load_vector<T, V, NP>(a.pre_gamma, 1.f, live, at, pre_gamma);
  float d_post_gamma[NP][V] = {}, d_pre_gamma[NP][V] = {}, d_post_beta[NP][V] = {}, d_pre_beta[NP][V] = {};
  const T *branch = static_cast<const T*>(a.branch), *sum = static_cast<const T*>(a.residual);
  const T *sum_grad = static_cast<const T*>(a.sum_grad), *out_grad = static_cast<const T*>(a.out_grad);

  for (long long unit = team; unit < units; unit += teams) {
    int group, part, first, last;
    unit_rows(a, unit, group, part, first, last);
    float gate[NP][V], d_gate[NP][V] = {};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      Piece<T, V> g;
      if (a.gate != nullptr && live[p]) g.load(static_cast<const T*>(a.gate) + (size_t)group * a.channels + at[p]);
#pragma unroll
      for (int i = 0; i < V; ++i) gate[p][i] = a.gate != nullptr && live[p] ? activate(a.gate_activation, g.get(i)) : 1.f;
    }
    Piece<T, V> next_f[NP], next_s[NP], next_ds[NP], next_do[NP];
    float next_stats[4];
    auto request = [&](int row) {
      const size_t base = (size_t)row * a.channels;
#pragma unroll
      for (int p = 0; p < NP; ++p)
        if (live[p]) {
          next_f[p].load(branch + base + at[p]);
          next_s[p].load(sum + base + at[p]);
          if (sum_grad != nullptr) next_ds[p].load(sum_grad + base + at[p]);
          next_do[p].load(out_grad + base + at[p]);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) next_stats[i] = a.statistics[(size_t)i * a.rows + row];
    };
    if (first < last) request(first);
    for (int row = first; row < last; ++row) {
      const float mean1 = next_stats[0], r1 = next_stats[1], mean2 = next_stats[2], r2 = next_stats[3];
      float u[NP][V], hat[NP][V], f[NP][V], ds[NP][V];
      float a1 = 0.f, a2 = 0.f;
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float g = live[p] ? next_do[p].get(i) : 0.f;
          hat[p][i] = live[p] ? (next_s[p].get(i) - mean2) * r2 : 0.f;
          f[p][i] = live[p] ? (next_f[p].get(i) - mean1) * r1 : 0.f;
          ds[p][i] = live[p] && sum_grad != nullptr ? next_ds[p].get(i) : 0.f;
          u[p][i] = g * pre_gamma[p].get(i);
          d_pre_gamma[p][i] += g * hat[p][i];
          if constexpr (LAYER) d_pre_beta[p][i] += g;
          a1 += u[p][i] * hat[p][i];
          if constexpr (LAYER) a2 += u[p][i];
        }
      if (row + 1 < last) request(row + 1);
      const size_t base = (size_t)row * a.channels;
      if (a.pre_norm != PDNN_NORM_NONE) {
        const float2 s = team_sum(a1, a2);
        a1 = s.x * a.inv_channels;
        a2 = LAYER && a.pre_norm == PDNN_NORM_LAYER ? s.y * a.inv_channels : 0.f;
      } else {
        a1 = a2 = 0.f;
      }
      float b1 = 0.f, b2 = 0.f;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
#pragma unroll
        for (int i = 0; i < V; ++i) ds[p][i] += r2 * (u[p][i] - hat[p][i] * a1 - a2);
        if (live[p] && a.residual_grad != nullptr) {
          Piece<T, V> o;
#pragma unroll
          for (int i = 0; i < V; ++i) o.set(i, ds[p][i]);
          o.store(static_cast<T*>(a.residual_grad) + base + at[p]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = ds[p][i] * a.scale;
          float n = f[p][i] * post_gamma[p].get(i);
          if constexpr (LAYER) n += post_beta[p].get(i);
          d_gate[p][i] += d * n;
          const float dn = d * gate[p][i];
          d_post_gamma[p][i] += dn * f[p][i];
          if constexpr (LAYER) d_post_beta[p][i] += dn;
          u[p][i] = live[p] ? dn * post_gamma[p].get(i) : 0.f;
          b1 += u[p][i] * f[p][i];
          if constexpr (LAYER) b2 += u[p][i];
        }
      }
      if (a.post_norm != PDNN_NORM_NONE) {
        const float2 s = team_sum(b1, b2);
        b1 = s.x * a.inv_channels;
        b2 = LAYER && a.post_norm == PDNN_NORM_LAYER ? s.y * a.inv_channels : 0.f;
      } else {
        b1 = b2 = 0.f;
      }
#pragma unroll
      for (int p = 0; p < NP; ++p)
        if (live[p] && a.branch_grad != nullptr) {
          Piece<T, V> o;
#pragma unroll
          for (int i = 0; i < V; ++i) o.set(i, r1 * (u[p][i] - f[p][i] * b1 - b2));
          o.store(static_cast<T*>(a.branch_grad) + base + at[p]);
        }
    }
    if (a.gate_grad != nullptr) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
        if (live[p]) {
          if (a.parts == 1) {
            Piece<T, V> g, o;
            g.load(static_cast<const T*>(a.gate) + (size_t)group * a.channels + at[p]);
#pragma unroll
            for (int i = 0; i < V; ++i) o.set(i, d_gate[p][i] * activation_slope(a.gate_activation, g.get(i)));
            o.store(static_cast<T*>(a.gate_grad) + (size_t)group * a.channels + at[p]);
          } else {
            float* to = a.gate_partial + ((size_t)part * groups + group) * a.channels + at[p];
#pragma unroll
            for (int i = 0; i < V; ++i) to[i] = d_gate[p][i];
          }
        }
    }
  }
  if (a.partial != nullptr) {
    float* line = a.partial + (size_t)team * a.vectors * a.channels;
#pragma unroll
    for (int p = 0; p < NP; ++p)
      if (live[p]) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (a.slot[0] >= 0) line[(size_t)a.slot[0] * a.channels + at[p] + i] = d_post_gamma[p][i];
          if (a.slot[2] >= 0) line[(size_t)a.slot[2] * a.channels + at[p] + i] = d_pre_gamma[p][i];
          if constexpr (LAYER) {
            if (a.slot[1] >= 0) line[(size_t)a.slot[1] * a.channels + at[p] + i] = d_post_beta[p][i];
            if (a.slot[3] >= 0) line[(size_t)a.slot[3] * a.channels + at[p] + i] = d_pre_beta[p][i];
          }
        }
      }
  }
}

// Rows that no team can keep: a block walks its row four times, and the partial sums over rows are lines in memory that
// the block adds to (nobody else touches them).
template <typename T>
__global__ void __launch_bounds__(1024) residual_norm_grad_long_kernel(const NormArgs a) {
  overlap_wait();
  __shared__ float2 slots[64];
  TeamSum<1024> team_sum{slots};
  const int groups = a.rows / a.rows_per_group;
  const long long units = (long long)groups * a.parts;
  const T *branch = static_cast<const T*>(a.branch), *sum = static_cast<const T*>(a.residual);
  const T *sum_grad = static_cast<const T*>(a.sum_grad), *out_grad = static_cast<const T*>(a.out_grad);
  float* line = a.partial != nullptr ? a.partial + (size_t)blockIdx.x * a.vectors * a.channels : nullptr;
  if (line != nullptr)
    for (int c = (int)threadIdx.x; c < a.channels; c += 1024)
      for (int k = 0; k < a.vectors; ++k) line[(size_t)k * a.channels + c] = 0.f;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    int group, part, first, last;
    unit_rows(a, unit, group, part, first, last);
    const T* gate = a.gate != nullptr ? static_cast<const T*>(a.gate) + (size_t)group * a.channels : nullptr;
    float* gate_line = a.gate_partial != nullptr ? a.gate_partial + ((size_t)part * groups + group) * a.channels : nullptr;
    if (gate_line != nullptr)
      for (int c = (int)threadIdx.x; c < a.channels; c += 1024) gate_line[c] = 0.f;
    for (int row = first; row < last; ++row) {
      const size_t base = (size_t)row * a.channels;
      float st[4];
      for (int i = 0; i < 4; ++i) st[i] = a.statistics[(size_t)i * a.rows + row];
      float a1 = 0.f, a2 = 0.f, b1 = 0.f, b2 = 0.f;
      // one element's way: gradient of the sum, of the normalised branch, and what the parameters receive
      struct Step { float ds, u, f, n, dn, g, hat; };
      auto step = [&](int c) {
        Step o;
        o.g = to_f32(out_grad[base + c]);
        o.hat = (to_f32(sum[base + c]) - st[2]) * st[3];
        const float u = o.g * (a.pre_gamma != nullptr ? to_f32(static_cast<const T*>(a.pre_gamma)[c]) : 1.f);
        o.ds = (sum_grad != nullptr ? to_f32(sum_grad[base + c]) : 0.f) + st[3] * (u - o.hat * a1 - a2);
        o.f = (to_f32(branch[base + c]) - st[0]) * st[1];
        const float gamma = a.post_gamma != nullptr ? to_f32(static_cast<const T*>(a.post_gamma)[c]) : 1.f;
        o.n = o.f * gamma + (a.post_beta != nullptr ? to_f32(static_cast<const T*>(a.post_beta)[c]) : 0.f);
        o.dn = o.ds * a.scale * (gate != nullptr ? activate(a.gate_activation, to_f32(gate[c])) : 1.f);
        o.u = o.dn * gamma;
        return o;
      };
      if (a.pre_norm != PDNN_NORM_NONE) {
        float p = 0.f, q = 0.f;
        for (int c = (int)threadIdx.x; c < a.channels; c += 1024) {
          const float g = to_f32(out_grad[base + c]) * (a.pre_gamma != nullptr ? to_f32(static_cast<const T*>(a.pre_gamma)[c]) : 1.f);
          p += g * ((to_f32(sum[base + c]) - st[2]) * st[3]);
          q += g;
        }
        const float2 s = team_sum(p, q);
        a1 = s.x * a.inv_channels;
        a2 = a.pre_norm == PDNN_NORM_LAYER ? s.y * a.inv_channels : 0.f;
      }
      if (a.post_norm != PDNN_NORM_NONE) {
        float p = 0.f, q = 0.f;
        for (int c = (int)threadIdx.x; c < a.channels; c += 1024) {
          const Step o = step(c);
          p += o.u * o.f;
          q += o.u;
        }
        const float2 s = team_sum(p, q);
        b1 = s.x * a.inv_channels;
        b2 = a.post_norm == PDNN_NORM_LAYER ? s.y * a.inv_channels : 0.f;
      }
      __syncthreads();  // (the results may take the place of the inputs)
      for (int c = (int)threadIdx.x; c < a.channels; c += 1024) {
        const Step o = step(c);
        if (a.residual_grad != nullptr) static_cast<T*>(a.residual_grad)[base + c] = from_f32<T>(o.ds);
        if (a.branch_grad != nullptr) static_cast<T*>(a.branch_grad)[base + c] = from_f32<T>(st[1] * (o.u - o.f * b1 - b2));
        if (line != nullptr) {
          const float add[4] = {o.dn * o.f, o.dn, o.g * o.hat, o.g};
          for (int k = 0; k < 4; ++k)
            if (a.slot[k] >= 0) line[(size_t)a.slot[k] * a.channels + c] += add[k];
        }
        if (gate_line != nullptr) gate_line[c] += o.ds * a.scale * o.n;
      }
    }
  }
}

// What becomes of the sums over rows.
template <typename T>
struct StoreVectors {
  T* to[4];
  int channels;
  __device__ __forceinline__ void operator()(size_t i, float sum) const {
    const int which = (int)(i / channels);
    to[which][i % channels] = from_f32<T>(sum);
  }
};
template <typename T>
struct StoreGate {
  T* to;
  const T* gate;
  int activation;
  __device__ __forceinline__ void operator()(size_t i, float sum) const {
    to[i] = from_f32<T>(sum * activation_slope(activation, to_f32(gate[i])));
  }
};

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

// The smallest team that keeps a row of `pieces` packets or elements; 0 where none does.
template <typename F>
int with_shape(bool packets, int pieces, F&& f) {
  if (packets) {
    if (pieces <= 32) return f(Shape<32, 1>{});
    if (pieces <= 64) return f(Shape<32, 2>{});
    if (pieces <= 128) return f(Shape<128, 1>{});
    if (pieces <= 256) return f(Shape<256, 1>{});
    if (pieces <= 512) return f(Shape<512, 1>{});
    if (pieces <= 1024) return f(Shape<512, 2>{});
    return 0;
  }
  if (pieces <= 128) return f(Shape<32, 4>{});
  if (pieces <= 512) return f(Shape<128, 4>{});
  if (pieces <= 1024) return f(Shape<256, 4>{});
  if (pieces <= 2048) return f(Shape<512, 4>{});
  if (pieces <= 4096) return f(Shape<512, 8>{});
  return 0;
}

int check_params(const char* what, int dtype, const PdnnResidualNormParams& p) {
  if (dtype < PDNN_F32 || dtype > PDNN_BF16) return fail(PDNN_INVALID_PARAMETER, "%s: unknown dtype %d", what, dtype);
  if (p.rows < 0 || p.channels <= 0) return fail(PDNN_INVALID_PARAMETER, "%s: %d rows of %d channels", what, p.rows, p.channels);
  for (int kind : {p.post_norm, p.pre_norm})
    if (kind < PDNN_NORM_NONE || kind > PDNN_NORM_LAYER) return fail(PDNN_INVALID_PARAMETER, "%s: unknown norm %d", what, kind);
  if (p.gate_groups < 0 || (p.gate_groups > 0 && p.rows % p.gate_groups != 0))
    return fail(PDNN_INVALID_PARAMETER, "%s: %d rows do not make %d groups", what, p.rows, p.gate_groups);
  if (!known_activation(p.gate_activation))
    return fail(PDNN_INVALID_PARAMETER, "%s: unknown activation %d", what, p.gate_activation);
  if (!(p.epsilon >= 0.f)) return fail(PDNN_INVALID_PARAMETER, "%s: epsilon must not be negative", what);
  return PDNN_OK;
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

bool all_aligned(std::initializer_list<const void*> list) {
  for (const void* p : list)
    if (!aligned16(p)) return false;
  return true;
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
  return dispatch(dtype, [&](auto type) {
    using T = decltype(type);
    constexpr int N = Vec16<T>::N;
    const bool packets = p.channels % N == 0 && all_aligned({t.branch, t.residual, t.post_gamma, t.post_beta, t.gate,
                                                             t.pre_gamma, t.pre_beta, t.sum, t.output});
    const int pieces = packets ? p.channels / N : p.channels;
    const int known = with_shape(packets, pieces, [&](auto shape) {
      constexpr int TEAM = decltype(shape)::team, NP = decltype(shape)::np, kTeams = block_of(TEAM) / TEAM;
      // (as many teams as the device holds at 64 registers a thread or so, with a row or more to each)
      const long long wave = (long long)sms * std::max(1024 / block_of(TEAM), 1);
      const unsigned grid = (unsigned)std::min<long long>(wave, ((long long)p.rows + kTeams - 1) / kTeams);
      if (packets)
        launch_overlapped(residual_norm_kernel<T, N, TEAM, NP>, grid, block_of(TEAM), s, a);
      else
        launch_overlapped(residual_norm_kernel<T, 1, TEAM, NP>, grid, block_of(TEAM), s, a);
      return 1;
    });
    if (known == 0) {
      const unsigned grid = (unsigned)std::min(p.rows, 2 * sms);
      if (packets)
        launch_overlapped(residual_norm_long_kernel<T, N>, grid, 1024, s, a);
      else
        launch_overlapped(residual_norm_long_kernel<T, 1>, grid, 1024, s, a);
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
    constexpr int N = Vec16<T>::N;
    const bool packets = p.channels % N == 0 &&
                         all_aligned({t.branch, t.sum, t.post_gamma, t.post_beta, t.gate, t.pre_gamma, g.sum_grad, g.output_grad,
                                      g.branch_grad, g.residual_grad, g.gate_grad});
    const int pieces = packets ? p.channels / N : p.channels, groups = p.rows / a.rows_per_group;
    // The cut of the groups for at most `wave` teams, and scratch for what the teams leave: a line to a team of the grid (of
    // which a block has `to_block`) and one to a group's part.  Returns the blocks, 0 where there is no scratch.
    void* scratch = nullptr;
    long long teams = 0;
    auto plan = [&](long long wave, int to_block, bool direct) {
      a.parts = (int)std::max<long long>(1, std::min<long long>(wave / groups, a.rows_per_group));
      const long long blocks = (std::min<long long>(wave, (long long)groups * a.parts) + to_block - 1) / to_block;
      teams = blocks * to_block;
      const size_t lines = a.vectors > 0 ? (size_t)teams * a.vectors * p.channels : 0;
      const size_t gates = g.gate_grad != nullptr && !(direct && a.parts == 1) ? (size_t)groups * a.parts * p.channels : 0;
      if (lines + gates > 0) {
        if (cudaMallocAsync(&scratch, (lines + gates) * sizeof(float), s) != cudaSuccess) {
          cudaGetLastError();
          scratch = nullptr;
          return 0u;
        }
        a.partial = lines > 0 ? static_cast<float*>(scratch) : nullptr;
        a.gate_partial = gates > 0 ? static_cast<float*>(scratch) + lines : nullptr;
      }
      return (unsigned)blocks;
    };
    unsigned grid = 0;
    const int known = with_shape(packets, pieces, [&](auto shape) {
      constexpr int TEAM = decltype(shape)::team, NP = decltype(shape)::np, kThreads = block_of(TEAM), kTeams = kThreads / TEAM;
      // One block of 512 threads to an SM (its sums and the next row take most of the registers), or as many threads.
      const long long wave = std::min<long long>((long long)sms * std::max(512 / kThreads, 1) * kTeams, p.rows);
      grid = plan(wave, kTeams, true);
      if (grid == 0) return 1;
      if (packets && layer)
        launch_overlapped(residual_norm_grad_kernel<T, N, TEAM, NP, true>, grid, kThreads, s, a);
      else if (packets)
        launch_overlapped(residual_norm_grad_kernel<T, N, TEAM, NP, false>, grid, kThreads, s, a);
      else if (layer)
        launch_overlapped(residual_norm_grad_kernel<T, 1, TEAM, NP, true>, grid, kThreads, s, a);
      else
        launch_overlapped(residual_norm_grad_kernel<T, 1, TEAM, NP, false>, grid, kThreads, s, a);
      return 1;
    });
    if (known == 0) {
      grid = plan(std::min<long long>(p.rows, 2ll * sms), 1, false);
      if (grid > 0) launch_overlapped(residual_norm_grad_long_kernel<T>, grid, 1024, s, a);
    }
    if (grid == 0) return fail(PDNN_ALLOCATION_PROBLEM, "%s: cannot allocate scratch", what);
    int status = check_launch(what);
    if (status == PDNN_OK && a.partial != nullptr) {
      StoreVectors<T> store;
      store.channels = p.channels;
      for (int i = 0; i < 4; ++i)
        if (a.slot[i] >= 0) store.to[a.slot[i]] = static_cast<T*>(vectors[i]);
      launch_column_sums(a.partial, (int)teams, (size_t)a.vectors * p.channels, sms, s, store);
      status = check_launch(what);
    }
    if (status == PDNN_OK && a.gate_partial != nullptr) {
      launch_column_sums(a.gate_partial, a.parts, (size_t)groups * p.channels, sms, s,
                         StoreGate<T>{static_cast<T*>(g.gate_grad), static_cast<const T*>(t.gate), p.gate_activation});
      status = check_launch(what);
    }
    if (scratch != nullptr) cudaFreeAsync(scratch, s);
    return status;
  });
}

}  // namespace pdnn
