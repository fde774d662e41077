// The operators around a block's matrix products through the C++ templates, against the formulas in double on the host.
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

#include "portdnn/backend/cuda_backend.h"
#include "portdnn/matmul/launch.h"
#include "portdnn/policy_loss/launch.h"
#include "portdnn/residual_norm/launch.h"

namespace sb = sycldnn::backend;

static int failures = 0;
static void check(bool ok, const char* what) {
  if (!ok) {
    std::printf("FAILED: %s (%s)\n", what, pdnn_last_error());
    ++failures;
  }
}

struct Device {
  float* p = nullptr;
  size_t n;
  explicit Device(const std::vector<float>& v) : n(v.size()) {
    cudaMalloc(reinterpret_cast<void**>(&p), n * sizeof(float));
    cudaMemcpy(p, v.data(), n * sizeof(float), cudaMemcpyHostToDevice);
  }
  explicit Device(size_t count) : Device(std::vector<float>(count, -7.f)) {}
  ~Device() { cudaFree(p); }
  std::vector<float> host() const {
    std::vector<float> v(n);
    cudaMemcpy(v.data(), p, n * sizeof(float), cudaMemcpyDeviceToHost);
    return v;
  }
};

static std::vector<float> normal(size_t n, unsigned seed, float std = 1.f) {
  std::mt19937 g(seed);
  std::normal_distribution<float> d(0.f, std);
  std::vector<float> v(n);
  for (float& x : v) x = d(g);
  return v;
}

// (sums of at most 64 products of normal numbers: 2^-18 of the terms' sizes, which are below 100)
static bool close(double got, double want) { return std::fabs(got - want) <= 100. / (1 << 18); }

int main() {
  int devices = 0;
  if (cudaGetDeviceCount(&devices) != cudaSuccess || devices == 0) {
    std::printf("no CUDA device\n");
    return 1;
  }
  cudaStream_t stream;
  cudaStreamCreate(&stream);
  sb::CUDABackend backend{stream};

  const int m = 20, k = 36, n = 24;
  const auto x = normal(m * k, 1), w = normal(k * n, 2, 0.3f), b = normal(n, 3), r = normal(m * n, 4), dy = normal(m * n, 5);
  Device dx(x), dw(w), db(b), dr(r), ddy(dy), out(m * n), pre(m * n), gx(m * k), gw(k * n), gb(n);
  PdnnMatmulParams mp = {m, k, n, 0, 0, 0, 0};
  PdnnMatmulEpilogue me = {db.p, PDNN_ACT_RELU, 0.5f, dr.p, 0, pre.p, 0};
  auto st = sycldnn::matmul::launch_fused<float, false>(dx.p, dw.p, out.p, mp, me, backend);
  check(st.status == sycldnn::StatusCode::OK, "launch_fused");
  PdnnMatmulGradient mg = {};
  mg.activation = PDNN_ACT_RELU;
  mg.scale = 0.5f;
  mg.pre_activation = pre.p;
  mg.input_activation = PDNN_ACT_NONE;
  mg.lhs_grad = gx.p;
  mg.rhs_grad = gw.p;
  mg.bias_grad = gb.p;
  st = sycldnn::matmul::launch_fused_gradient<float, false>(ddy.p, dx.p, dw.p, mp, mg, backend, {st.event});
  check(st.status == sycldnn::StatusCode::OK, "launch_fused_gradient");
  st.event.wait_and_throw();
  const auto ho = out.host(), hp = pre.host(), hx = gx.host(), hw = gw.host(), hb = gb.host();
  std::vector<double> z(m * n), dz(m * n);
  bool ok = true;
  for (int i = 0; i < m; ++i)
    for (int j = 0; j < n; ++j) {
      double s = b[j];
      for (int c = 0; c < k; ++c) s += (double)x[i * k + c] * w[c * n + j];
      z[i * n + j] = s;
      // (where z is next to 0 the stored one decides which side the gradient takes)
      dz[i * n + j] = hp[i * n + j] > 0.f ? 0.5 * dy[i * n + j] : 0.;
      ok = ok && close(hp[i * n + j], s) && close(ho[i * n + j], r[i * n + j] + 0.5 * std::fmax(s, 0.));
    }
  check(ok, "matrix product with its epilogue");
  ok = true;
  for (int i = 0; i < m; ++i)
    for (int c = 0; c < k; ++c) {
      double s = 0;
      for (int j = 0; j < n; ++j) s += dz[i * n + j] * w[c * n + j];
      ok = ok && close(hx[i * k + c], s);
    }
  for (int j = 0; j < n; ++j) {
    double t = 0;
    for (int i = 0; i < m; ++i) t += dz[i * n + j];
    ok = ok && close(hb[j], t);
    for (int c = 0; c < k; ++c) {
      double s = 0;
      for (int i = 0; i < m; ++i) s += x[i * k + c] * dz[i * n + j];
      ok = ok && close(hw[c * n + j], s);
    }
  }
  check(ok, "gradients of the matrix product");

  // norms: root mean square behind the block, the next block's too
  Device branch(x), residual(normal(m * k, 6)), gamma(normal(k, 7)), sum(m * k), normed(m * k), statistics(4 * m);
  PdnnResidualNormParams np = {m, k, PDNN_NORM_RMS, PDNN_NORM_RMS, 0, PDNN_ACT_NONE, 1.f, 1e-5f};
  PdnnResidualNormTensors nt = {};
  nt.branch = branch.p;
  nt.residual = residual.p;
  nt.post_gamma = gamma.p;
  nt.sum = sum.p;
  nt.output = normed.p;
  nt.statistics = statistics.p;
  auto ns = sycldnn::residual_norm::launch<float>(np, nt, backend);
  check(ns.status == sycldnn::StatusCode::OK, "residual_norm::launch");
  Device dsum(m * k), dgamma(k), dbranch(m * k);
  PdnnResidualNormGradients ng = {};
  ng.output_grad = branch.p;
  ng.residual_grad = dsum.p;
  ng.branch_grad = dbranch.p;
  ng.post_gamma_grad = dgamma.p;
  ns = sycldnn::residual_norm::launch_gradient<float>(np, nt, ng, backend);
  check(ns.status == sycldnn::StatusCode::OK, "residual_norm::launch_gradient");
  ns.event.wait_and_throw();
  const auto hs = sum.host(), hn = normed.host(), hg = gamma.host(), hr = residual.host(), hd = dsum.host();
  ok = true;
  for (int i = 0; i < m; ++i) {
    double q = 0, p = 0, inner = 0;
    for (int c = 0; c < k; ++c) q += (double)x[i * k + c] * x[i * k + c];
    const double r1 = 1 / std::sqrt(q / k + 1e-5);
    std::vector<double> s(k);
    for (int c = 0; c < k; ++c) {
      s[c] = hr[i * k + c] + hg[c] * r1 * x[i * k + c];
      p += s[c] * s[c];
    }
    const double r2 = 1 / std::sqrt(p / k + 1e-5);
    for (int c = 0; c < k; ++c) inner += x[i * k + c] * s[c] * r2 / k;
    for (int c = 0; c < k; ++c)
      ok = ok && close(hs[i * k + c], s[c]) && close(hn[i * k + c], s[c] * r2) &&
           close(hd[i * k + c], r2 * (x[i * k + c] - s[c] * r2 * inner));
  }
  check(ok, "norms and the gradient of the sum");

  // loss: one token of each row of x
  std::vector<int> targets(m);
  for (int i = 0; i < m; ++i) targets[i] = i % k;
  int* dt = nullptr;
  cudaMalloc(reinterpret_cast<void**>(&dt), m * sizeof(int));
  cudaMemcpy(dt, targets.data(), m * sizeof(int), cudaMemcpyHostToDevice);
  Device adv(normal(m, 8)), loss(size_t(1)), token(m), logp(m), grad(m * k);
  PdnnPolicyLossParams lp = {m, k, 4, 0.2f, 0.2f, 0.f, 1.f, 1.f, k, k};
  PdnnPolicyLossTensors lt = {};
  lt.logits = dx.p;
  lt.targets = dt;
  lt.advantages = adv.p;
  lt.loss = loss.p;
  lt.token_loss = token.p;
  lt.logp = logp.p;
  lt.grad = grad.p;
  auto ls = sycldnn::policy_loss::launch<float>(lp, lt, backend);
  check(ls.status == sycldnn::StatusCode::OK, "policy_loss::launch");
  ls.event.wait_and_throw();
  const auto ha = adv.host(), hl = loss.host(), hlp = logp.host(), hgr = grad.host();
  ok = true;
  double all = 0;
  for (int i = 0; i < m; ++i) {
    double s = 0;
    for (int c = 0; c < k; ++c) s += std::exp((double)x[i * k + c]);
    all -= ha[i];  // the ratio to itself is 1
    ok = ok && close(hlp[i], x[i * k + targets[i]] - std::log(s));
    for (int c = 0; c < k; ++c) ok = ok && close(hgr[i * k + c], -ha[i] * ((c == targets[i]) - std::exp((double)x[i * k + c]) / s));
  }
  check(ok && close(hl[0], all), "policy loss");

  // refusals come back as the reference's status codes
  lp.temperature = 0.f;
  check(sycldnn::policy_loss::launch<float>(lp, lt, backend).status == sycldnn::StatusCode::InvalidParameter, "a temperature of 0");
  np.epsilon = -1.f;
  check(sycldnn::residual_norm::launch<float>(np, nt, backend).status == sycldnn::StatusCode::InvalidParameter, "a negative epsilon");
  mp.k = 0;
  check(sycldnn::matmul::launch_fused<float, false>(dx.p, dw.p, out.p, mp, me, backend).status == sycldnn::StatusCode::InvalidParameter,
        "a product without terms");
  cudaFree(dt);
  cudaStreamDestroy(stream);
  if (failures == 0) std::printf("all checks passed\n");
  return failures != 0;
}
