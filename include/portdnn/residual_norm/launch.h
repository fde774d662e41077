// The norms around a block with its gate and residual sum, in the manner of the reference's launch headers (it has no such
// operator): sum = residual + scale * act(gate) * post_norm(branch), output = pre_norm(sum), and the gradients.
#ifndef PORTDNN_B200_RESIDUAL_NORM_LAUNCH_H_
#define PORTDNN_B200_RESIDUAL_NORM_LAUNCH_H_
#include <vector>

#include "portdnn/backend/cuda_backend.h"
#include "portdnn/status.h"

namespace sycldnn {
namespace residual_norm {

/** Forward, on tensors of type T: see PdnnResidualNormParams and PdnnResidualNormTensors. */
template <typename T, typename Backend>
SNNStatus launch(PdnnResidualNormParams const& params, PdnnResidualNormTensors const& tensors, Backend& backend,
                 const std::vector<Event>& events = {}) {
  for (const Event& e : events) e.make_stream_wait(backend.get_queue());
  const int st = pdnn_residual_norm(backend::dtype_of<T>::value, &params, &tensors, backend.get_queue());
  return SNNStatus{Event{backend.get_queue()}, StatusCode(st)};
}

/** Gradients: see PdnnResidualNormGradients. */
template <typename T, typename Backend>
SNNStatus launch_gradient(PdnnResidualNormParams const& params, PdnnResidualNormTensors const& tensors,
                          PdnnResidualNormGradients const& gradients, Backend& backend, const std::vector<Event>& events = {}) {
  for (const Event& e : events) e.make_stream_wait(backend.get_queue());
  const int st = pdnn_residual_norm_gradient(backend::dtype_of<T>::value, &params, &tensors, &gradients, backend.get_queue());
  return SNNStatus{Event{backend.get_queue()}, StatusCode(st)};
}

}  // namespace residual_norm
}  // namespace sycldnn
#endif
