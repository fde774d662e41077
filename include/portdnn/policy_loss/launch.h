// The clipped policy loss of sampled tokens and its gradient, in the manner of the reference's launch headers (it has no such
// operator).
#ifndef PORTDNN_B200_POLICY_LOSS_LAUNCH_H_
#define PORTDNN_B200_POLICY_LOSS_LAUNCH_H_
#include <vector>

#include "portdnn/backend/cuda_backend.h"
#include "portdnn/status.h"

namespace sycldnn {
namespace policy_loss {

/** Loss, log-probabilities and, where tensors.grad is given, the gradient of logits of type T: see PdnnPolicyLossParams. */
template <typename T, typename Backend>
SNNStatus launch(PdnnPolicyLossParams const& params, PdnnPolicyLossTensors const& tensors, Backend& backend,
                 const std::vector<Event>& events = {}) {
  for (const Event& e : events) e.make_stream_wait(backend.get_queue());
  const int st = pdnn_policy_loss(backend::dtype_of<T>::value, &params, &tensors, backend.get_queue());
  return SNNStatus{Event{backend.get_queue()}, StatusCode(st)};
}

}  // namespace policy_loss
}  // namespace sycldnn
#endif
