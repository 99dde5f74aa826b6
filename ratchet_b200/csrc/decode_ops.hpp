// Host-side checks of the operators around the Linears (rt_residual_norm, rt_log_probs); no CUDA in this file.
#pragma once
#include "spec.hpp"

namespace rt {

Status check_residual_norm(const rt_residual_norm &op);
Status check_log_probs(const rt_log_probs &op);

} // namespace rt
