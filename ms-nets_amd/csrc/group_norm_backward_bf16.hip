// Group norm backward, bfloat16 (group_norm_backward.h).
#include "group_norm_backward.h"

int msnet::gn::backward_bf16(const Backward& f, const BackwardPlan& p, int act, void* ws) { return backward_t<__bf16>(f, p, act, ws); }
