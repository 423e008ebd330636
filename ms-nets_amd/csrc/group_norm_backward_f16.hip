// Group norm backward, float16 (group_norm_backward.h).
#include "group_norm_backward.h"

int msnet::gn::backward_f16(const Backward& f, const BackwardPlan& p, int act, void* ws) { return backward_t<_Float16>(f, p, act, ws); }
