// Group norm of float32 (the kernels are templates: one type a file, compiled side by side).
#include "group_norm_kernels.h"

template int gn_forward<float, 4>(const gn_args&, const gn_plan&, hipStream_t);
template int gn_backward<float, 4>(const gn_args&, const gn_plan&, void*, void*, hipStream_t);
