// Group norm of bfloat16 (the kernels are templates: one type a file, compiled side by side).
#include "group_norm_kernels.h"

template int gn_forward<ogl_bf16, 8>(const gn_args&, const gn_plan&, hipStream_t);
template int gn_backward<ogl_bf16, 8>(const gn_args&, const gn_plan&, void*, void*, hipStream_t);
