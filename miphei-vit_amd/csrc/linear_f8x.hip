// mvit_linear kernels: e4m3 operands, f32 y
#include "linear_launch.hpp"

template int mvit_linear::dispatch<mvit_linear::F8X, true>(const mvit_linear::Args&, bool, hipStream_t);
template int mvit_linear::dispatch_parts<mvit_linear::F8X>(const mvit_linear::Args&, bool, int, hipStream_t);
