// mvit_linear kernels: 16-bit operands, f32 y
#include "linear_launch.hpp"

template int mvit_linear::dispatch<mvit_linear::H16, true>(const mvit_linear::Args&, bool, hipStream_t);
template int mvit_linear::dispatch_parts<mvit_linear::H16>(const mvit_linear::Args&, bool, int, hipStream_t);
