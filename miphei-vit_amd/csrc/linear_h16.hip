// mvit_linear kernels: 16-bit operands, 16-bit y
#include "linear_launch.hpp"

template int mvit_linear::dispatch<mvit_linear::H16, false>(const mvit_linear::Args&, bool, hipStream_t);
