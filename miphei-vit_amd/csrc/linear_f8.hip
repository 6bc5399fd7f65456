// mvit_linear kernels: e4m3 operands, 16-bit y
#include "linear_launch.hpp"

template int mvit_linear::dispatch<mvit_linear::F8, false>(const mvit_linear::Args&, bool, hipStream_t);
