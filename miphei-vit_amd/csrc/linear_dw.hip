// mvit_linear kernels: the gradient's product dW = dz^T x, 16-bit
#include "linear_launch.hpp"

template int mvit_linear::dispatch_grad<mvit_linear::DW>(const mvit_linear::Args&, int, hipStream_t);
