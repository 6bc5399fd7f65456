// mvit_linear kernels: the gradient's product dx = dz W, 16-bit
#include "linear_launch.hpp"

template int mvit_linear::dispatch_grad<mvit_linear::DX>(const mvit_linear::Args&, int, hipStream_t);
