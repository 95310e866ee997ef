#include "layer_norm.cuh"
namespace luna::norm {
template int run<double>(Order, const Params&, const Operands&, cudaStream_t);
}
