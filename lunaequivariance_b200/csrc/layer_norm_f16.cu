#include "layer_norm.cuh"
namespace luna::norm {
template int run<rows::f16>(Order, const Params&, const Operands&, cudaStream_t);
}
