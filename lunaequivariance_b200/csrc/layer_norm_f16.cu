#include "layer_norm.cuh"
namespace luna::norm {
template int run<rows::f16>(Order, const Params&, const Call&, cudaStream_t);
}
