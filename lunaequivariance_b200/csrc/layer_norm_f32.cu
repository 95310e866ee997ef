#include "layer_norm.cuh"
namespace luna::norm {
template int run<float>(Order, const Params&, const Call&, cudaStream_t);
}
