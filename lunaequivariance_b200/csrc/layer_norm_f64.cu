#include "layer_norm.cuh"
namespace luna::norm {
template int run<double>(Order, const Params&, const Call&, cudaStream_t);
}
