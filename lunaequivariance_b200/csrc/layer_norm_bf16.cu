#include "layer_norm.cuh"
namespace luna::norm {
template int run<rows::bf16>(Order, const Params&, const Call&, cudaStream_t);
}
