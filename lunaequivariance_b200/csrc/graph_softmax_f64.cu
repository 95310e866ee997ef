#include "graph_softmax.cuh"
namespace luna::softmax {
template LUNA_SOFTMAX_RUN(double);
}
