// Translation unit of the memory-bound layers: layer norm and 8-bit activation
// checkpoints.
#include "act8.cu"
#include "layer_norm.cu"
