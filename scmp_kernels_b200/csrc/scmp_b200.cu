// Translation unit of the SC matmul: its kernels share one device error
// record, so they are compiled together instead of with -rdc. The layers
// around it are units of their own (norms.cu, linears.cu).
#include "tables.cu"
#include "quant.cu"
#include "gemm_simt.cu"
#include "gemm_tc.cu"
#include "api.cu"
#include "levels.cu"
#include "quant_ref.cu"
#include "noalloc.cu"
