// Attention kernels for heads of 64 values (qmv_attn.cuh).
#include "qmv_attn.cuh"

namespace qmv {
template int attn_dispatch<2>(const AttnParams&, int, const AttnPlan&, cudaStream_t);
}
