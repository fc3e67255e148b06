// Attention kernels for heads of 128 values (qmv_attn.cuh).
#include "qmv_attn.cuh"

namespace qmv {
template int attn_dispatch<4>(const AttnParams&, int, const AttnPlan&, cudaStream_t);
}
