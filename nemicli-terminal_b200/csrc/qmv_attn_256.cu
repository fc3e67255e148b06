// Attention kernels for heads of 256 values (qmv_attn.cuh).
#include "qmv_attn.cuh"

namespace qmv {
template int attn_dispatch<8>(const AttnParams&, int, const AttnPlan&, cudaStream_t);
}
