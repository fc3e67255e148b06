// Attention kernels of many query rows for heads of 64 values (qmv_attn_tc.cuh).
#include "qmv_attn_tc.cuh"

namespace qmv {
template int attn_tc_dispatch<2>(const AttnParams&, int, cudaStream_t);
}
