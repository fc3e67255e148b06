// Attention kernels of many query rows for heads of 128 values (qmv_attn_tc.cuh).
#include "qmv_attn_tc.cuh"

namespace qmv {
template int attn_tc_dispatch<4>(const AttnParams&, int, cudaStream_t);
}
