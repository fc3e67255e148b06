// Attention kernels of many query rows for heads of 256 values (qmv_attn_tc.cuh).
#include "qmv_attn_tc.cuh"

namespace qmv {
template int attn_tc_dispatch<8>(const AttnParams&, int, cudaStream_t);
}
