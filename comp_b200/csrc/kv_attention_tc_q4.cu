// The tensor-core attention kernels over q4_0 caches.
#include "kv_attention_tc.cuh"

namespace b2q {

int launch_attention_tc_q4(const AttnParams& p, int dim, int sms, cudaStream_t stream) {
  return launch_attention_tc_fmt<0>(p, dim, sms, stream);
}

int kv_attention_tc_q4_error(int* code, int clear) { return read_error_word(g_device_error, code, clear); }

}  // namespace b2q
