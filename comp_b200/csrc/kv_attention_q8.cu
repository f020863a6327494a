// The streaming attention kernels over q8_0 caches.
#include "kv_attention.cuh"

namespace b2q {

int launch_attention_q8(const AttnParams& p, int dim, int rows, int sms, int64_t max_len, cudaStream_t stream) {
  return launch_attention_fmt<2>(p, dim, rows, sms, max_len, stream);
}

int kv_attention_q8_error(int* code, int clear) { return read_error_word(g_device_error, code, clear); }

}  // namespace b2q
