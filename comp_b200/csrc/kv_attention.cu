// Attention over the quantized cache: argument checks, the plan (row tiles, key splits), and the join of split keys.
#include "kv_attention.cuh"

namespace b2q {

struct AttnPlan {
  bool tc;  // the tensor-core kernels
  int rows, row_tiles, sms;
  size_t part_m, joins, bytes;  // workspace: partial outputs, then references and sums, then the joins
};

// 16-bit calls with at least so many query rows a sequence and KV head take the tensor-core kernels (those with heads of 256
// and lse stay with the streaming one). Measured, us, streaming / tensor cores: 16 sequences of 4096 keys, 8 KV heads of 128,
// bf16: 48 rows 95 / 91, 64 rows 120 / 93, 256 rows 417 / 126; f16: 48 rows 95 / 119, 64 rows 120 / 121, 80 rows 145 / 123;
// one of 8192, bf16: 23 / 25 at 48, 63 / 39 at 256; 16 of 4096, heads of 256, bf16: 154 / 174 at 32, 223 / 163 at 48; f16: 222
// / 266 at 48, 291 / 270 at 64. (One of 500 keys, bf16: 16 / 15 at 48, 21 / 27 at 256: that little work is launches and tile
// ends.) Else the rows of a tile are 8, or 16 where more have to read the cache anyway (heads of 256 leave registers for 8).
static int least_tc_rows(const b2q_attention_args& a) { return a.dtype == B2Q_DTYPE_F16 ? 64 : 48; }

static AttnPlan plan_attention(const b2q_kv_cache& c, const b2q_attention_args& a) {
  AttnPlan pl;
  const int group = a.q_heads / c.heads;
  const int64_t max_q = !a.cu_q ? 1 : (a.max_q > 0 && a.max_q < a.T ? a.max_q : a.T);
  const int64_t rows = max_q * group;
  pl.tc = rows >= least_tc_rows(a) && a.dtype != B2Q_DTYPE_F32 && !(c.dim == 256 && a.lse);
  if (pl.tc)
    pl.rows = c.dim == 256 ? kTcRows / 2 : kTcRows;
  else
    pl.rows = rows > 8 && c.dim != 256 ? 16 : 8;
  pl.row_tiles = (int)((rows + pl.rows - 1) / pl.rows);
  DeviceInfo di;
  pl.sms = device_info(&di) == B2Q_OK ? di.sms : 148;
  const size_t ctas = (size_t)pl.sms * (pl.tc ? 1 : kMaxCtasPerSm);
  pl.part_m = 2 * ctas * pl.rows * c.dim * 4;
  pl.joins = pl.part_m + 2 * ctas * pl.rows * 8;
  pl.bytes = pl.joins + ctas * sizeof(AttnJoin);
  return pl;
}

int allow_smem_once(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return B2Q_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(B2Q_ECUDA, "b2q_attention: %s", cudaGetErrorString(e));
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return B2Q_OK;
}

static int check_attention(const char* who, const b2q_kv_cache* c, const b2q_attention_args* a) {
  int rc = check_kv_cache(who, c);
  if (rc) return rc;
  if (!a) return fail(B2Q_EINVAL, "%s: null arguments", who);
  if (a->T < 0 || a->batch < 0 || a->table_pages < 0 || a->max_q < 0 || a->max_len < 0)
    return fail(B2Q_EINVAL, "%s: negative size", who);
  if (a->q_heads < 1 || a->q_heads > 65536 || a->q_heads % c->heads)
    return fail(B2Q_EINVAL, "%s: %d query heads over %d KV heads", who, a->q_heads, c->heads);
  if (a->dtype < 0 || a->dtype > 2) return fail(B2Q_EINVAL, "%s: dtype %d", who, a->dtype);
  if (!(a->scale > 0.f) || a->scale > 1e30f) return fail(B2Q_EINVAL, "%s: scale must be positive", who);
  if (!(a->softcap == 0.f || (a->softcap >= 1e-20f && a->softcap <= 1e20f)))
    return fail(B2Q_EINVAL, "%s: softcap must be 0 (none) or from 1e-20 to 1e20", who);
  if (a->window < 0) return fail(B2Q_EINVAL, "%s: window must not be negative", who);
  if (!a->cu_q && a->T != a->batch)
    return fail(B2Q_EINVAL, "%s: without cu_q there is one query token a sequence (T=%lld, batch=%lld)", who,
                (long long)a->T, (long long)a->batch);
  if (a->T == 0 || a->batch == 0) return B2Q_OK;
  if (!a->q || !a->out || !a->lens || (a->table_pages && !a->table)) return fail(B2Q_EINVAL, "%s: null pointer", who);
  if (a->table_stride < a->table_pages)
    return fail(B2Q_EINVAL, "%s: table_stride %lld < table_pages %lld", who, (long long)a->table_stride,
                (long long)a->table_pages);
  if (a->table_pages * c->page > (int64_t)INT_MAX - 65536)
    return fail(B2Q_ERANGE, "%s: a table of %lld pages of %d tokens", who, (long long)a->table_pages, c->page);
  const int64_t mult = 16 / dtype_size(a->dtype);
  if (!aligned(a->q, 16) || a->q_st % mult || a->q_sh % mult)
    return fail(B2Q_EALIGN, "%s: q must be 16-byte aligned, in its strides too", who);
  if (!aligned(a->out, 16) || !aligned(a->table, 4) || !aligned(a->lens, 4))
    return fail(B2Q_EALIGN, "%s: misaligned pointer", who);
  if (a->T * a->q_heads > INT_MAX) return fail(B2Q_ERANGE, "%s: T=%lld", who, (long long)a->T);
  return B2Q_OK;
}

}  // namespace b2q

using namespace b2q;

extern "C" {

size_t b2q_attention_workspace_size(const b2q_kv_cache* cache, const b2q_attention_args* args) {
  if (check_attention("b2q_attention_workspace_size", cache, args) || args->T == 0 || args->batch == 0) return 0;
  return plan_attention(*cache, *args).bytes;
}

int b2q_attention(const b2q_kv_cache* cache, const b2q_attention_args* args, void* workspace, size_t workspace_bytes,
                  b2q_stream_t stream) {
  const char* who = "b2q_attention";
  int rc = check_attention(who, cache, args);
  if (rc) return rc;
  const b2q_attention_args& a = *args;
  const b2q_kv_cache& c = *cache;
  if (a.T == 0 || a.batch == 0) return B2Q_OK;
  const AttnPlan pl = plan_attention(c, a);
  if (!workspace || workspace_bytes < pl.bytes || !aligned(workspace, 16))
    return fail(B2Q_EINVAL, "%s: needs a 16-byte aligned workspace of %zu bytes", who, pl.bytes);
  if (a.batch * pl.row_tiles > INT_MAX / 2) return fail(B2Q_ERANGE, "%s: too many tiles", who);
  AttnParams p = {};
  p.q = a.q, p.out = a.out, p.lse = a.lse;
  p.kq = c.kq, p.vq = c.vq;
  p.ks = reinterpret_cast<const uint16_t*>(c.ks), p.vs = reinterpret_cast<const uint16_t*>(c.vs);
  p.table = a.table, p.lens = a.lens, p.cu_q = a.cu_q, p.prefix = a.prefix, p.starts = a.starts, p.slopes = a.slopes;
  p.part_o = static_cast<float*>(workspace);
  p.part_m = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + pl.part_m);
  p.joins = reinterpret_cast<AttnJoin*>(static_cast<uint8_t*>(workspace) + pl.joins);
  p.q_st = a.q_st, p.q_sh = a.q_sh, p.T = a.T, p.table_stride = a.table_stride, p.pages = c.pages;
  p.table_pages = (int)a.table_pages, p.batch = (int)a.batch, p.q_heads = a.q_heads, p.heads = c.heads;
  p.group = a.q_heads / c.heads;
  while ((1 << p.page_shift) < c.page) ++p.page_shift;
  p.row_tiles = pl.row_tiles, p.dtype = a.dtype;
  p.window = a.window;
  p.scale = a.scale, p.softcap = a.softcap;
  if (pl.tc)
    return c.fmt == B2Q_FMT_Q4_0 ? launch_attention_tc_q4(p, c.dim, pl.sms, (cudaStream_t)stream)
                                 : launch_attention_tc_q8(p, c.dim, pl.sms, (cudaStream_t)stream);
  const int64_t held = a.table_pages * c.page, max_len = a.max_len > 0 && a.max_len < held ? a.max_len : held;
  return c.fmt == B2Q_FMT_Q4_0 ? launch_attention_q4(p, c.dim, pl.rows, pl.sms, max_len, (cudaStream_t)stream)
                               : launch_attention_q8(p, c.dim, pl.rows, pl.sms, max_len, (cudaStream_t)stream);
}

}  // extern "C"
