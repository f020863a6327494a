// Attention over the quantized cache: argument checks, the plan (row tiles, key splits), and the join of split keys.
#include "kv_attention.cuh"

namespace b2q {

// Joins the key splits of a row: one warp a row, its lanes over the dimension.
__global__ void __launch_bounds__(128) attention_join_kernel(const AttnParams p, int dim, int64_t rows) {
  pdl_wait_then_trigger();
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  if (p.cu_q && row / p.q_heads >= p.cu_q[p.batch]) return;  // a row of no sequence: nothing was computed for it
  const float2* pm = p.part_m + row * p.splits;
  float m = kNoRef;
  bool bad = false;
  for (int s = lane; s < p.splits; s += 32) {
    const float v = pm[s].x;
    m = fmaxf(m, v), bad |= isnan(v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  bad = __any_sync(0xffffffffu, bad);
  float l = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const float* po = p.part_o + row * p.splits * dim;
  for (int s = 0; s < p.splits; ++s) {
    const float2 v = pm[s];
    const float f = bad ? NAN : exp2_approx(v.x - m);
    l += v.y * f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < dim) y[i] += po[(int64_t)s * dim + i * 32 + lane] * f;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 + lane < dim) store_elt(p.out, row * dim + i * 32 + lane, p.dtype, y[i] * inv);
  if (p.lse && lane == 0) p.lse[row] = (m + log2f(l)) * kLn2;
}

struct AttnPlan {
  int rows, row_tiles, splits;
  size_t part_o, bytes;  // workspace: partial outputs, then references and sums
};

static AttnPlan plan_attention(const b2q_kv_cache& c, const b2q_attention_args& a) {
  AttnPlan pl;
  const int group = a.q_heads / c.heads;
  const int64_t max_q = !a.cu_q ? 1 : (a.max_q > 0 && a.max_q < a.T ? a.max_q : a.T);
  const int64_t rows = max_q * group;
  pl.rows = rows > 8 && c.dim != 256 ? 16 : 8;
  pl.row_tiles = (int)((rows + pl.rows - 1) / pl.rows);
  DeviceInfo di;
  const int sms = device_info(&di) == B2Q_OK ? di.sms : 148;
  // key splits: enough CTAs for two waves of two per SM, each with at least 256 keys
  const int64_t tasks = a.batch * c.heads * pl.row_tiles;
  const int64_t most = (a.max_len + 255) / 256;
  int64_t splits = (4 * sms + tasks - 1) / tasks;
  if (splits > most) splits = most;
  if (a.window > 0 && max_q == 1 && splits > (a.window + 511) / 256) splits = (a.window + 511) / 256;
  if (splits > 256) splits = 256;
  if (splits < 1) splits = 1;
  pl.splits = (int)splits;
  pl.part_o = pl.bytes = 0;
  if (splits > 1) {
    const size_t n = (size_t)a.T * a.q_heads * splits;
    pl.part_o = (n * c.dim * 4 + 255) / 256 * 256;
    pl.bytes = pl.part_o + n * 8;
  }
  return pl;
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
  if (!(a->softcap >= 0.f)) return fail(B2Q_EINVAL, "%s: softcap must not be negative", who);
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
  if (!aligned(a->q, dtype_size(a->dtype)) || !aligned(a->out, 16) || !aligned(a->table, 4) || !aligned(a->lens, 4))
    return fail(B2Q_EALIGN, "%s: misaligned pointer", who);
  if (a->T * a->q_heads / c->heads > INT_MAX / 2) return fail(B2Q_ERANGE, "%s: T=%lld", who, (long long)a->T);
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
  if (pl.bytes && (!workspace || workspace_bytes < pl.bytes || !aligned(workspace, 16)))
    return fail(B2Q_EINVAL, "%s: needs a 16-byte aligned workspace of %zu bytes", who, pl.bytes);
  if (a.batch * c.heads * pl.row_tiles * pl.splits > INT_MAX)
    return fail(B2Q_ERANGE, "%s: too many tiles", who);
  AttnParams p = {};
  p.q = a.q, p.out = a.out, p.lse = a.lse;
  p.kq = c.kq, p.vq = c.vq;
  p.ks = reinterpret_cast<const uint16_t*>(c.ks), p.vs = reinterpret_cast<const uint16_t*>(c.vs);
  p.table = a.table, p.lens = a.lens, p.cu_q = a.cu_q, p.prefix = a.prefix, p.starts = a.starts, p.slopes = a.slopes;
  p.part_o = static_cast<float*>(workspace);
  p.part_m = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + pl.part_o);
  p.q_st = a.q_st, p.q_sh = a.q_sh, p.T = a.T, p.table_stride = a.table_stride, p.pages = c.pages;
  p.table_pages = (int)a.table_pages, p.batch = (int)a.batch, p.q_heads = a.q_heads, p.heads = c.heads;
  p.group = a.q_heads / c.heads;
  while ((1 << p.page_shift) < c.page) ++p.page_shift;
  p.splits = pl.splits, p.row_tiles = pl.row_tiles, p.window = a.window, p.dtype = a.dtype;
  p.scale = a.scale, p.softcap = a.softcap;
  rc = c.fmt == B2Q_FMT_Q4_0 ? launch_attention_q4(p, c.dim, pl.rows, (cudaStream_t)stream)
                             : launch_attention_q8(p, c.dim, pl.rows, (cudaStream_t)stream);
  if (rc || pl.splits == 1) return rc;
  const int64_t rows = a.T * a.q_heads;
  launch_maybe_pdl(attention_join_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, (cudaStream_t)stream, p,
                   c.dim, rows);
  return after_launch("attention_join");
}

}  // extern "C"
