// ns_path_commit: the accepted path's keys and values move to the end of the context, every layer in
// one launch.  No reference counterpart (it never caches tokens that it may drop).
//
// Pure traffic of a few hundred bytes per head: latency counts.  One thread owns one 16-byte column
// (a 2- or 4-byte one where rows are not 16-byte aligned) of one head's rows and moves them in path
// order.  The path ascends, so a row's target is never a later row's source (i < j gives
// i <= path[i] < path[j]) and a thread may load a batch of rows ahead of its stores; columns are
// independent, so nothing waits on another thread.  Measured (device time of a call in a captured graph,
// 36 layers of 8 heads): one sequence, 16 nodes, fp32, 3.0 us; 8 sequences, 64 nodes, bf16, 15 us
// (50 MB, 3.4 TB/s): the loads of a batch of 8 rows wait for the path, then for memory.
#include "tree.cuh"

namespace ns {

constexpr int kCommitThreads = 128;
constexpr int kCommitBatch = 8;  // rows in flight per thread

template <typename Col>
__global__ void __launch_bounds__(kCommitThreads) path_commit_kernel(const __grid_constant__ ns_path_commit_t p,
                                                                     int cols) {
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.y;
  const int len = tree_len(p.lens, b, p.max_ctx), n = p.n_accepted[b];
  const int32_t* path = p.path + (int64_t)b * p.T;
  bool bad = len < 0 || n < -1 || n >= p.T;
  for (int i = 0; i <= n && !bad; ++i) {
    const int at = path[i];
    bad = at < i || at >= p.T || len + at >= p.max_ctx || (i > 0 && at <= path[i - 1]);
  }
  const bool first = blockIdx.x == 0 && threadIdx.x == 0;
  if (first) {
    if (bad) raise_device_error(NS_DEVERR_ROUTE);
    p.new_lens[b] = bad ? p.lens[b] : len + 1 + n;
  }
  if (bad) return;
  const int rows = p.n_layer * 2 * p.n_head_kv;  // (layer, key or value, head)
  const int i0 = blockIdx.x * kCommitThreads + threadIdx.x;
  if (i0 >= rows * cols) return;
  const int c = i0 % cols, h = i0 / cols % p.n_head_kv, lv = i0 / cols / p.n_head_kv;
  const int64_t* st = lv & 1 ? p.vc_stride : p.kc_stride;
  char* cache = static_cast<char*>(lv & 1 ? p.v_cache[lv >> 1] : p.k_cache[lv >> 1]);
  const int esize = p.dtype == NS_F32 ? 4 : 2;
  char* base = cache + (b * st[0] + h * st[1] + len * st[2]) * esize + (int64_t)c * sizeof(Col);
  const int64_t step = st[2] * esize;
  for (int i = 0; i <= n; i += kCommitBatch) {
    Col x[kCommitBatch];
#pragma unroll
    for (int j = 0; j < kCommitBatch; ++j)
      if (i + j <= n && path[i + j] != i + j) x[j] = *reinterpret_cast<const Col*>(base + path[i + j] * step);
#pragma unroll
    for (int j = 0; j < kCommitBatch; ++j)
      if (i + j <= n && path[i + j] != i + j) *reinterpret_cast<Col*>(base + (i + j) * step) = x[j];
  }
}

}  // namespace ns

extern "C" int ns_path_commit(const ns_path_commit_t* p, ns_stream_t stream) {
  using namespace ns;
  if (!p) return fail(NS_ERR_INVALID, "ns_path_commit: null parameters");
  if (p->n_layer < 0 || p->n_layer > NS_COMMIT_MAX_LAYERS)
    return fail(NS_ERR_INVALID, "ns_path_commit: %d layers (at most %d)", p->n_layer, NS_COMMIT_MAX_LAYERS);
  if (p->B < 0 || p->T < 1 || p->n_head_kv < 1 || p->head_dim < 1 || p->max_ctx < 0)
    return fail(NS_ERR_INVALID, "ns_path_commit: bad B, T, head count, head_dim or max_ctx");
  if (p->T > INT32_MAX - p->max_ctx)  // slots are counted in 32 bits
    return fail(NS_ERR_UNSUPPORTED, "ns_path_commit: caches of %d slots, %d nodes", p->max_ctx, p->T);
  if (!float_type_ok(p->dtype)) return fail(NS_ERR_INVALID, "ns_path_commit: bad dtype %d", p->dtype);
  if (p->B > 65535) return fail(NS_ERR_UNSUPPORTED, "ns_path_commit: %d sequences (at most 65535)", p->B);
  if (p->B == 0) return NS_OK;
  if (!p->lens || !p->path || !p->n_accepted || !p->new_lens)
    return fail(NS_ERR_INVALID, "ns_path_commit: null lens, path, n_accepted or new_lens");
  if (p->new_lens == p->lens) return fail(NS_ERR_INVALID, "ns_path_commit: new_lens must not be lens");
  const int64_t esize = float_size(p->dtype), row = p->head_dim * esize;
  bool vec = row % 16 == 0 && strides_multiple(p->kc_stride, 3, 16 / esize) && strides_multiple(p->vc_stride, 3, 16 / esize);
  for (int l = 0; l < p->n_layer; ++l) {
    if (!p->k_cache[l] || !p->v_cache[l]) return fail(NS_ERR_INVALID, "ns_path_commit: layer %d has a null cache", l);
    vec = vec && aligned_to(p->k_cache[l], 16) && aligned_to(p->v_cache[l], 16);
  }
  const int cols = (int)(vec ? row / 16 : p->head_dim);
  const int64_t n = (int64_t)p->n_layer * 2 * p->n_head_kv * cols;
  if (n > (1ll << 30)) return fail(NS_ERR_UNSUPPORTED, "ns_path_commit: %d layers of %d heads of %d", p->n_layer,
                                   p->n_head_kv, p->head_dim);
  const dim3 grid((unsigned)std::max<int64_t>(1, (n + kCommitThreads - 1) / kCommitThreads), (unsigned)p->B);
  if (vec)
    NS_CUDA_TRY(launch_pdl(path_commit_kernel<uint4>, grid, kCommitThreads, 0, stream, 1, *p, cols));
  else if (esize == 4)
    NS_CUDA_TRY(launch_pdl(path_commit_kernel<uint32_t>, grid, kCommitThreads, 0, stream, 1, *p, cols));
  else
    NS_CUDA_TRY(launch_pdl(path_commit_kernel<uint16_t>, grid, kCommitThreads, 0, stream, 1, *p, cols));
  return NS_OK;
}
