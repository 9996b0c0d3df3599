// ns_tree_verify: walk of a drafted tree against the target's logits, from given random numbers.
// No reference counterpart (it decodes greedily, one token a step).
//
// The walk is serial (which row comes next depends on what was accepted), a row is V logits, and a
// tree's rows are mostly never looked at: only the rows of the nodes that the walk stands on are read.
// One thread-block cluster walks one sequence; CTA r of it holds slice r of the vocabulary.  A row
// costs one pass (scaled logits into shared memory, running maximum, sum of exponentials and lowest
// index of the maximum per thread) and one exchange through distributed shared memory; every CTA
// then holds the row's maximum and sum, and takes the same decisions from the same bits.  With
//   r_0 = p = exp(s - m) / Z,  q_0 = q,
//   rejecting c:  w = max(r_j - q_j, 0),  z = sum w,  r_{j+1} = w / z,  q_{j+1} = q_j / (1 - q_j(c)), q_{j+1}(c) = 0,
// a rejection costs a pass over the slice and an exchange of z.  (c needs no zero in the slice's q:
// w(c) = 0, since it was rejected with u < 1, and stays 0.)
// The next token maximises r(x) / race(x): scores, unlike a cumulative sum over the vocabulary, do not
// depend on the order of a summation.
#include "tree.cuh"

namespace ns {

constexpr int kVerifyThreads = 512;
constexpr int kVerifyMaxCluster = 16;
constexpr int kVerifyMaxSlice = 25600;  // logits of one CTA: two fp32 buffers of it in shared memory

struct VerifyPart {  // one CTA's part of an exchange
  float m, z;
  int idx, pad;
};

struct VerifySmem {
  VerifyPart part[2];                       // by parity of the exchange, read by the whole cluster
  VerifyPart all;                           // its outcome, for this CTA's threads
  float red_m[kVerifyThreads / 32], red_z[kVerifyThreads / 32];
  int red_i[kVerifyThreads / 32];
  int tok[kTreeMax * 16], par[kTreeMax * 16];  // up to 1024 nodes
};

constexpr int kVerifyMaxNodes = kTreeMax * 16;

struct VerifyArgs {
  ns_tree_verify_t p;
  int slice;
};

__device__ __forceinline__ float clean_logit(float x) {
  return x <= 3.402823466e38f ? x : (x != x ? -INFINITY : 3.402823466e38f);
}

// Outcome over the cluster of (max with lowest index) and sum scaled to the maximum: parts (m, z, idx)
// combine to m = max, z = sum z_i exp(m_i - m).  SCALED = false: z is a plain sum.
template <bool SCALED>
__device__ __forceinline__ void verify_combine(float& m, float& z, int& i, float m2, float z2, int i2, float inv_t) {
  if (SCALED) {
    const float mx = fmaxf(m, m2);
    const float ref = mx == -INFINITY ? 0.f : mx;
    z = z * expf((m - ref) * inv_t) + z2 * expf((m2 - ref) * inv_t);
  } else {
    z += z2;
  }
  if (m2 > m || (m2 == m && i2 < i)) {
    m = m2;
    i = i2;
  }
}

template <bool SCALED>
__device__ __forceinline__ VerifyPart verify_exchange(VerifySmem& S, float m, float z, int i, int cluster, int& round,
                                                      float inv_t = 1.f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    verify_combine<SCALED>(m, z, i, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, z, o),
                           __shfl_xor_sync(0xffffffffu, i, o), inv_t);
  if (lane == 0) S.red_m[warp] = m, S.red_z[warp] = z, S.red_i[warp] = i;
  __syncthreads();
  VerifyPart& mine = S.part[round & 1];
  if (warp == 0) {
    const bool has = lane < kVerifyThreads / 32;
    m = has ? S.red_m[lane] : -INFINITY, z = has ? S.red_z[lane] : 0.f, i = has ? S.red_i[lane] : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      verify_combine<SCALED>(m, z, i, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, z, o),
                             __shfl_xor_sync(0xffffffffu, i, o), inv_t);
    if (lane == 0) mine = VerifyPart{m, z, i, 0};
  }
  if (cluster > 1) {
    // one barrier per exchange: a slot is written again two exchanges later, past the barrier between
    cluster_sync_all();
    if (warp == 0) {
      m = -INFINITY, z = 0.f, i = 0x7fffffff;
      if (lane < cluster) {
        const uint32_t a = mapa_shared(smem_addr(&mine), lane);
        m = ld_cluster_f32(a), z = ld_cluster_f32(a + 4), i = __float_as_int(ld_cluster_f32(a + 8));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        verify_combine<SCALED>(m, z, i, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, z, o),
                               __shfl_xor_sync(0xffffffffu, i, o), inv_t);
    }
  }
  if (threadIdx.x == 0) S.all = VerifyPart{m, z, i, 0};
  __syncthreads();
  ++round;
  const VerifyPart r = S.all;
  __syncthreads();
  return r;
}

__global__ void __launch_bounds__(kVerifyThreads) tree_verify_kernel(const __grid_constant__ VerifyArgs a, int cluster) {
  const ns_tree_verify_t& p = a.p;
  extern __shared__ __align__(16) uint8_t verify_smem[];
  VerifySmem& S = *reinterpret_cast<VerifySmem*>(verify_smem);
  float* cur = reinterpret_cast<float*>(verify_smem + sizeof(VerifySmem));  // scaled logits, then r times z
  float* nxt = cur + a.slice;
  const int tid = threadIdx.x;
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int b = blockIdx.x / cluster;
  const int lo = min(p.V, rank * a.slice), n_el = min(p.V, lo + a.slice) - lo;
  griddep_wait();
  griddep_launch_dependents();

  for (int t = tid; t < p.T; t += kVerifyThreads) {
    S.tok[t] = p.tokens[(int64_t)b * p.T + t];
    S.par[t] = p.parents ? p.parents[(int64_t)b * p.T + t] : t - 1;
    if (rank == 0) p.path[(int64_t)b * p.T + t] = -1;
  }
  const float temp = p.temperature ? p.temperature[b] : 1.f;
  const bool greedy = temp == 0.f;
  const float inv_t = greedy ? 1.f : 1.f / temp;
  __syncthreads();
  const bool root_ok = S.par[0] == -1;
  if (!root_ok && tid == 0 && rank == 0) raise_device_error(NS_DEVERR_ROUTE);

  int node = 0, n_acc = 0, token = -1, round = 0;
  while (root_ok) {
    if (rank == 0 && tid == 0) p.path[(int64_t)b * p.T + n_acc] = node;
    // the row: scaled logits of the slice, their maximum (lowest index) and sum of exponentials
    const int64_t row = b * p.l_stride[0] + node * p.l_stride[1];
    float m = -INFINITY, z = 0.f;
    int idx = 0x7fffffff;
    for (int e0 = tid; e0 < n_el; e0 += 8 * kVerifyThreads) {
      float x[8];
      load_floats<8>(p.logits, p.dtype, [&](int u) -> int64_t {
        const int e = e0 + u * kVerifyThreads;
        return e < n_el ? row + lo + e : -1;
      }, x);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int e = e0 + u * kVerifyThreads;
        if (e >= n_el) break;
        const float s = clean_logit(x[u]);
        cur[e] = s;
        if (s > m) {
          z = z * expf((m - s) * inv_t) + 1.f;
          m = s, idx = lo + e;
        } else if (s != -INFINITY) {
          z += expf((s - m) * inv_t);
        }
      }
    }
    const VerifyPart top = verify_exchange<true>(S, m, z, idx, cluster, round, inv_t);
    if (top.m == -INFINITY) break;  // nothing to choose from
    const float mx = top.m;
    if (greedy) {
      int child = -1;
      for (int c = node + 1; c < p.T && child < 0; ++c)
        if (S.par[c] == node && S.tok[c] == top.idx) child = c;
      if (child < 0) {
        token = top.idx;
        break;
      }
      node = child;
      ++n_acc;
      continue;
    }

    // r(x) = fresh ? exp(s - mx) / zr : cur / zr;  q(x) = draft * qs, or all on the child
    float zr = top.z, qs = 1.f;
    bool fresh = true;
    const int64_t drow = b * p.d_stride[0] + node * p.d_stride[1];
    int accepted = -1;
    for (int c = node + 1; c < p.T && accepted < 0; ++c) {
      if (S.par[c] != node) continue;
      const int tc = S.tok[c];
      const bool in_v = tc >= 0 && tc < p.V;
      float q = !p.draft_probs ? 1.f : in_v ? load_float(p.draft_probs, p.draft_dtype, drow + tc) * qs : 0.f;
      if (p.draft_probs)  // a token rejected before has no mass left
        for (int d = node + 1; d < c; ++d) q = S.par[d] == node && S.tok[d] == tc ? 0.f : q;
      float r = 0.f;
      if (fresh) {
        if (in_v) r = expf((clean_logit(load_float(p.logits, p.dtype, row + tc)) - mx) * inv_t) / zr;
      } else {  // its owner has it; everyone else adds zero
        const bool own_it = tc >= lo && tc < lo + n_el;
        r = verify_exchange<false>(S, 0.f, own_it && tid == 0 ? cur[tc - lo] : 0.f, 0, cluster, round).z / zr;
      }
      if (p.uniforms[(int64_t)b * p.T + c] * q < r) {
        accepted = c;
        break;
      }
      // rejected: w = max(r - q, 0) over the slice
      float zn = 0.f;
      for (int e = tid; e < n_el; e += kVerifyThreads) {
        const float rx = (fresh ? expf((cur[e] - mx) * inv_t) : cur[e]) / zr;
        const float qx = p.draft_probs ? load_float(p.draft_probs, p.draft_dtype, drow + lo + e) * qs
                                       : (lo + e == tc ? 1.f : 0.f);
        const float w = fmaxf(rx - qx, 0.f);
        nxt[e] = w;
        zn += w;
      }
      const VerifyPart sum = verify_exchange<false>(S, 0.f, zn, 0, cluster, round);
      if (sum.z > 0.f) {
        float* swap = cur;
        cur = nxt;
        nxt = swap;
        zr = sum.z;
        fresh = false;
      }
      if (p.draft_probs) qs = 1.f - q > 0.f ? qs / (1.f - q) : 0.f;
    }
    if (accepted >= 0) {
      node = accepted;
      ++n_acc;
      continue;
    }
    // the next token: the largest r / race
    float best = -INFINITY;
    int at = 0x7fffffff;
    for (int e = tid; e < n_el; e += kVerifyThreads) {
      const float rx = fresh ? expf((cur[e] - mx) * inv_t) : cur[e];
      const float sc = rx > 0.f ? rx / p.race[(int64_t)b * p.V + lo + e] : -INFINITY;
      if (sc > best) best = sc, at = lo + e;
    }
    const VerifyPart win = verify_exchange<false>(S, best, 0.f, at, cluster, round);
    token = win.idx < p.V ? win.idx : -1;
    break;
  }
  if (rank == 0 && tid == 0) {
    p.n_accepted[b] = n_acc;
    p.next_token[b] = token;
  }
  if (cluster > 1) cluster_sync_all();  // every CTA's shared memory stays until the last exchange is read
}

static int verify_max_cluster() {
  static int best[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 8;
  if (best[dev]) return best[dev];
  int n = 0, found = 8;
  const int smem = (int)sizeof(VerifySmem) + 8 * kVerifyMaxSlice;
  if (cudaFuncSetAttribute(tree_verify_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
      cudaFuncSetAttribute(tree_verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kVerifyMaxCluster);
    cfg.blockDim = dim3(kVerifyThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kVerifyMaxCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, tree_verify_kernel, &cfg) == cudaSuccess && n >= 1) found = kVerifyMaxCluster;
  }
  (void)cudaGetLastError();
  best[dev] = found;
  return found;
}

}  // namespace ns

extern "C" int ns_tree_verify(const ns_tree_verify_t* p, ns_stream_t stream) {
  using namespace ns;
  if (!p) return fail(NS_ERR_INVALID, "ns_tree_verify: null parameters");
  if (p->B < 0 || p->T < 1 || p->V < 1) return fail(NS_ERR_INVALID, "ns_tree_verify: B %d, T %d, V %d", p->B, p->T, p->V);
  if (!float_type_ok(p->dtype) || (p->draft_probs && !float_type_ok(p->draft_dtype)))
    return fail(NS_ERR_INVALID, "ns_tree_verify: bad dtype %d / %d", p->dtype, p->draft_dtype);
  if (p->T > kVerifyMaxNodes) return fail(NS_ERR_UNSUPPORTED, "ns_tree_verify: %d nodes (at most %d)", p->T, kVerifyMaxNodes);
  if (p->V > kVerifyMaxSlice * 8)
    return fail(NS_ERR_UNSUPPORTED, "ns_tree_verify: a vocabulary of %d (at most %d)", p->V, kVerifyMaxSlice * 8);
  if (p->B == 0) return NS_OK;
  if (!p->tokens || !p->logits || !p->uniforms || !p->race || !p->path || !p->n_accepted || !p->next_token)
    return fail(NS_ERR_INVALID, "ns_tree_verify: null pointer");
  int cluster = verify_max_cluster();
  while (cluster > 1 && p->V <= 1024 * (cluster / 2)) cluster /= 2;
  if ((int64_t)p->B * cluster > (1 << 30)) return fail(NS_ERR_UNSUPPORTED, "ns_tree_verify: %d sequences", p->B);
  VerifyArgs args;
  args.p = *p;
  args.slice = (p->V + cluster - 1) / cluster;
  const size_t smem = sizeof(VerifySmem) + 2 * sizeof(float) * (size_t)args.slice;
  NS_CUDA_TRY(cudaFuncSetAttribute(tree_verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)sizeof(VerifySmem) + 8 * kVerifyMaxSlice));
  NS_CUDA_TRY(launch_pdl(tree_verify_kernel, dim3((unsigned)(p->B * cluster)), kVerifyThreads, smem, stream, cluster, args,
                         cluster));
  return NS_OK;
}
