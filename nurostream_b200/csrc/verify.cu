// ns_tree_verify: walk of a drafted tree against the target's logits, from given random numbers.
// No reference counterpart (it decodes greedily, one token a step).
//
// The walk is serial (which row comes next depends on what was accepted), a row is V logits, and a
// tree's rows are mostly never looked at: only the rows of the nodes that the walk stands on are read.
// One thread-block cluster walks one sequence; CTA r of it holds slice r of the vocabulary.  A row
// costs one pass (logits into shared memory, running maximum, sum of exponentials and lowest index of
// the maximum per thread) and one exchange through distributed shared memory; every CTA then holds
// the row's maximum and sum, and takes the same decisions from the same bits.  While the decisions are
// made, the rows they may need next (the first child's logits, the draft's, the race) come into L2.  With
//   r_0 = p = exp(s - m) / Z,  q_0 = q,
//   rejecting c:  w = max(r_j - q_j, 0),  z = sum w,  r_{j+1} = w / z,  q_{j+1} = q_j / (1 - q_j(c)), q_{j+1}(c) = 0,
// a rejection costs a pass over the slice and an exchange of z, or, when no child is left, nothing of its
// own: the pass that draws the token takes it out.  r at the other children follows by the same steps
// on scalars.  (c needs no zero in the slice's q: w(c) = 0, since it was rejected with u < 1, and stays 0.)
// Measured (device time of a call in a captured graph, vocabulary of 201,088): one chain of 8 nodes, fp32,
// 12.8 us (two rows and the race: 2.4 MB); 16 trees of 32 nodes, bf16 logits and fp32 draft, 58 us, as long
// as the longest walk among them.  A step of a walk is a pass of 4 to 7 thousand cycles (one load's latency,
// then about ten instructions a logit) and an exchange of 2.5 to 3.5 thousand (reductions, cluster
// barrier, remote reads): both are latency, the bytes would take a tenth.
// The next token maximises r(x) / race(x): scores, unlike a cumulative sum over the vocabulary, do not
// depend on the order of a summation.
#include "tree.cuh"

namespace ns {

constexpr int kVerifyThreads = 512;
constexpr int kVerifyMaxCluster = 16;
constexpr int kVerifyMaxSlice = 25600;  // logits of one CTA: two fp32 buffers of it in shared memory
constexpr int kVerifyMaxNodes = 1024;
constexpr int kVerifyUnits = 2;         // loads of four values that a thread keeps in flight, of each row
constexpr int kVerifyRowUnits = 4;      // and where there is one row (more of either spills)

struct VerifyPart {  // one CTA's part of an exchange
  float m, z;
  int idx, pad;
};

struct VerifySmem {
  VerifyPart part[2];                       // by parity of the exchange, read by the whole cluster
  VerifyPart all[2];                        // its outcome, for this CTA's threads
  float red_m[kVerifyThreads / 32], red_z[kVerifyThreads / 32];
  int red_i[kVerifyThreads / 32];
};

struct VerifyArgs {
  ns_tree_verify_t p;
  int slice;      // a multiple of 8
  int cluster;
};

// Shared memory after VerifySmem: two slices, then per node its token, parent, uniform number, logit, draft
// probability, first child and next sibling.
static size_t verify_smem_bytes(int slice, int T) {
  return sizeof(VerifySmem) + 2 * sizeof(float) * (size_t)slice + 6 * sizeof(float) * (size_t)((T + 3) / 4 * 4);
}

__device__ __forceinline__ float clean_logit(float x) {
  return fminf(fmaxf(x, -INFINITY), 3.402823466e38f);  // (a NaN loses to any number)
}

// Four consecutive values of a row from element i on, 0 past `n`; vec: i is on 16 (8) bytes.
__device__ __forceinline__ void load_row4(const void* p, int dtype, int64_t i, bool vec, int n, float (&x)[4]) {
  if (vec && n >= 4) {
    if (dtype == NS_F32) {
      const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
      if (dtype == NS_F16) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
      } else {
        x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xFFFF0000u);
        x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xFFFF0000u);
      }
    }
  } else {
    load_floats<4>(p, dtype, [&](int u) -> int64_t { return u < n ? i + u : -1; }, x);
  }
}
__device__ __forceinline__ bool row_vec(const void* p, int dtype, int64_t i) {
  return (reinterpret_cast<uintptr_t>(p) + i * (dtype == NS_F32 ? 4 : 2)) % (dtype == NS_F32 ? 16 : 8) == 0;
}

// A row's slice asked into L2: whole lines, a thread each.
__device__ __forceinline__ void verify_prefetch(const void* p, int dtype, int64_t i, int n) {
  const int es = dtype == NS_F32 ? 4 : 2;
  const char* c = static_cast<const char*>(p) + i * es;
  for (int64_t o = (int64_t)threadIdx.x * 128; o < (int64_t)n * es; o += kVerifyThreads * 128)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(c + o));
}

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Outcome over a warp of parts (m, z, i): m the maximum, i the lowest index that has it, z the sum, with
// SCALED each scaled from its own maximum to m (c: log2 e over the temperature).
template <bool SCALED>
__device__ __forceinline__ void verify_combine(float& m, float& z, int& i, float c) {
  const float top = warp_max(m);
  if (SCALED && top != -INFINITY) z *= ex2((m - top) * c);
  z = warp_sum(z);
  i = (int)__reduce_min_sync(0xffffffffu, m == top ? (unsigned)i : 0x7fffffffu);
  m = top;
}

// The outcome over the cluster, the same bits in every CTA.
template <bool SCALED>
__device__ __forceinline__ VerifyPart verify_exchange(VerifySmem& S, float m, float z, int i, int cluster, int& round,
                                                      float c = 1.f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  verify_combine<SCALED>(m, z, i, c);
  if (lane == 0) S.red_m[warp] = m, S.red_z[warp] = z, S.red_i[warp] = i;
  __syncthreads();
  VerifyPart& mine = S.part[round & 1];
  if (warp == 0) {
    const bool has = lane < kVerifyThreads / 32;
    m = has ? S.red_m[lane] : -INFINITY, z = has ? S.red_z[lane] : 0.f, i = has ? S.red_i[lane] : 0x7fffffff;
    verify_combine<SCALED>(m, z, i, c);
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
      verify_combine<SCALED>(m, z, i, c);
    }
  }
  VerifyPart& all = S.all[round & 1];
  if (threadIdx.x == 0) all = VerifyPart{m, z, i, 0};
  __syncthreads();
  ++round;
  return all;
}

__global__ void __launch_bounds__(kVerifyThreads, 2) tree_verify_kernel(const __grid_constant__ VerifyArgs a) {
  const ns_tree_verify_t& p = a.p;
  extern __shared__ __align__(16) uint8_t verify_smem[];
  VerifySmem& S = *reinterpret_cast<VerifySmem*>(verify_smem);
  float* cur = reinterpret_cast<float*>(verify_smem + sizeof(VerifySmem));  // the row's logits, then r times zr
  float* nxt = cur + a.slice;
  const int n_pad = (p.T + 3) / 4 * 4;
  int* s_tok = reinterpret_cast<int*>(nxt + a.slice);
  int* s_par = s_tok + n_pad;
  float* s_uni = reinterpret_cast<float*>(s_par + n_pad);
  float* s_log = s_uni + n_pad;   // of the children of the node at hand: their logit there
  float* s_drf = s_log + n_pad;   // and draft probability
  int16_t* s_kid = reinterpret_cast<int16_t*>(s_drf + n_pad);  // a node's first child, -1: none
  int16_t* s_sib = s_kid + n_pad;                              // its next sibling
  const int tid = threadIdx.x, cluster = a.cluster;
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int b = blockIdx.x / cluster;
  const int lo = min(p.V, rank * a.slice), n_el = min(p.V, lo + a.slice) - lo, n_unit = (n_el + 3) / 4;
  griddep_wait();
  griddep_launch_dependents();

  verify_prefetch(p.race, NS_F32, (int64_t)b * p.V + lo, n_el);  // the walk's last pass reads it
  for (int t = tid; t < p.T; t += kVerifyThreads) {
    s_tok[t] = p.tokens[(int64_t)b * p.T + t];
    s_par[t] = p.parents ? p.parents[(int64_t)b * p.T + t] : t - 1;
    s_uni[t] = p.uniforms[(int64_t)b * p.T + t];
    if (rank == 0) p.path[(int64_t)b * p.T + t] = t == 0 ? 0 : -1;
  }
  const float temp = p.temperature ? p.temperature[b] : 1.f;
  const bool greedy = temp == 0.f;
  // exp(x / temperature) = 2^(c x), c finite: a subnormal temperature would make it infinite, and the maximum's
  // own distance of zero NaN
  const float cf = greedy ? 1.f : 1.4426950408889634f / fmaxf(temp, 1.17549435e-38f);
  __syncthreads();
  for (int t = tid; t < p.T; t += kVerifyThreads) {  // the tree as lists of children in node order
    int kid = -1, sib = -1;
    for (int d = p.T - 1; d > t; --d) {
      kid = s_par[d] == t ? d : kid;
      sib = s_par[d] == s_par[t] ? d : sib;
    }
    s_kid[t] = (int16_t)kid;
    s_sib[t] = (int16_t)sib;
    // a parent out of order, below -2 or unused: the walk never comes to the node, but the tree is wrong
    const int up = s_par[t];
    if (rank == 0 && (up >= t || up < -2 || (up >= 0 && s_par[up] == -2))) raise_device_error(NS_DEVERR_ROUTE);
  }
  __syncthreads();
  const bool root_ok = s_par[0] == -1;
  if (!root_ok && tid == 0 && rank == 0) {
    raise_device_error(NS_DEVERR_ROUTE);
    p.path[(int64_t)b * p.T] = -1;
  }

  int node = 0, n_acc = 0, token = -1, round = 0;
  while (root_ok) {
    const int64_t row = b * p.l_stride[0] + node * p.l_stride[1], drow = b * p.d_stride[0] + node * p.d_stride[1];
    // the row: its slice to shared memory, maximum (lowest index) and sum of exponentials
    float m = -INFINITY, z = 0.f;
    int idx = 0x7fffffff;
    const bool lvec = row_vec(p.logits, p.dtype, row + lo);
    for (int e0 = tid; e0 < n_unit; e0 += kVerifyRowUnits * kVerifyThreads) {
      float x[kVerifyRowUnits][4];
#pragma unroll
      for (int u = 0; u < kVerifyRowUnits; ++u) {
        const int e = (e0 + u * kVerifyThreads) * 4;
        if (e < n_el) load_row4(p.logits, p.dtype, row + lo + e, lvec, n_el - e, x[u]);
      }
#pragma unroll
      for (int u = 0; u < kVerifyRowUnits; ++u) {
        const int e = (e0 + u * kVerifyThreads) * 4;
        if (e >= n_el) break;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[u][k] = e + k < n_el ? clean_logit(x[u][k]) : -INFINITY;
        *reinterpret_cast<float4*>(cur + e) = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
        const float top = fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3]));
        if (top > m) {
          z *= ex2((m - top) * cf);
          m = top;
          if (greedy) idx = lo + e + (x[u][0] == top ? 0 : x[u][1] == top ? 1 : x[u][2] == top ? 2 : 3);
        }
        if (greedy || m == -INFINITY) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k) z += ex2((x[u][k] - m) * cf);
      }
    }
    // what the decisions need of the children
    const int first_kid = s_kid[node];
    for (int c = node + 1 + tid; c < p.T; c += kVerifyThreads)
      if (s_par[c] == node) {
        const int t = s_tok[c];
        const bool in_v = t >= 0 && t < p.V;
        s_log[c] = in_v ? clean_logit(load_float(p.logits, p.dtype, row + t)) : -INFINITY;
        s_drf[c] = !p.draft_probs ? 1.f : in_v ? load_float(p.draft_probs, p.draft_dtype, drow + t) : 0.f;
      }
    if (!greedy && first_kid >= 0) {
      if (p.draft_probs) verify_prefetch(p.draft_probs, p.draft_dtype, drow + lo, n_el);
      verify_prefetch(p.logits, p.dtype, b * p.l_stride[0] + first_kid * p.l_stride[1] + lo, n_el);
    }
    const VerifyPart top = verify_exchange<true>(S, m, z, idx, cluster, round, cf);
    if (top.m == -INFINITY) break;  // nothing to choose from
    const float mx = top.m;
    int took = -1;
    if (greedy) {
      for (int c = first_kid; c >= 0 && took < 0; c = s_sib[c])
        if (s_tok[c] == top.idx) took = c;
      if (took < 0) {
        token = top.idx;
        break;
      }
    } else {
      // r(x) = (fresh ? 2^((cur - mx) cf) : cur) / zr;  q(x) = draft * qs, or all on the child
      float zr = top.z, qs = 1.f;
      bool fresh = true;
      int last = -1;  // the child whose rejection is still to be taken out of r
      float last_q = 0.f;
      const bool dvec = p.draft_probs && row_vec(p.draft_probs, p.draft_dtype, drow + lo);
      // one pass over the slice, four values at a time: r as it stands, and max(r - q, 0)
      auto pass = [&](bool with_q, const float* aux, auto&& body) {
        const float rz = 1.f / zr;
        const bool avec = aux && row_vec(aux, NS_F32, 0);
        for (int e0 = tid; e0 < n_unit; e0 += kVerifyUnits * kVerifyThreads) {
          float q[kVerifyUnits][4], y[kVerifyUnits][4];
#pragma unroll
          for (int u = 0; u < kVerifyUnits; ++u) {
            const int e = (e0 + u * kVerifyThreads) * 4;
            if (with_q && p.draft_probs && e < n_el) load_row4(p.draft_probs, p.draft_dtype, drow + lo + e, dvec, n_el - e, q[u]);
          }
#pragma unroll
          for (int u = 0; u < kVerifyUnits; ++u) {
            const int e = (e0 + u * kVerifyThreads) * 4;
            if (aux && e < n_el) load_row4(aux, NS_F32, e, avec, n_el - e, y[u]);
          }
#pragma unroll
          for (int u = 0; u < kVerifyUnits; ++u) {
            const int e = (e0 + u * kVerifyThreads) * 4;
            if (e >= n_el) break;
            const float4 c = *reinterpret_cast<const float4*>(cur + e);
            float w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              w[k] = (fresh ? ex2((w[k] - mx) * cf) : w[k]) * rz;
              if (with_q) w[k] = fmaxf(w[k] - (p.draft_probs ? q[u][k] * qs : lo + e + k == s_tok[last] ? 1.f : 0.f), 0.f);
              if (e + k >= n_el) w[k] = 0.f;
            }
            body(e, w, y[u]);
          }
        }
      };
      for (int c = first_kid; c >= 0; c = s_sib[c]) {
        if (last >= 0) {  // the rejection before this child: w = max(r - q, 0) and its sum
          float zn = 0.f;
          pass(true, nullptr, [&](int e, const float (&w)[4], const float (&)[4]) {
            *reinterpret_cast<float4*>(nxt + e) = make_float4(w[0], w[1], w[2], w[3]);
            zn += (w[0] + w[1]) + (w[2] + w[3]);
          });
          const VerifyPart sum = verify_exchange<false>(S, 0.f, zn, 0, cluster, round);
          // r at the children still to come, by the same steps
          for (int d = c + tid; d < p.T; d += kVerifyThreads)
            if (s_par[d] == node) {
              const float r = (fresh ? ex2((s_log[d] - mx) * cf) : s_log[d]) * (1.f / zr);
              const float q = p.draft_probs ? s_drf[d] * qs : s_tok[d] == s_tok[last] ? 1.f : 0.f;
              if (sum.z > 0.f) s_log[d] = fmaxf(r - q, 0.f);
            }
          if (sum.z > 0.f) {
            float* swap = cur;
            cur = nxt;
            nxt = swap;
            zr = sum.z;
            fresh = false;
          }
          if (p.draft_probs) qs = 1.f - last_q > 0.f ? qs / (1.f - last_q) : 0.f;
          last = -1;
          __syncthreads();
        }
        const float r = (fresh ? ex2((s_log[c] - mx) * cf) : s_log[c]) * (1.f / zr);
        float q = s_drf[c] * qs;
        if (p.draft_probs)  // a token rejected before has no mass left
          for (int d = first_kid; d < c; d = s_sib[d]) q = s_tok[d] == s_tok[c] ? 0.f : q;
        if (s_uni[c] * q < r) {
          took = c;
          break;
        }
        last = c, last_q = q;
      }
      if (took < 0) {
        // the next token: the largest r / race, the last rejection taken out on the way; when it leaves
        // nothing, r as it was
        for (int with_q = last >= 0; with_q >= 0; --with_q) {
          float best = -INFINITY;
          int at = 0x7fffffff;
          pass(with_q != 0, p.race + (int64_t)b * p.V + lo, [&](int e, const float (&w)[4], const float (&x)[4]) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float sc = w[k] > 0.f ? __fdividef(w[k], x[k]) : -INFINITY;
              if (sc > best) best = sc, at = lo + e + k;
            }
          });
          const VerifyPart win = verify_exchange<false>(S, best, 0.f, at, cluster, round);
          token = win.idx < p.V ? win.idx : -1;
          if (token >= 0) break;
        }
        break;
      }
    }
    node = took;
    ++n_acc;
    if (rank == 0 && tid == 0) p.path[(int64_t)b * p.T + n_acc] = node;
    __syncthreads();  // the children's values and the slice are written anew
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
  const int smem = (int)verify_smem_bytes(kVerifyMaxSlice, 64);
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
  // 4096 logits of a CTA at the least: below that the exchanges cost more than the passes (vocabulary of 4000,
  // 16 chains: one CTA 20.2 us, four 24.1; of 32000: 8 CTAs 29.3, 16 32.2; of 201088: 8 CTAs 68.4, 16 52.0)
  while (cluster > 1 && p->V <= 4096 * (cluster / 2)) cluster /= 2;
  if ((int64_t)p->B * cluster > (1 << 30)) return fail(NS_ERR_UNSUPPORTED, "ns_tree_verify: %d sequences", p->B);
  VerifyArgs args;
  args.p = *p;
  args.cluster = cluster;
  args.slice = ((p->V + cluster - 1) / cluster + 7) / 8 * 8;
  const size_t smem = verify_smem_bytes(args.slice, p->T);
  NS_CUDA_TRY(cudaFuncSetAttribute(tree_verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)verify_smem_bytes(kVerifyMaxSlice, kVerifyMaxNodes)));
  NS_CUDA_TRY(launch_pdl(tree_verify_kernel, dim3((unsigned)(p->B * cluster)), kVerifyThreads, smem, stream, cluster, args));
  return NS_OK;
}
