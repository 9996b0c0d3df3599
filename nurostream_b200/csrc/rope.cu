// ns_rope_append: rotary positions of new tokens and their append to the cache, one launch.
//
// Stands in for apply_rope (neurostream/compute/ops.py:136-151) and KVCache.append
// (neurostream/model/qwen3.py:74-85), for batches, drafted trees, partial and interleaved rotation:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin
// over the pairs of the first rotary_dim dims, the table row being the token's position.
//
// Pure traffic: q, k and v are read once and written once.  A thread owns one unit: U elements of
// each half (16 bytes of a 16-bit type), or U elements of an interleaved, passed-through or value
// row, so the partner of every element is in its registers.  U = 8 needs 16-byte aligned rows and
// a rotation that divides into such units; U = 1 (a pair of elements) takes everything else.
#include "tree.cuh"

namespace ns {

constexpr int kRopeThreads = 128;

// N consecutive elements of type DT at element i, widened / rounded.  N = 8: 16-byte accesses.
template <int DT, int N>
__device__ __forceinline__ void load_n(const void* p, int64_t i, float (&x)[N]) {
  if constexpr (N == 8 && DT == NS_F32) {
    const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = f[0], b = f[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else if constexpr (N == 8) {
    const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == NS_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        x[2 * j] = f.x, x[2 * j + 1] = f.y;
      } else {
        x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = load_float(p, DT, i + j);
  }
}

template <int N>
__device__ __forceinline__ void store_n(void* p, int dt, int64_t i, const float (&x)[N]) {
  if constexpr (N == 8) {
    if (dt == NS_F32) {
      float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
      f[0] = make_float4(x[0], x[1], x[2], x[3]);
      f[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (dt == NS_F16) {
          const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) store_float(p, dt, i + j, x[j]);
  }
}

template <int DT, int U>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ ns_rope_append_t p) {
  const int lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch_dependents();
  // units of one head: rotating ones (pairs or octets), then passed-through ones
  const int half = p.rotary_dim / 2;
  const int pair = U == 8 ? 8 : 2;  // elements of an interleaved unit
  const int n_rot = p.interleaved ? p.rotary_dim / pair : half / U;
  const int n_head_units = n_rot + (p.head_dim - p.rotary_dim) / U, n_val_units = p.head_dim / U;
  const int nq = p.q ? p.n_head * n_head_units : 0, nk = p.k ? p.n_head_kv * n_head_units : 0;
  const int nv = p.v ? p.n_head_kv * n_val_units : 0;

  for (int64_t tok = blockIdx.y; tok < (int64_t)p.B * p.T; tok += gridDim.y) {
    const int b = (int)(tok / p.T), t = (int)(tok % p.T);
    const int len = tree_len(p.lens, b, p.max_ctx);
    int depth = t;
    bool used = true, bad = len < 0;
    if (p.parents) {  // the warp holds the sequence's parents, two per lane; the walk is shuffles
      const int32_t* par = p.parents + (int64_t)b * p.T;
      const int p0 = lane < p.T ? par[lane] : -2, p1 = lane + 32 < p.T ? par[lane + 32] : -2;
      const uint64_t m = tree_mask(t, [&](int i) {
        const int lo = __shfl_sync(0xffffffffu, p0, i & 31), hi = __shfl_sync(0xffffffffu, p1, i & 31);
        return i < 32 ? lo : hi;
      }, &bad);
      used = m != 0;
      depth = __popcll(m) - 1;
    }
    const int64_t slot = (int64_t)len + t;
    if (used && slot >= p.max_ctx && (p.k || p.v)) bad = true;
    int64_t pos = used ? (int64_t)len + depth : 0;
    if (used && p.positions) pos = p.positions[tok];
    if (used && (pos < 0 || pos >= p.n_pos)) bad = true;
    if (bad) {
      used = false;
      if (threadIdx.x == 0 && blockIdx.x == 0) raise_device_error(NS_DEVERR_ROUTE);
    }
    const float* cs = p.rope_cos + pos * p.table_stride;
    const float* sn = p.rope_sin + pos * p.table_stride;

    for (int i = blockIdx.x * kRopeThreads + threadIdx.x; i < nq + nk + nv; i += gridDim.x * kRopeThreads) {
      if (i >= nq && !used) continue;
      const void* src;
      void* dst;
      int64_t so, dofs;
      int u, dt = DT;
      if (i < nq) {
        const int h = i / n_head_units;
        u = i % n_head_units;
        src = p.q, dst = p.q_out;
        so = b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2];
        dofs = b * p.qo_stride[0] + t * p.qo_stride[1] + h * p.qo_stride[2];
      } else if (i < nq + nk) {
        const int h = (i - nq) / n_head_units;
        u = (i - nq) % n_head_units;
        src = p.k, dst = p.k_cache, dt = p.cache_dtype;
        so = b * p.k_stride[0] + t * p.k_stride[1] + h * p.k_stride[2];
        dofs = b * p.kc_stride[0] + h * p.kc_stride[1] + slot * p.kc_stride[2];
      } else {
        const int h = (i - nq - nk) / n_val_units;
        u = (i - nq - nk) % n_val_units;
        so = b * p.v_stride[0] + t * p.v_stride[1] + h * p.v_stride[2] + u * U;
        dofs = b * p.vc_stride[0] + h * p.vc_stride[1] + slot * p.vc_stride[2] + u * U;
        float x[U];
        load_n<DT, U>(p.v, so, x);
        store_n<U>(p.v_cache, p.cache_dtype, dofs, x);
        continue;
      }
      if (u >= n_rot) {  // passed through
        const int d = p.rotary_dim + (u - n_rot) * U;
        float x[U];
        load_n<DT, U>(src, so + d, x);
#pragma unroll
        for (int j = 0; j < U; ++j) x[j] = used ? x[j] : 0.f;
        store_n<U>(dst, dt, dofs + d, x);
      } else if (p.interleaved) {
        constexpr int N = U == 8 ? 8 : 2;
        float x[N], c[N / 2], s[N / 2];
        load_n<DT, N>(src, so + u * N, x);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) c[j] = cs[u * (N / 2) + j], s[j] = sn[u * (N / 2) + j];
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          const float a = x[2 * j], d = x[2 * j + 1];
          x[2 * j] = used ? a * c[j] - d * s[j] : 0.f;
          x[2 * j + 1] = used ? d * c[j] + a * s[j] : 0.f;
        }
        store_n<N>(dst, dt, dofs + u * N, x);
      } else {
        float x[U], y[U], c[U], s[U];
        load_n<DT, U>(src, so + u * U, x);
        load_n<DT, U>(src, so + half + u * U, y);
        load_n<NS_F32, U>(cs, u * U, c);
        load_n<NS_F32, U>(sn, u * U, s);
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const float a = x[j], d = y[j];
          x[j] = used ? a * c[j] - d * s[j] : 0.f;
          y[j] = used ? d * c[j] + a * s[j] : 0.f;
        }
        store_n<U>(dst, dt, dofs + u * U, x);
        store_n<U>(dst, dt, dofs + half + u * U, y);
      }
    }
  }
}

template <int DT>
static cudaError_t rope_launch(const ns_rope_append_t& p, bool vec, ns_stream_t stream) {
  const int U = vec ? 8 : 1;
  const int n_rot = p.interleaved ? p.rotary_dim / (vec ? 8 : 2) : p.rotary_dim / 2 / U;
  const int head_units = n_rot + (p.head_dim - p.rotary_dim) / U;
  const int units = (p.q ? p.n_head * head_units : 0) + (p.k ? p.n_head_kv * head_units : 0) +
                    (p.v ? p.n_head_kv * (p.head_dim / U) : 0);
  const int64_t tokens = (int64_t)p.B * p.T;
  dim3 grid((unsigned)((units + kRopeThreads - 1) / kRopeThreads), (unsigned)std::min<int64_t>(tokens, 65535));
  return vec ? launch_pdl(rope_append_kernel<DT, 8>, grid, kRopeThreads, 0, stream, 1, p)
             : launch_pdl(rope_append_kernel<DT, 1>, grid, kRopeThreads, 0, stream, 1, p);
}

}  // namespace ns

extern "C" int ns_rope_append(const ns_rope_append_t* p, ns_stream_t stream) {
  using namespace ns;
  if (!p) return fail(NS_ERR_INVALID, "ns_rope_append: null parameters");
  if (p->B < 0 || p->T < 0) return fail(NS_ERR_INVALID, "ns_rope_append: B %d, T %d", p->B, p->T);
  if (!float_type_ok(p->dtype) || !float_type_ok(p->cache_dtype))
    return fail(NS_ERR_INVALID, "ns_rope_append: bad dtype %d / %d", p->dtype, p->cache_dtype);
  if (p->head_dim < 1 || p->rotary_dim < 0 || p->rotary_dim > p->head_dim || p->rotary_dim % 2)
    return fail(NS_ERR_INVALID, "ns_rope_append: rotary_dim %d of head_dim %d (even, at most head_dim)", p->rotary_dim,
                p->head_dim);
  if (p->n_head < 0 || p->n_head_kv < 0 || p->max_ctx < 0 || p->n_pos < 0)
    return fail(NS_ERR_INVALID, "ns_rope_append: negative head count, max_ctx or n_pos");
  if (p->parents && p->T > NS_TREE_MAX_NODES)
    return fail(NS_ERR_UNSUPPORTED, "ns_rope_append: a tree of %d nodes (at most %d)", p->T, NS_TREE_MAX_NODES);
  if (p->B == 0 || p->T == 0) return NS_OK;
  if (!p->lens || !p->rope_cos || !p->rope_sin) return fail(NS_ERR_INVALID, "ns_rope_append: null lens or tables");
  if ((p->q && !p->q_out) || (p->k && !p->k_cache) || (p->v && !p->v_cache))
    return fail(NS_ERR_INVALID, "ns_rope_append: an input without its output");
  if ((int64_t)(p->n_head + 2 * (int64_t)p->n_head_kv) * p->head_dim > (1 << 28))
    return fail(NS_ERR_UNSUPPORTED, "ns_rope_append: %d + 2 x %d heads of %d", p->n_head, p->n_head_kv, p->head_dim);
  if ((!p->q || !p->n_head) && ((!p->k && !p->v) || !p->n_head_kv)) return NS_OK;
  // 16-byte units where every row starts on 16 bytes and the rotation divides into them
  const int64_t m = p->dtype == NS_F32 ? 4 : 8, mc = p->cache_dtype == NS_F32 ? 4 : 8;
  bool vec = p->head_dim % 8 == 0 && p->rotary_dim % (p->interleaved ? 8 : 16) == 0 && p->table_stride % 4 == 0 &&
             aligned_to(p->rope_cos, 16) && aligned_to(p->rope_sin, 16);
  if (p->q)
    vec = vec && aligned_to(p->q, 16) && aligned_to(p->q_out, 16) && strides_multiple(p->q_stride, 3, m) &&
          strides_multiple(p->qo_stride, 3, m);
  if (p->k)
    vec = vec && aligned_to(p->k, 16) && aligned_to(p->k_cache, 16) && strides_multiple(p->k_stride, 3, m) &&
          strides_multiple(p->kc_stride, 3, mc);
  if (p->v)
    vec = vec && aligned_to(p->v, 16) && aligned_to(p->v_cache, 16) && strides_multiple(p->v_stride, 3, m) &&
          strides_multiple(p->vc_stride, 3, mc);
  switch (p->dtype) {
    case NS_F32: NS_CUDA_TRY(rope_launch<NS_F32>(*p, vec, stream)); break;
    case NS_F16: NS_CUDA_TRY(rope_launch<NS_F16>(*p, vec, stream)); break;
    default: NS_CUDA_TRY(rope_launch<NS_BF16>(*p, vec, stream)); break;
  }
  return NS_OK;
}
