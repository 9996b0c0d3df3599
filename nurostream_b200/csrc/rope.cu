// ns_rope_append: rotary positions of new tokens and their append to the cache, one launch.
//
// Stands in for apply_rope (neurostream/compute/ops.py:136-151) and KVCache.append
// (neurostream/model/qwen3.py:74-85), for batches, drafted trees, partial and interleaved rotation:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin
// over the pairs of the first rotary_dim dims, the table row being the token's position.
//
// Pure traffic: q, k and v are read once and written once; what costs beside it are index arithmetic and
// the table.  A unit is two octets of a row, with 8 whole pairs in it where it rotates, so the partner of
// every element is in the thread's registers.  A thread keeps one unit of the row and takes it through
// the heads of one token: one table slice, one division, for all of them.  The heads' elements are read
// before the token's position is known (length, then depth in the tree, then the table's row: each
// waits for the one before).  Rows that do not divide into octets on 16 bytes go pair by pair.
// Measured (device time of a call in a captured graph, 80 heads): one token, fp32, 2.7 us; 528 tree tokens
// of 128 dims, bf16, 7.7 us (2.8 TB/s); 4,098 prompt tokens 41 us (4.1 TB/s, where a copy has 6.5): bound by
// issue (300 instructions a unit before the addresses ran along) and by blocks that live for one
// token; blocks that stay and fetch the next token ahead by cp.async were slower (48 us).
#include <type_traits>

#include "tree.cuh"

namespace ns {

constexpr int kRopeThreads = 128;

// Eight consecutive values rounded to type dt at element i, on 16 bytes.
__device__ __forceinline__ void store8(void* p, int dt, int64_t i, const float (&x)[8]) {
  if (dt == NS_F32) {
    float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    f[0] = make_float4(x[0], x[1], x[2], x[3]);
    f[1] = make_float4(x[4], x[5], x[6], x[7]);
    return;
  }
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

// Eight values of type DT from their registers.
template <int DT>
__device__ __forceinline__ void widen8(const uint4* v, float (&x)[8]) {
  if constexpr (DT == NS_F32) {
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(w[j]);
  } else {
    const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == NS_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        x[2 * j] = f.x, x[2 * j + 1] = f.y;
      } else {
        x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
}

// Where token t of sequence b stands: its cache slot, its table row, and whether it is used at all.  The
// whole warp calls it (the walk up the tree is shuffles: the warp holds the parents, two per lane).
struct RopeAt {
  int64_t slot, pos;
  bool used;
};
__device__ __forceinline__ RopeAt rope_at_token(const ns_rope_append_t& p, int64_t tok, int b, int t) {
  const int lane = threadIdx.x & 31;
  const int len = tree_len(p.lens, b, p.max_ctx);
  int depth = t;
  bool used = true, bad = len < 0;
  if (p.parents) {
    const int32_t* par = p.parents + (int64_t)b * p.T;
    const int p0 = lane < p.T ? par[lane] : -2, p1 = lane + 32 < p.T ? par[lane + 32] : -2;
    const uint64_t m = tree_mask(t, [&](int i) { return __shfl_sync(0xffffffffu, i < 32 ? p0 : p1, i & 31); }, &bad);
    used = m != 0;
    depth = __popcll(m) - 1;
  }
  RopeAt at;
  at.slot = (int64_t)len + t;
  if (used && at.slot >= p.max_ctx && (p.k || p.v)) bad = true;
  at.pos = used ? (int64_t)len + depth : 0;
  if (used && p.positions) at.pos = p.positions[tok];
  if (used && (at.pos < 0 || at.pos >= p.n_pos)) bad = true;
  if (bad) {
    used = false;
    if (threadIdx.x == 0 && blockIdx.x == 0) raise_device_error(NS_DEVERR_ROUTE);
  }
  at.used = used;
  if (!used) at.pos = 0;
  return at;
}

constexpr int kRopeRowThreads = 256;

// NU: heads a thread reads side by side (gridDim.x > 1 shares a token's heads out when tokens are few).
// CT: type of the caches.  The index arithmetic of a row is as long as its rotation, so the addresses of
// the three kinds of rows run along and a row picks its own.
template <int DT, int CT, bool INTER, int NU>
__global__ void __launch_bounds__(kRopeRowThreads) rope_rows_kernel(const __grid_constant__ ns_rope_append_t p) {
  constexpr int ES = DT == NS_F32 ? 4 : 2, CS = CT == NS_F32 ? 4 : 2;
  const int per = p.head_dim / 16, n_rot = p.rotary_dim / 16;  // units of a row, and the rotating ones
  const int row0 = threadIdx.x / per, u = threadIdx.x % per, step = kRopeRowThreads / per;
  const int nq = p.q ? p.n_head : 0, nk = p.k ? p.n_head_kv : 0, nv = p.v ? p.n_head_kv : 0, rows = nq + nk + nv;
  const bool rotates = u < n_rot;
  // first elements of the unit's octets
  const int d0 = !rotates || INTER ? 16 * u : 8 * u, d1 = !rotates || INTER ? 16 * u + 8 : p.rotary_dim / 2 + 8 * u;
  const int first_row = row0 + blockIdx.x * step * NU, jump = step * NU * gridDim.x;
  griddep_wait();
  griddep_launch_dependents();
  for (int64_t tok = blockIdx.y; tok < (int64_t)p.B * p.T; tok += gridDim.y) {
    const int b = (int)(tok / p.T), t = (int)(tok % p.T);
    // the row of each kind at index first_row of the list (q, k, v), and the way to the next
    const char* qs = static_cast<const char*>(p.q) + (b * p.q_stride[0] + t * p.q_stride[1] + first_row * p.q_stride[2] + d0) * ES;
    const char* ks = static_cast<const char*>(p.k) + (b * p.k_stride[0] + t * p.k_stride[1] + (first_row - nq) * p.k_stride[2] + d0) * ES;
    const char* vs = static_cast<const char*>(p.v) + (b * p.v_stride[0] + t * p.v_stride[1] + (first_row - nq - nk) * p.v_stride[2] + d0) * ES;
    const int64_t qstep = step * p.q_stride[2] * ES, kstep = step * p.k_stride[2] * ES, vstep = step * p.v_stride[2] * ES;
    const int64_t ostep = step * p.qo_stride[2] * ES, kcstep = step * p.kc_stride[1] * CS, vcstep = step * p.vc_stride[1] * CS;
    char *qd = nullptr, *kd = nullptr, *vd = nullptr;
    bool first = true;
    RopeAt at{0, 0, false};
    float c[8], s[8];
    for (int r0 = first_row; r0 - row0 < rows; r0 += jump) {
      uint4 raw[NU][DT == NS_F32 ? 4 : 2];
#pragma unroll
      for (int k = 0; k < NU; ++k) {
        const int r = r0 + k * step;
        const char* f = r < nq ? qs : r < nq + nk ? ks : vs;
        qs += qstep, ks += kstep, vs += vstep;
        if (row0 >= step || r >= rows) continue;
        const char* f1 = f + (d1 - d0) * ES;
        if constexpr (DT == NS_F32) {
          raw[k][0] = *reinterpret_cast<const uint4*>(f), raw[k][1] = *reinterpret_cast<const uint4*>(f + 16);
          raw[k][2] = *reinterpret_cast<const uint4*>(f1), raw[k][3] = *reinterpret_cast<const uint4*>(f1 + 16);
        } else {
          raw[k][0] = *reinterpret_cast<const uint4*>(f), raw[k][1] = *reinterpret_cast<const uint4*>(f1);
        }
      }
      if (gridDim.x > 1) qs += (jump / step - NU) * qstep, ks += (jump / step - NU) * kstep, vs += (jump / step - NU) * vstep;
      if (first) {
        first = false;
        at = rope_at_token(p, tok, b, t);
        if (rotates) {
          const uint4* ct = reinterpret_cast<const uint4*>(p.rope_cos + at.pos * p.table_stride + 8 * u);
          const uint4* st = reinterpret_cast<const uint4*>(p.rope_sin + at.pos * p.table_stride + 8 * u);
          const uint4 cr[2] = {ct[0], ct[1]}, sr[2] = {st[0], st[1]};
          widen8<NS_F32>(cr, c);
          widen8<NS_F32>(sr, s);
        }
        qd = static_cast<char*>(p.q_out) + (b * p.qo_stride[0] + t * p.qo_stride[1] + first_row * p.qo_stride[2] + d0) * ES;
        kd = static_cast<char*>(p.k_cache) + (b * p.kc_stride[0] + (first_row - nq) * p.kc_stride[1] + at.slot * p.kc_stride[2] + d0) * CS;
        vd = static_cast<char*>(p.v_cache) + (b * p.vc_stride[0] + (first_row - nq - nk) * p.vc_stride[1] + at.slot * p.vc_stride[2] + d0) * CS;
      }
#pragma unroll
      for (int k = 0; k < NU; ++k) {
        const int r = r0 + k * step;
        char* dst = r < nq ? qd : r < nq + nk ? kd : vd;
        qd += ostep, kd += kcstep, vd += vcstep;
        if (row0 >= step || r >= rows || (r >= nq && !at.used)) continue;
        float x[8], y[8];
        widen8<DT>(raw[k], x);
        widen8<DT>(raw[k] + (DT == NS_F32 ? 2 : 1), y);
        if (rotates && r < nq + nk) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            // pair j: its members are x[j], y[j], or neighbours 2j, 2j + 1 of the sixteen
            float& a = INTER ? (j < 4 ? x[2 * (j & 3)] : y[2 * (j & 3)]) : x[j];
            float& d = INTER ? (j < 4 ? x[2 * (j & 3) + 1] : y[2 * (j & 3) + 1]) : y[j];
            const float a0 = a, e0 = d;
            a = a0 * c[j] - e0 * s[j];
            d = e0 * c[j] + a0 * s[j];
          }
        }
        if (r < nq) {
          if (!at.used)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.f;
          store8(dst, DT, 0, x);
          store8(dst, DT, d1 - d0, y);
        } else {
          store8(dst, CT, 0, x);
          store8(dst, CT, d1 - d0, y);
        }
      }
      if (gridDim.x > 1) qd += (jump / step - NU) * ostep, kd += (jump / step - NU) * kcstep, vd += (jump / step - NU) * vcstep;
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(kRopeThreads) rope_pairs_kernel(const __grid_constant__ ns_rope_append_t p) {
  griddep_wait();
  griddep_launch_dependents();
  // units of one head: its pairs, then the elements passed through
  const int half = p.rotary_dim / 2, n_rot = half;
  const int n_head_units = n_rot + (p.head_dim - p.rotary_dim), n_val_units = p.head_dim;
  const int nq = p.q ? p.n_head * n_head_units : 0, nk = p.k ? p.n_head_kv * n_head_units : 0;
  const int nv = p.v ? p.n_head_kv * n_val_units : 0;

  for (int64_t tok = blockIdx.y; tok < (int64_t)p.B * p.T; tok += gridDim.y) {
    const int b = (int)(tok / p.T), t = (int)(tok % p.T);
    const RopeAt at = rope_at_token(p, tok, b, t);
    const bool used = at.used;
    const int64_t slot = at.slot, pos = at.pos;
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
        so = b * p.v_stride[0] + t * p.v_stride[1] + h * p.v_stride[2] + u;
        dofs = b * p.vc_stride[0] + h * p.vc_stride[1] + slot * p.vc_stride[2] + u;
        store_float(p.v_cache, p.cache_dtype, dofs, load_float(p.v, DT, so));
        continue;
      }
      if (u >= n_rot) {  // passed through
        const int d = p.rotary_dim + (u - n_rot);
        store_float(dst, dt, dofs + d, used ? load_float(src, DT, so + d) : 0.f);
        continue;
      }
      const int d0 = p.interleaved ? 2 * u : u, d1 = p.interleaved ? 2 * u + 1 : half + u;
      const float x = load_float(src, DT, so + d0), y = load_float(src, DT, so + d1), c = cs[u], s = sn[u];
      store_float(dst, dt, dofs + d0, used ? x * c - y * s : 0.f);
      store_float(dst, dt, dofs + d1, used ? y * c + x * s : 0.f);
    }
  }
}

template <int DT>
static cudaError_t rope_launch(const ns_rope_append_t& p, bool vec, ns_stream_t stream) {
  const int64_t tokens = (int64_t)p.B * p.T;
  const unsigned gy = (unsigned)std::min<int64_t>(tokens, 65535);
  const int rows = (p.q ? p.n_head : 0) + (p.k ? p.n_head_kv : 0) + (p.v ? p.n_head_kv : 0);
  if (!vec) {
    const int64_t units = (int64_t)((p.q ? p.n_head : 0) + (p.k ? p.n_head_kv : 0)) * (p.head_dim - p.rotary_dim / 2) +
                          (int64_t)(p.v ? p.n_head_kv : 0) * p.head_dim;
    return launch_pdl(rope_pairs_kernel<DT>, dim3((unsigned)((units + kRopeThreads - 1) / kRopeThreads), gy), kRopeThreads, 0,
                      stream, 1, p);
  }
  const int step = kRopeRowThreads / (p.head_dim / 16), parts = (rows + step - 1) / step;
  // Few tokens: a block for every part of a token's heads; more: a block a token, four heads in flight a
  // thread.  Measured for 80 heads of 128 in 16 bits (us, parts / whole): 32 tokens 2.5 / 3.2, 128 tokens
  // 4.4 / 3.2, 528 tokens 10.9 / 6.3.
  const bool split = tokens * parts <= 148;
  const dim3 grid(split ? (unsigned)parts : 1u, gy);
  auto run = [&](auto ct, auto inter) {
    constexpr int CT = decltype(ct)::value, NU = DT == NS_F32 ? 2 : 4;
    constexpr bool INTER = decltype(inter)::value;
    return split ? launch_pdl(rope_rows_kernel<DT, CT, INTER, 1>, grid, kRopeRowThreads, 0, stream, 1, p)
                 : launch_pdl(rope_rows_kernel<DT, CT, INTER, NU>, grid, kRopeRowThreads, 0, stream, 1, p);
  };
  auto by_layout = [&](auto ct) { return p.interleaved ? run(ct, std::true_type{}) : run(ct, std::false_type{}); };
  switch (p.cache_dtype) {
    case NS_F32: return by_layout(std::integral_constant<int, NS_F32>{});
    case NS_F16: return by_layout(std::integral_constant<int, NS_F16>{});
    default: return by_layout(std::integral_constant<int, NS_BF16>{});
  }
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
  // (a node whose position is no row of the tables reads row 0 and drops it)
  if (p->n_pos == 0) return fail(NS_ERR_INVALID, "ns_rope_append: tables without rows");
  if ((p->q && !p->q_out) || (p->k && !p->k_cache) || (p->v && !p->v_cache))
    return fail(NS_ERR_INVALID, "ns_rope_append: an input without its output");
  if ((int64_t)(p->n_head + 2 * (int64_t)p->n_head_kv) * p->head_dim > (1 << 28))
    return fail(NS_ERR_UNSUPPORTED, "ns_rope_append: %d + 2 x %d heads of %d", p->n_head, p->n_head_kv, p->head_dim);
  if ((!p->q || !p->n_head) && ((!p->k && !p->v) || !p->n_head_kv)) return NS_OK;
  // octets where every row starts on 16 bytes and the row and its rotation are whole units
  const int64_t m = p->dtype == NS_F32 ? 4 : 8, mc = p->cache_dtype == NS_F32 ? 4 : 8;
  bool vec = p->head_dim % 16 == 0 && p->head_dim <= 16 * kRopeRowThreads && p->rotary_dim % 16 == 0 && p->table_stride % 4 == 0 &&
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
