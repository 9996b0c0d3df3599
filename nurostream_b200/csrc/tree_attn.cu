// ns_tree_attn: attention of every node of a drafted tree over its sequence's cache.
//
// Generalises the core of neurostream/model/gpt_oss.py:73-114 (sink_attention over a KV cache, with the
// sliding window) from one token to B sequences of T nodes:
//   out[t] = sum_j p_j v_j / (sum_j p_j + e^(sink - m)),  p_j = e^(s_j - m),  s_j = scale q_t . k_j
// over the keys j that node t sees: the context below lens[b] (within the window) and its ancestors.
//
// The rep query heads of a kv head and the T nodes are the rows of one matrix (rows = T * rep), so the
// keys and values of a kv head are read once for all of them.  An item is (sequence, kv head, tile of
// rows); its keys are walked in blocks with a running maximum and sum.  Contexts differ, are known on
// the device alone and are long, so the blocks of all items are one list, cut into equal runs, one per
// CTA: every SM gets the same work whatever the lengths are.  A run that covers an item writes the
// result; an item cut between CTAs leaves partial (maximum, sum, output) rows in the workspace, and a
// second kernel joins them in order of the keys (results do not depend on timing).
//
// Within a CTA eight warps are WM groups of 16 rows by WK = 8 / WM groups of keys, so that a single
// row's 16-row tile still keeps eight warps on the stream; the key groups join through shared memory.
// Blocks arrive by cp.async in a ring of three stages.  16-bit products are mma.m16n8k16; fp32
// products split each operand into two tf32 parts and add three mma.m16n8k8 (the product of the two
// low parts, 2^-22 of the whole, is dropped), and the sum over a block joins the running output in
// plain fp32 additions.  What the parts cannot hold (infinities, values that round to one) comes out as
// NaN: such a score is computed again in plain fp32, and such a row of the output by the second kernel.
//
// Measured (device time of a call in a captured graph, 64 query and 8 kv heads of 64, fp32, 2048 keys,
// sinks): one token 13.4 us, of which the blocks themselves take 7 and the join 4.5; a tree of 16 nodes
// (128 rows) 31.5 us.  The bytes would take 1.3 us: one token is bound by the chain of dependent steps
// (length, run, block, partial rows, join), the tree by issue and the latency of its products (tensor pipe
// 30 % busy, 1.7 instructions a cycle: three products each, and the parts are split anew by every warp).
// Looking through every block's values for them at once took 3 to 15 % more for few rows (4 sequences of 8192
// keys, heads of 128: one token 98 us against 85); cvt to tf32 in place of the integer split 30 %.
#include <type_traits>

#include "tree.cuh"

namespace ns {

constexpr int kTaWarps = 8;
constexpr int kTaThreads = kTaWarps * 32;
constexpr int kTaStages = 3;

template <int DT, int HD>
struct TaCfg {
  static constexpr int kEl = DT == NS_F32 ? 4 : 2;       // bytes per element
  static constexpr int kBlock = DT == NS_F32 ? 64 : 128;  // keys per block
  static constexpr int kRowBytes = HD * kEl;
  static constexpr int kTile = kBlock * kRowBytes;        // bytes of a key (or value) block
  static constexpr int kSmem = kTaStages * 2 * kTile;
  static constexpr int kCtas = 2 * (kSmem + 4096) <= 227 * 1024 ? 2 : 1;  // of one SM
};

struct TaArgs {
  ns_tree_attn_t p;
  int rep;         // query heads per kv head
  int tile_rows;   // rows of a tile
  int row_tiles;   // tiles of rows of one (sequence, kv head)
  int block;       // keys of a block
  int vec;         // bit 0, 1: rows of q, out start on 16 bytes (tensor-core kernel)
  int grid;        // runs, at most: none is empty (ta_runs)
  float* part_o;   // [2 * grid][rows per tile][HD]
  float* part_ml;  // [2 * grid][rows per tile][2]
};

struct TaShared {
  uint64_t anc[kTreeMax];   // of the sequence at hand
  int depth[kTreeMax], par[kTreeMax];
  int max_depth;
  uint32_t bad_keys[2][4];  // keys of the block whose values the products cannot take; of every other block
  float wm[kTaWarps][16], wl[kTaWarps][16];
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Probabilities are relative to the running maximum and are divided by their sum last, so a running output is up to
// as many times a value as there are keys: the largest values would overflow where the result does not.  In the
// types that have fp32's range all of them are 2^-kTaShift of that, which is exact (2^24 keys, each up to 2^8:
// the tensor-core kernel's maximum may lag), and a sink's share is scaled alike.  At the other end the last
// bits of sums below 2^-94 (5e-29) are lost.  fp16's values get to neither.
template <int DT>
constexpr float kTaShift = DT == NS_F16 ? 0.f : 32.f;
static_assert(kTaShift<NS_F32> == 32.f, "0x1p-32f in tree_attn_kernel");

// The factor of a row: one over its sum l relative to maximum m, with the head's sink (in units of log2) in it.
template <int DT>
__device__ __forceinline__ float ta_row_scale(float m, float l, const float* sinks, int h) {
  if (!sinks) return 1.f / l;
  const float sk = sinks[h] * 1.4426950408889634f, mm = fmaxf(m, sk);
  return ex2(m - mm) / fmaf(l, ex2(m - mm), ex2(sk - mm - kTaShift<DT>));
}

// The maximum that a part of a row is stored with: -inf marks an unused node, whose row is zero.  A used one's is
// finite or above even where the part has none (no key of it is seen, or every score is NaN or -inf; the
// part's sum, zero or NaN, tells the rest).
__device__ __forceinline__ float ta_part_max(bool used, float m) {
  return used ? fmaxf(m, -3.402823466e38f) : -INFINITY;
}

// Keys [lo, hi) of sequence b that any node may see, and how many blocks they are.
struct TaSpan {
  int lo, hi, len;
};
__device__ __forceinline__ TaSpan ta_span(const ns_tree_attn_t& p, int b) {
  const int n = tree_len(p.lens, b, p.max_ctx);
  if (n < 0) return TaSpan{0, 0, 0};
  const int lo = p.window > 0 ? max(0, n - p.window + 1) : 0;
  return TaSpan{lo, min(n + p.T, p.max_ctx), n};
}

// Position in the list of all blocks: sequences in order, then kv heads, row tiles, blocks of keys.
struct TaPos {
  int b, h, rt, blk, nblk;
};

// Runs of a list of `total` blocks, and the first block of run i.
__device__ __forceinline__ int ta_runs(const TaArgs& a, int64_t total) { return (int)(total < a.grid ? total : a.grid); }
__device__ __forceinline__ int64_t ta_first_unit(int64_t total, int runs, int i) { return total * i / runs; }

// The sequence and offset of unit u, by a walk over the sequences (all threads alike).
__device__ __forceinline__ int64_t ta_total(const TaArgs& a, int BN) {
  int64_t n = 0;
  for (int b = 0; b < a.p.B; ++b) {
    const TaSpan s = ta_span(a.p, b);
    n += (int64_t)((s.hi - s.lo + BN - 1) / BN);
  }
  return n * a.p.n_head_kv * a.row_tiles;
}

// The same by a warp, a sequence per lane.
__device__ __forceinline__ int64_t ta_total_warp(const TaArgs& a, int BN, int lane) {
  int64_t n = 0;
  for (int b = lane; b < a.p.B; b += 32) {
    const TaSpan s = ta_span(a.p, b);
    n += (int64_t)((s.hi - s.lo + BN - 1) / BN);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * a.p.n_head_kv * a.row_tiles;
}

__device__ __forceinline__ TaPos ta_locate(const TaArgs& a, int BN, int64_t u) {
  const int per = a.p.n_head_kv * a.row_tiles;
  for (int b = 0; b < a.p.B; ++b) {
    const TaSpan s = ta_span(a.p, b);
    const int nblk = (s.hi - s.lo + BN - 1) / BN;
    const int64_t here = (int64_t)nblk * per;
    if (u < here) {
      const int item = (int)(u / nblk);
      return TaPos{b, item / a.row_tiles, item % a.row_tiles, (int)(u % nblk), nblk};
    }
    u -= here;
  }
  return TaPos{a.p.B, 0, 0, 0, 1};
}

__device__ __forceinline__ void ta_next(const TaArgs& a, int BN, TaPos& x) {
  if (++x.blk < x.nblk) return;
  x.blk = 0;
  if (++x.rt < a.row_tiles) return;
  x.rt = 0;
  if (++x.h < a.p.n_head_kv) return;
  x.h = 0;
  do {
    if (++x.b >= a.p.B) return;
    const TaSpan s = ta_span(a.p, x.b);
    x.nblk = (s.hi - s.lo + BN - 1) / BN;
  } while (x.nblk == 0);
}

// ---- tensor-core products

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int DT>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == NS_F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo: hi is x rounded to the 11 significant bits of tf32, lo what is left of it, of which the tensor core
// drops the bits below its own 11 (at most the last bit of x, 2^-23 of it, which rounding would be off by too).
// NaN stays NaN in one part or both.  Infinities and values that round to one (kTf32Top and above) come out
// as parts whose products add to NaN: what is NaN is done again in plain fp32.
__device__ __forceinline__ void tf32_split(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = (x + 0x1000u) & 0xFFFFE000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
constexpr uint32_t kTf32Top = 0x7F7FF000u;
template <int DT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (DT == NS_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Whether 16 bytes of shared memory hold a value that the products cannot take: one that is not finite (in 16 bits:
// an exponent of ones, to which adding one carries into the sign's place, that the mask has cleared), in fp32
// also one that tf32_split makes infinite (kTf32Top carries there with what is added).
template <int DT>
__device__ __forceinline__ uint32_t not_finite(uint32_t saddr) {
  uint32_t w[4];
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(saddr) : "memory");
  constexpr uint32_t m = DT == NS_F32 ? 0x7FFFFFFFu : DT == NS_F16 ? 0x7C007C00u : 0x7F807F80u;
  constexpr uint32_t one = DT == NS_F32 ? 0x80000000u - kTf32Top : DT == NS_F16 ? 0x04000400u : 0x00800080u;
  constexpr uint32_t top = DT == NS_F32 ? 0x80000000u : 0x80008000u;
  return (((w[0] & m) + one) | ((w[1] & m) + one) | ((w[2] & m) + one) | ((w[3] & m) + one)) & top;
}

// 16-byte copy into shared memory, zeros when `ok` is false (nothing is read then).
__device__ __forceinline__ void cp_async16_z(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

template <int DT, int HD, int WM>
__global__ void __launch_bounds__(kTaThreads, (TaCfg<DT, HD>::kCtas)) tree_attn_kernel(const __grid_constant__ TaArgs a) {
  using Cfg = TaCfg<DT, HD>;
  constexpr int BN = Cfg::kBlock, EL = Cfg::kEl, RB = Cfg::kRowBytes;
  constexpr int WK = kTaWarps / WM, MR = 16 * WM, KW = BN / WK, SB = DT == NS_F32 ? (KW < 16 ? KW : 16) : (KW < 32 ? KW : 32);
  constexpr int CH = RB / 16;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t ta_smem[];
  __shared__ TaShared S;
  const ns_tree_attn_t& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp % WM, wk = warp / WM;
  const int g = lane >> 2, tq = lane & 3;
  const uint32_t sbase = smem_addr(ta_smem);

  griddep_wait();
  griddep_launch_dependents();
  const int64_t total = ta_total(a, BN);
  const int runs = ta_runs(a, total);
  if ((int)blockIdx.x >= runs) return;
  const int64_t u0 = ta_first_unit(total, runs, blockIdx.x), u1 = ta_first_unit(total, runs, blockIdx.x + 1);

  TaPos ld = ta_locate(a, BN, u0), at = ld;
  const int row_chunks = p.head_dim * EL / 16;
  auto load_block = [&](int stage) {  // the block at `ld` into a stage; rows past the end and dims past head_dim are zeros
    const TaSpan s = ta_span(p, ld.b);
    const int k0 = s.lo + ld.blk * BN;
    const char* kb = static_cast<const char*>(p.k_cache) + (ld.b * p.kc_stride[0] + ld.h * p.kc_stride[1]) * EL;
    const char* vb = static_cast<const char*>(p.v_cache) + (ld.b * p.vc_stride[0] + ld.h * p.vc_stride[1]) * EL;
    const uint32_t dk = sbase + stage * 2 * Cfg::kTile, dv = dk + Cfg::kTile;
#pragma unroll
    for (int i = 0; i < BN * CH / kTaThreads; ++i) {
      const int c = tid + i * kTaThreads, r = c / CH, ch = c % CH;
      const bool ok = k0 + r < s.hi && ch < row_chunks;
      const int64_t key = ok ? k0 + r : s.lo;
      const int cc = ok ? ch : 0;
      const uint32_t off = r * RB + ((ch ^ (r & 7)) << 4);
      cp_async16_z(dk + off, kb + key * p.kc_stride[2] * EL + cc * 16, ok);
      cp_async16_z(dv + off, vb + key * p.vc_stride[2] * EL + cc * 16, ok);
    }
  };

  if (tid < 8) S.bad_keys[tid >> 2][tid & 3] = 0;
  int scan = 0;  // which of bad_keys the block uses

  int64_t ul = u0;
#pragma unroll
  for (int i = 0; i < kTaStages - 1; ++i) {
    if (ul < u1) {
      load_block(i);
      ta_next(a, BN, ld);
      ++ul;
    }
    cp_async_commit();
  }

  const float sc_hi = p.scale * 1.4426950408889634f;
  const float sc_lo = fmaf(p.scale, 1.4426950408889634f, -sc_hi) + p.scale * 1.925963033500e-8f;

  float o[HD / 8][4];
  float m[2], l[2];
  uint32_t qf[DT == NS_F32 ? HD / 8 : HD / 16][4];  // this warp's queries as A fragments
  uint64_t anc[2] = {0, 0};
  int dep[2] = {0, 0}, cur_b = -1;
  bool fresh = true;
  int first_blk = 0;

  int stage = 0;
  for (int64_t u = u0; u < u1; ++u) {
    const TaSpan sp = ta_span(p, at.b);
    if (fresh) {  // a new item: its tree and this thread's two rows
      first_blk = at.blk;
      if (at.b != cur_b) {
        __syncthreads();
        if (tid == 0) S.max_depth = 0;
        if (tid < p.T) S.par[tid] = p.parents ? p.parents[(int64_t)at.b * p.T + tid] : tid - 1;
        __syncthreads();
        if (tid < p.T) {
          bool bad = false;
          uint64_t mk = p.parents ? tree_mask(tid, [&](int i) { return S.par[i]; }, &bad) : chain_mask(tid);
          if (mk && sp.len + tid >= p.max_ctx) mk = 0, bad = true;
          if (bad) raise_device_error(NS_DEVERR_ROUTE);
          S.anc[tid] = mk;
          S.depth[tid] = __popcll(mk) - 1;
          atomicMax(&S.max_depth, __popcll(mk) - 1);
        }
        __syncthreads();
        cur_b = at.b;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = at.rt * MR + wm * 16 + g + 8 * i, t = r / a.rep;
        anc[i] = t < p.T ? S.anc[t] : 0;
        dep[i] = t < p.T ? S.depth[t] : 0;
        m[i] = -INFINITY, l[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = at.rt * MR + wm * 16 + g + 8 * i, t = r / a.rep, hr = r % a.rep;
        const int64_t qo = at.b * p.q_stride[0] + t * p.q_stride[1] + (at.h * a.rep + hr) * p.q_stride[2];
        if constexpr (DT != NS_F32) {
          const uint16_t* q = static_cast<const uint16_t*>(p.q) + qo;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int hlf = 0; hlf < 2; ++hlf) {
              const int d = kk * 16 + hlf * 8 + 2 * tq;
              uint32_t w = 0;
              if (t < p.T && d < p.head_dim) w = (uint32_t)q[d] | ((uint32_t)q[d + 1] << 16);
              qf[kk][hlf * 2 + i] = w;
            }
        } else {
          const float* q = static_cast<const float*>(p.q) + qo;
#pragma unroll
          for (int kk = 0; kk < HD / 8; ++kk)
#pragma unroll
            for (int hlf = 0; hlf < 2; ++hlf) {
              const int d = kk * 8 + hlf * 4 + tq;
              qf[kk][hlf * 2 + i] = t < p.T && d < p.head_dim ? __float_as_uint(q[d]) : 0u;
            }
        }
      }
      fresh = false;
    }

    cp_async_wait<kTaStages - 2>();
    __syncthreads();
    // the next block goes into the stage that was used last, unless an item's end still needs it
    const bool last_of_item = at.blk + 1 == at.nblk || u + 1 == u1;
    const int free_stage = (stage + kTaStages - 1) % kTaStages;
    if (ul < u1) {
      load_block(free_stage);
      ta_next(a, BN, ld);
      ++ul;
    }
    cp_async_commit();

    const uint32_t ks = sbase + stage * 2 * Cfg::kTile, vs = ks + Cfg::kTile;
    const int k0 = sp.lo + at.blk * BN;
    // a block needs no mask when every row sees all of it
    const bool masked = k0 + BN > sp.len || (p.window > 0 && sp.len + S.max_depth - k0 >= p.window);
    auto sees = [&](int i, int key) {  // whether this thread's row i sees a key of the item
      if (key < sp.len) return anc[i] != 0 && (p.window == 0 || sp.len + dep[i] - key < p.window);
      const int nd = key - sp.len;
      return nd < p.T && nd < kTreeMax && (anc[i] >> nd & 1) && (p.window == 0 || dep[i] - S.depth[nd] < p.window);
    };
    // Values that not every row sees may hold anything: rows of the block that hold what the products cannot take
    // are set to zero here and added, for the rows that see them, from the cache below.
    if (masked) {
      scan ^= 1;
      if (tid < 4) S.bad_keys[scan ^ 1][tid] = 0;  // for the next block that looks; its last readers are past the barrier
#pragma unroll 4
      for (int i = 0; i < BN * CH / kTaThreads; ++i) {
        const int c = tid + i * kTaThreads;
        if (not_finite<DT>(vs + c * 16)) atomicOr(&S.bad_keys[scan][c / CH >> 5], 1u << (c / CH & 31));
      }
      __syncthreads();
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < BN / 32; ++i) any |= S.bad_keys[scan][i];
      if (any) {
        for (int c = tid; c < BN * CH; c += kTaThreads)
          if (S.bad_keys[scan][c / CH >> 5] >> (c / CH & 31) & 1) sts128(vs + c * 16, 0, 0, 0, 0);
        __syncthreads();
      }
    }

#pragma unroll 1
    for (int sb = 0; sb < KW / SB; ++sb) {
      const int kr = wk * KW + sb * SB;  // first key row of the sub-block within the block
      float s[SB / 8][4];
#pragma unroll
      for (int i = 0; i < SB / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
      if constexpr (DT != NS_F32) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
          for (int n = 0; n < SB / 16; ++n) {  // 16 keys x 16 dims: two n-tiles of B fragments
            uint32_t kf[4];
            const int r = kr + n * 16 + (lane & 7) + ((lane >> 4) << 3), ch = kk * 2 + ((lane >> 3) & 1);
            ldsm4(kf, ks + r * RB + ((ch ^ (r & 7)) << 4));
            mma16<DT>(s[2 * n], qf[kk], kf[0], kf[1]);
            mma16<DT>(s[2 * n + 1], qf[kk], kf[2], kf[3]);
          }
      } else {
#pragma unroll
        for (int kk = 0; kk < HD / 8; ++kk) {
          uint32_t ah[4], al[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) tf32_split(qf[kk][j], ah[j], al[j]);
#pragma unroll
          for (int n = 0; n < SB / 8; ++n) {
            const int r = kr + n * 8 + g;
            uint32_t bh0, bl0, bh1, bl1;
            tf32_split(lds32(ks + r * RB + (((2 * kk) ^ (r & 7)) << 4) + 4 * tq), bh0, bl0);
            tf32_split(lds32(ks + r * RB + (((2 * kk + 1) ^ (r & 7)) << 4) + 4 * tq), bh1, bl1);
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            mma8(c, al, bh0, bh1);
            mma8(c, ah, bl0, bl1);
            mma8(c, ah, bh0, bh1);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] += c[j];
          }
        }
      }
      // scores in units of log2, masked; running maximum
      float mx[2] = {m[0], m[1]};
      if (masked) {
#pragma unroll
        for (int n = 0; n < SB / 8; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!sees(j >> 1, k0 + kr + n * 8 + 2 * tq + (j & 1))) s[n][j] = -INFINITY;
          }
      }
      if constexpr (DT == NS_F32) {  // scores that came out as NaN: the products may not have taken q or k
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < SB / 8; ++n) sum[0] += s[n][0] + s[n][1], sum[1] += s[n][2] + s[n][3];
        if (__any_sync(0xffffffffu, (anc[0] && sum[0] != sum[0]) || (anc[1] && sum[1] != sum[1]))) {
#pragma unroll 1
          for (int e = 0; e < SB / 2; ++e) {
            const int n = e >> 2, j = e & 3, r = at.rt * MR + wm * 16 + g + 8 * (j >> 1);
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < SB / 2; ++i) x = i == e ? s[i >> 2][i & 3] : x;
            if (x != x && (j >> 1 ? anc[1] : anc[0])) {
              const float* q = static_cast<const float*>(p.q) + at.b * p.q_stride[0] + r / a.rep * p.q_stride[1] +
                               (at.h * a.rep + r % a.rep) * p.q_stride[2];
              const float* k = static_cast<const float*>(p.k_cache) + at.b * p.kc_stride[0] + at.h * p.kc_stride[1] +
                               (int64_t)(k0 + kr + n * 8 + 2 * tq + (j & 1)) * p.kc_stride[2];
              x = 0.f;
#pragma unroll 8
              for (int d = 0; d < p.head_dim; ++d) x = fmaf(q[d], k[d], x);
            }
#pragma unroll
            for (int i = 0; i < SB / 2; ++i)
              if (i == e) s[i >> 2][i & 3] = x;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < SB / 8; ++n) {
        mx[0] = fmaxf(mx[0], fmaxf(s[n][0], s[n][1]) * sc_hi);
        mx[1] = fmaxf(mx[1], fmaxf(s[n][2], s[n][3]) * sc_hi);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      }
      float corr[2], ref[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ref[i] = mx[i] == -INFINITY ? 0.f : mx[i];
        corr[i] = ex2(m[i] - ref[i]);
        m[i] = mx[i];
        l[i] *= corr[i];
      }
#pragma unroll
      for (int n = 0; n < SB / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = s[n][j];
          // (kTaShift in fp32 as a factor: added to the exponent it would cost that its last bits)
          const float e = DT != NS_F32      ? fmaf(x, sc_hi, -kTaShift<DT> - ref[j >> 1])
                          : x != -INFINITY ? fmaf(x, sc_lo, fmaf(x, sc_hi, -ref[j >> 1]))
                                           : -INFINITY;
          s[n][j] = DT == NS_F32 ? ex2(e) * 0x1p-32f : ex2(e);
          l[j >> 1] += s[n][j];
        }
      if constexpr (DT != NS_F32) {
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          o[i][0] *= corr[0], o[i][1] *= corr[0];
          o[i][2] *= corr[1], o[i][3] *= corr[1];
        }
#pragma unroll
        for (int kk = 0; kk < SB / 16; ++kk) {
          // probabilities rounded to 16 bits: half an ulp each, as large as the output's own rounding
          const uint32_t pf[4] = {pack16<DT>(s[2 * kk][0], s[2 * kk][1]), pack16<DT>(s[2 * kk][2], s[2 * kk][3]),
                                  pack16<DT>(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                                  pack16<DT>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            uint32_t vf[4];
            const int r = kr + kk * 16 + (lane & 15), ch = n * 2 + (lane >> 4);
            ldsm4_t(vf, vs + r * RB + ((ch ^ (r & 7)) << 4));
            mma16<DT>(o[2 * n], pf, vf[0], vf[1]);
            mma16<DT>(o[2 * n + 1], pf, vf[2], vf[3]);
          }
        }
      } else {
        // keys 2t and 2t+1 of an octet stand at k = t and t + 4, where the score fragments have them
        uint32_t ph[SB / 8][4], pl[SB / 8][4];
#pragma unroll
        for (int kk = 0; kk < SB / 8; ++kk) {
          tf32_split(__float_as_uint(s[kk][0]), ph[kk][0], pl[kk][0]);
          tf32_split(__float_as_uint(s[kk][2]), ph[kk][1], pl[kk][1]);
          tf32_split(__float_as_uint(s[kk][1]), ph[kk][2], pl[kk][2]);
          tf32_split(__float_as_uint(s[kk][3]), ph[kk][3], pl[kk][3]);
        }
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
#pragma unroll
          for (int kk = 0; kk < SB / 8; ++kk) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            const int r = kr + kk * 8 + 2 * tq, ch = n * 2 + (g >> 2);
            uint32_t bh0, bl0, bh1, bl1;
            tf32_split(lds32(vs + r * RB + ((ch ^ (r & 7)) << 4) + 4 * (g & 3)), bh0, bl0);
            tf32_split(lds32(vs + (r + 1) * RB + ((ch ^ ((r + 1) & 7)) << 4) + 4 * (g & 3)), bh1, bl1);
            mma8(c, pl[kk], bh0, bh1);
            mma8(c, ph[kk], bl0, bl1);
            mma8(c, ph[kk], bh0, bh1);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][j] = kk == 0 ? fmaf(o[n][j], corr[j >> 1], c[j]) : o[n][j] + c[j];
          }
        }
      }
      if (masked) {  // the values left out, for the rows that see them
        uint32_t bad = S.bad_keys[scan][kr >> 5] >> (kr & 31);
        if constexpr (SB < 32) bad &= (1u << SB) - 1;
        while (bad) {
          const int kk = __ffs(bad) - 1;
          bad &= bad - 1;
          float pv[2] = {0.f, 0.f};
#pragma unroll
          for (int n = 0; n < SB / 8; ++n)
            if (n == kk >> 3) pv[0] = kk & 1 ? s[n][1] : s[n][0], pv[1] = kk & 1 ? s[n][3] : s[n][2];
          const int from = (lane & ~3) | ((kk & 7) >> 1);
          pv[0] = __shfl_sync(0xffffffffu, pv[0], from);
          pv[1] = __shfl_sync(0xffffffffu, pv[1], from);
          // (by the mask: a probability may be too small for its type and the value still count)
          const bool see[2] = {sees(0, k0 + kr + kk), sees(1, k0 + kr + kk)};
          const int64_t vrow = at.b * p.vc_stride[0] + at.h * p.vc_stride[1] + (int64_t)(k0 + kr + kk) * p.vc_stride[2];
#pragma unroll
          for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int d = n * 8 + 2 * tq + j;
              if (d >= p.head_dim) continue;
              const float v = load_float(p.v_cache, DT, vrow + d);
              if (see[0]) o[n][j] = fmaf(pv[0], v, o[n][j]);
              if (see[1]) o[n][2 + j] = fmaf(pv[1], v, o[n][2 + j]);
            }
          __syncwarp();  // the products of the next keys are .aligned
        }
      }
    }

    if (last_of_item) {
      // the row sums of the quad; then the key groups join in order through the stage just consumed
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      }
      const bool whole = first_blk == 0 && at.blk + 1 == at.nblk;
      if constexpr (WK > 1) {
        static_assert(kTaWarps * 16 * HD * 4 <= 2 * Cfg::kTile, "the join fits the stage");
        __syncthreads();  // every warp is done with the stage
        float* jo = reinterpret_cast<float*>(ta_smem + stage * 2 * Cfg::kTile);
        if (tq == 0) {
          S.wm[warp][g] = m[0], S.wm[warp][g + 8] = m[1];
          S.wl[warp][g] = l[0], S.wl[warp][g + 8] = l[1];
        }
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            jo[(warp * 16 + g + 8 * (j >> 1)) * HD + n * 8 + 2 * tq + (j & 1)] = o[n][j];
        __syncthreads();
      }
      // rows leave as whole rows: a warp takes row after row
      const int n_rows = min(MR, p.T * a.rep - at.rt * MR);
      const int slot = 2 * blockIdx.x + (u - at.blk <= u0 ? 0 : 1);
      if constexpr (WK > 1) {
        const float* jo = reinterpret_cast<const float*>(ta_smem + stage * 2 * Cfg::kTile);
        for (int r = warp; r < n_rows; r += kTaWarps) {
          const int grp = r / 16, ri = r % 16;
          float mt = -INFINITY, lt = 0.f, acc[HD / 32];
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) acc[i] = 0.f;
#pragma unroll
          for (int w = 0; w < WK; ++w) mt = fmaxf(mt, S.wm[w * WM + grp][ri]);
          const float ref = mt == -INFINITY ? 0.f : mt;
#pragma unroll
          for (int w = 0; w < WK; ++w) {
            const float f = ex2(S.wm[w * WM + grp][ri] - ref);
            lt = fmaf(S.wl[w * WM + grp][ri], f, lt);
#pragma unroll
            for (int i = 0; i < HD / 32; ++i)
              acc[i] = fmaf(jo[((w * WM + grp) * 16 + ri) * HD + lane + 32 * i], f, acc[i]);
          }
          const int row = at.rt * MR + r, t = row / a.rep, h = at.h * a.rep + row % a.rep;
          if (whole) {
            const bool live = S.anc[t] != 0;  // a used node sees itself at least
            const float scale = live ? ta_row_scale<DT>(mt, lt, p.sinks, h) : 0.f;
            const int64_t oo = at.b * p.o_stride[0] + t * p.o_stride[1] + h * p.o_stride[2];
#pragma unroll
            for (int i = 0; i < HD / 32; ++i)
              if (lane + 32 * i < p.head_dim) store_float(p.out, DT, oo + lane + 32 * i, live ? acc[i] * scale : 0.f);
          } else {
            float* po = a.part_o + ((int64_t)slot * MR + r) * HD;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) po[lane + 32 * i] = acc[i];
            if (lane == 0) {
              a.part_ml[((int64_t)slot * MR + r) * 2] = ta_part_max(S.anc[t] != 0, mt);
              a.part_ml[((int64_t)slot * MR + r) * 2 + 1] = lt;
            }
          }
        }
        __syncthreads();  // the stage may be filled again
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = wm * 16 + g + 8 * i;
          if (r >= n_rows) continue;
          const int row = at.rt * MR + r, t = row / a.rep, h = at.h * a.rep + row % a.rep;
          if (whole) {
            const bool live = anc[i] != 0;
            const float scale = live ? ta_row_scale<DT>(m[i], l[i], p.sinks, h) : 0.f;
            const int64_t oo = at.b * p.o_stride[0] + t * p.o_stride[1] + h * p.o_stride[2];
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int d = n * 8 + 2 * tq + j;
                if (d < p.head_dim) store_float(p.out, DT, oo + d, live ? o[n][2 * i + j] * scale : 0.f);
              }
          } else {
            float* po = a.part_o + ((int64_t)slot * MR + r) * HD;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
              *reinterpret_cast<float2*>(po + n * 8 + 2 * tq) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            if (tq == 0) {
              a.part_ml[((int64_t)slot * MR + r) * 2] = ta_part_max(anc[i] != 0, m[i]);
              a.part_ml[((int64_t)slot * MR + r) * 2 + 1] = l[i];
            }
          }
        }
      }
      fresh = true;
    }
    ta_next(a, BN, at);
    stage = (stage + 1) % kTaStages;
  }
}

// One fp32 row of the output over all of its keys in plain fp32, by a warp.  For rows that the tensor cores left with NaN in
// them although their sum is none: infinities, and values that round to one, in blocks without a mask.  A lane
// takes a key's score, then the warp the dims key after key.  Rare, and slow (2,048 rows of 8,192 keys 24 ms);
// kept to few registers, since they count for the kernels that call it.  A score of NaN ends it: the row is NaN as it stands.
template <int HD>
__device__ __noinline__ void ta_plain_row(const TaArgs& a, int b, int hk, int row) {
  constexpr int V = HD / 32;
  const ns_tree_attn_t& p = a.p;
  const int lane = threadIdx.x & 31, t = row / a.rep, h = hk * a.rep + row % a.rep;
  const TaSpan sp = ta_span(p, b);
  bool bad = false;
  const int32_t* par = p.parents + (int64_t)b * p.T;
  const uint64_t anc = p.parents ? tree_mask(t, [&](int i) { return par[i]; }, &bad) : chain_mask(t);
  const int dep = __popcll(anc) - 1;
  const float* q = static_cast<const float*>(p.q) + b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2];
  const float* kc = static_cast<const float*>(p.k_cache) + b * p.kc_stride[0] + hk * p.kc_stride[1];
  const float* vc = static_cast<const float*>(p.v_cache) + b * p.vc_stride[0] + hk * p.vc_stride[1] + lane * V;
  float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = 0.f;
  for (int c = sp.lo; c < sp.hi; c += 32) {
    const int key = c + lane, nd = key - sp.len;
    bool see = key < sp.hi;
    if (see && nd < 0) see = p.window == 0 || sp.len + dep - key < p.window;
    else if (see)  // (an ancestor's depth: the ancestors before it)
      see = nd < kTreeMax && (anc >> nd & 1) && (p.window == 0 || dep - __popcll(anc & ((1ull << nd) - 1)) < p.window);
    float x = 0.f;
    if (see) {
      const float4* k = reinterpret_cast<const float4*>(kc + (int64_t)key * p.kc_stride[2]);
#pragma unroll 2
      for (int d = 0; d < p.head_dim / 4; ++d) {
        const float4 y = k[d];
        x = fmaf(q[4 * d], y.x, x), x = fmaf(q[4 * d + 1], y.y, x), x = fmaf(q[4 * d + 2], y.z, x), x = fmaf(q[4 * d + 3], y.w, x);
      }
    }
    x = see ? x * p.scale * 1.4426950408889634f : -INFINITY;
    if (__any_sync(0xffffffffu, x != x)) return;
    float mn = fmaxf(m, x);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, i));
    const float ref = mn == -INFINITY ? 0.f : mn, f = ex2(m - ref), e = ex2(x - ref) * 0x1p-32f;
    m = mn;
    l = l * f + warp_sum(e);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] *= f;
    const uint32_t seen = __ballot_sync(0xffffffffu, see);
#pragma unroll 1
    for (int i = 0; i < 32; i += 4) {
      float v[4][V];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j)
          v[u][j] = (seen >> (i + u) & 1) && lane * V + j < p.head_dim ? vc[(int64_t)(c + i + u) * p.vc_stride[2] + j] : 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = __shfl_sync(0xffffffffu, e, i + u);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = fmaf(w, v[u][j], o[j]);
      }
    }
  }
  const float scale = ta_row_scale<NS_F32>(m, l, p.sinks, h);
  float* out = static_cast<float*>(p.out) + b * p.o_stride[0] + t * p.o_stride[1] + h * p.o_stride[2] + lane * V;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (lane * V + j < p.head_dim) out[j] = o[j] * scale;
}

// Joins the partial rows of items that were cut between runs.  A block takes a few rows of one item; the
// item's place in the list, and so which runs hold its parts, is worked out once.  WPR = 1: a warp
// takes whole rows, two or three parts each.  WPR = 8: few rows and many parts, a row's parts are shared
// among the block's warps.  The order of the sums is fixed: a result does not depend on timing.
// Rows that nothing was computed for (an empty or bad sequence) are zero.
constexpr int kJoinWarps = 8;
constexpr int kJoinRows = 4;  // rows a warp takes with WPR = 1

template <int DT, int HD, int WPR>
__global__ void __launch_bounds__(kJoinWarps * 32) tree_attn_join_kernel(const __grid_constant__ TaArgs a) {
  constexpr int V = HD / 32, RB = WPR == 1 ? kJoinWarps * kJoinRows : 1;
  const int BN = a.block, MR = a.tile_rows;
  __shared__ float so[WPR > 1 ? WPR : 1][HD], sm[WPR], sl[WPR];
  const ns_tree_attn_t& p = a.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int item = blockIdx.x, rt = item % a.row_tiles, hk = item / a.row_tiles % p.n_head_kv;
  const int b = item / a.row_tiles / p.n_head_kv;
  const int n_rows = min(MR, p.T * a.rep - rt * MR);
  const int r0 = blockIdx.y * RB;
  griddep_wait();
  griddep_launch_dependents();
  if (r0 >= n_rows) return;
  // blocks of all sequences, and of those before this one
  int64_t total = 0, before = 0;
  for (int i = lane; i < p.B; i += 32) {
    const TaSpan s = ta_span(p, i);
    const int n = (s.hi - s.lo + BN - 1) / BN;
    total += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  total *= (int64_t)p.n_head_kv * a.row_tiles;
  const int runs = ta_runs(a, total);
  const TaSpan sp = ta_span(p, b);
  const int nblk = (sp.hi - sp.lo + BN - 1) / BN;
  const int64_t s = (before * p.n_head_kv + (int64_t)hk * nblk) * a.row_tiles + (int64_t)rt * nblk, e = s + nblk;
  const int i0 = nblk ? (int)(((s + 1) * runs - 1) / total) : 0, i1 = nblk ? (int)((e * runs - 1) / total) : 0;
  const bool whole = nblk && i0 == i1;  // one run covered it
  // (fp32: a row's open blocks may have left NaN in it, see ta_plain_row)
  if (whole && (DT != NS_F32 || sp.len - sp.lo < BN)) return;
  const int n = whole ? 0 : i1 - i0 + 1;

  auto finish = [&](int r, float mt, float lt, float (&acc)[V]) {  // one row out
    const int row = rt * MR + r, t = row / a.rep, h = hk * a.rep + row % a.rep;
    const bool live = mt != -INFINITY;  // only an unused node's parts all say so (ta_part_max)
    const float scale = live ? ta_row_scale<DT>(mt, lt, p.sinks, h) : 0.f;
    const int64_t oo = b * p.o_stride[0] + t * p.o_stride[1] + h * p.o_stride[2] + lane * V;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = live ? acc[j] * scale : 0.f;
    if constexpr (DT != NS_F32 && V == 4) {
      uint16_t* out = static_cast<uint16_t*>(p.out) + oo;
      if ((reinterpret_cast<uintptr_t>(out) & 7) == 0 && lane * V + V <= p.head_dim) {
        *reinterpret_cast<uint2*>(out) = make_uint2(pack16<DT>(acc[0], acc[1]), pack16<DT>(acc[2], acc[3]));
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (lane * V + j < p.head_dim) store_float(p.out, DT, oo + j, acc[j]);
  };
  auto load_part = [&](int64_t at, float (&v)[V]) {
    const float* src = a.part_o + at * HD + lane * V;
    if constexpr (V == 4) {
      const float4 x = *reinterpret_cast<const float4*>(src);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(src);
      v[0] = x.x, v[1] = x.y;
    }
  };

  if constexpr (DT == NS_F32) {
    if (whole) {  // what the run wrote, the warp's rows side by side
      if (WPR > 1 && warp > 0) return;
      constexpr int R = WPR > 1 ? 1 : kJoinRows;
      bool odd[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int row = rt * MR + min(r0 + k * kJoinWarps + warp, n_rows - 1), t = row / a.rep;
        const float* out = static_cast<const float*>(p.out) + b * p.o_stride[0] + t * p.o_stride[1] +
                           (hk * a.rep + row % a.rep) * p.o_stride[2];
        odd[k] = false;
#pragma unroll
        for (int j = 0; j < V; ++j) odd[k] |= lane + 32 * j < p.head_dim && out[lane + 32 * j] != out[lane + 32 * j];
      }
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (__any_sync(0xffffffffu, odd[k]) && r0 + k * kJoinWarps + warp < n_rows)
          ta_plain_row<HD>(a, b, hk, rt * MR + r0 + k * kJoinWarps + warp);
      return;
    }
  }

  if constexpr (WPR == 1) {
    // the warp's rows side by side: their loads are in flight together
    float mt[kJoinRows], lt[kJoinRows], acc[kJoinRows][V];
#pragma unroll
    for (int k = 0; k < kJoinRows; ++k) {
      mt[k] = -INFINITY, lt[k] = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[k][j] = 0.f;
    }
    for (int i = 0; nblk && i < n; ++i) {
      const int64_t at = (int64_t)(2 * (i0 + i) + (i == 0 && ta_first_unit(total, runs, i0) < s ? 1 : 0)) * MR;
      float2 ml[kJoinRows];
      float v[kJoinRows][V];
#pragma unroll
      for (int k = 0; k < kJoinRows; ++k) {
        const int r = min(r0 + k * kJoinWarps + warp, n_rows - 1);
        ml[k] = *reinterpret_cast<const float2*>(a.part_ml + (at + r) * 2);
        load_part(at + r, v[k]);
      }
#pragma unroll
      for (int k = 0; k < kJoinRows; ++k) {
        const float mn = fmaxf(mt[k], ml[k].x), ref = mn == -INFINITY ? 0.f : mn;
        const float f = ex2(mt[k] - ref), fi = ex2(ml[k].x - ref);
        mt[k] = mn;
        lt[k] = lt[k] * f + ml[k].y * fi;
#pragma unroll
        for (int j = 0; j < V; ++j) acc[k][j] = acc[k][j] * f + v[k][j] * fi;
      }
    }
#pragma unroll
    for (int k = 0; k < kJoinRows; ++k) {
      const int r = r0 + k * kJoinWarps + warp;
      if (r >= n_rows) continue;
      finish(r, mt[k], lt[k], acc[k]);
    }
    if constexpr (DT == NS_F32) {
      bool odd = false;
#pragma unroll
      for (int k = 0; k < kJoinRows; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) odd |= acc[k][j] != acc[k][j];
      if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
        for (int k = 0; k < kJoinRows; ++k) {
          const int r = r0 + k * kJoinWarps + warp;
          bool mine = false;
#pragma unroll
          for (int j = 0; j < V; ++j) mine |= acc[k][j] != acc[k][j];
          if (__any_sync(0xffffffffu, mine) && r < n_rows && mt[k] != -INFINITY && lt[k] == lt[k])
            ta_plain_row<HD>(a, b, hk, rt * MR + r);
        }
      }
    }
  } else {
    float mt = -INFINITY, lt = 0.f, acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    const int from = n * warp / WPR, to = nblk ? n * (warp + 1) / WPR : 0;
    for (int c = from; c < to; c += 32) {
      float mi = -INFINITY, li = 0.f;
      int64_t base = 0;
      if (c + lane < to) {
        const int i = i0 + c + lane;
        base = (int64_t)(2 * i + (i == i0 && ta_first_unit(total, runs, i) < s ? 1 : 0)) * MR + r0;
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + base * 2);
        mi = ml.x, li = ml.y;
      }
      float mn = fmaxf(mt, mi);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float f = ex2(mt - ref), fi = ex2(mi - ref);
      mt = mn;
      lt = lt * f + warp_sum(li * fi);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] *= f;
      const int m = min(32, to - c);
      for (int i = 0; i < m; i += 4) {  // four parts in flight; past the end the last one again, not added
        float v[4][V], w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int src = min(i + k, m - 1);
          w[k] = __shfl_sync(0xffffffffu, fi, src);
          load_part(__shfl_sync(0xffffffffu, base, src), v[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] = i + k < m ? fmaf(v[k][j], w[k], acc[j]) : acc[j];
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) so[warp][lane * V + j] = acc[j];
    if (lane == 0) sm[warp] = mt, sl[warp] = lt;
    __syncthreads();
    if (warp == 0) {
      mt = -INFINITY;
#pragma unroll
      for (int w = 0; w < WPR; ++w) mt = fmaxf(mt, sm[w]);
      const float ref = mt == -INFINITY ? 0.f : mt;
      lt = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        const float f = ex2(sm[w] - ref);
        lt = fmaf(sl[w], f, lt);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = fmaf(so[w][lane * V + j], f, acc[j]);
      }
      finish(r0, mt, lt, acc);
      if constexpr (DT == NS_F32) {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < V; ++j) odd |= acc[j] != acc[j];
        if (__any_sync(0xffffffffu, odd) && mt != -INFINITY && lt == lt) ta_plain_row<HD>(a, b, hk, rt * MR + r0);
      }
    }
  }
  if (lane == 0 && warp == 0 && r0 == 0 && (p.lens[b] < 0 || p.lens[b] > p.max_ctx)) raise_device_error(NS_DEVERR_ROUTE);
}

// ---- host

// Runs of a launch, at most: the workspace is sized for it without asking the device.
constexpr int kTaMaxSms = 160;

static int ta_groups(const ns_tree_attn_t* p) {  // WM: 16-row groups of a tile
  const int rows = p->T * (p->n_head / p->n_head_kv);
  return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8;
}

template <int DT, int HD>
static int ta_join(const TaArgs& a, ns_stream_t stream) {
  const int64_t items = (int64_t)a.p.B * a.p.n_head_kv * a.row_tiles;
  const int rows = std::min(a.tile_rows, a.p.T * a.rep);
  if (items > INT32_MAX) return fail(NS_ERR_UNSUPPORTED, "ns_tree_attn: %lld tiles of rows", (long long)items);
  // Few rows have many parts: they are shared out among the warps.  Whole calls measured (us, shared / a warp
  // a row): 64 rows of 33 parts 13.1 / 28.0, 1024 rows 30.3 / 53.4, 4096 rows 39.9 / 29.5.
  if (items * rows <= 1024)
    NS_CUDA_TRY(launch_pdl(tree_attn_join_kernel<DT, HD, kJoinWarps>, dim3((unsigned)items, rows), kJoinWarps * 32, 0, stream, 1, a));
  else
    NS_CUDA_TRY(launch_pdl(tree_attn_join_kernel<DT, HD, 1>,
                           dim3((unsigned)items, (rows + kJoinWarps * kJoinRows - 1) / (kJoinWarps * kJoinRows)),
                           kJoinWarps * 32, 0, stream, 1, a));
  return NS_OK;
}

template <int DT, int HD, int WM>
static int ta_run(const ns_tree_attn_t* p, void* ws, ns_stream_t stream, size_t* bytes) {
  constexpr int MR = 16 * WM, max_grid = kTaMaxSms * TaCfg<DT, HD>::kCtas;
  const size_t o_bytes = (size_t)2 * max_grid * MR * HD * sizeof(float);
  if (bytes) {
    *bytes = o_bytes + (size_t)2 * max_grid * MR * 2 * sizeof(float);
    return NS_OK;
  }
  TaArgs a = {};
  a.p = *p;
  a.rep = p->n_head / p->n_head_kv;
  a.tile_rows = MR;
  a.row_tiles = (p->T * a.rep + MR - 1) / MR;
  a.block = TaCfg<DT, HD>::kBlock;
  a.part_o = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + o_bytes);
  int sms = 0;
  int st = num_sms(&sms);
  if (st) return st;
  const size_t smem = TaCfg<DT, HD>::kSmem;
  NS_CUDA_TRY(cudaFuncSetAttribute(tree_attn_kernel<DT, HD, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  a.grid = std::min(sms, kTaMaxSms) * TaCfg<DT, HD>::kCtas;
  NS_CUDA_TRY(launch_pdl(tree_attn_kernel<DT, HD, WM>, dim3(a.grid), kTaThreads, smem, stream, 1, a));
  return ta_join<DT, HD>(a, stream);
}

#include "tree_attn_tc.cuh"

template <int DT, int HD>
static int ta_by_rows(const ns_tree_attn_t* p, void* ws, ns_stream_t stream, size_t* bytes) {
  if constexpr (DT != NS_F32)
    if (ta_takes_tc(p)) return ta_run_tc<DT, HD>(p, ws, stream, bytes);
  switch (ta_groups(p)) {
    case 1: return ta_run<DT, HD, 1>(p, ws, stream, bytes);
    case 2: return ta_run<DT, HD, 2>(p, ws, stream, bytes);
    case 4: return ta_run<DT, HD, 4>(p, ws, stream, bytes);
    default: return ta_run<DT, HD, 8>(p, ws, stream, bytes);
  }
}

// Launches the call, or with `bytes` says what workspace it takes.
static int ta_dispatch(const ns_tree_attn_t* p, void* ws, ns_stream_t stream, size_t* bytes) {
  const bool wide = p->head_dim > 64;
  switch (p->dtype) {
    case NS_F32: return wide ? ta_by_rows<NS_F32, 128>(p, ws, stream, bytes) : ta_by_rows<NS_F32, 64>(p, ws, stream, bytes);
    case NS_F16: return wide ? ta_by_rows<NS_F16, 128>(p, ws, stream, bytes) : ta_by_rows<NS_F16, 64>(p, ws, stream, bytes);
    default: return wide ? ta_by_rows<NS_BF16, 128>(p, ws, stream, bytes) : ta_by_rows<NS_BF16, 64>(p, ws, stream, bytes);
  }
}

static int ta_check(const ns_tree_attn_t* p) {
  if (!p) return fail(NS_ERR_INVALID, "ns_tree_attn: null parameters");
  if (p->B < 0 || p->T < 0 || p->max_ctx < 1 || p->window < 0)
    return fail(NS_ERR_INVALID, "ns_tree_attn: B %d, T %d, max_ctx %d, window %d", p->B, p->T, p->max_ctx, p->window);
  // slots are counted in 32 bits, up to the nodes and a block past the last one
  if (p->max_ctx > INT32_MAX - 1024) return fail(NS_ERR_UNSUPPORTED, "ns_tree_attn: caches of %d slots", p->max_ctx);
  if (!float_type_ok(p->dtype)) return fail(NS_ERR_INVALID, "ns_tree_attn: bad dtype %d", p->dtype);
  if (p->T > NS_TREE_MAX_NODES)
    return fail(NS_ERR_UNSUPPORTED, "ns_tree_attn: %d nodes (at most %d)", p->T, NS_TREE_MAX_NODES);
  if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8)
    return fail(NS_ERR_UNSUPPORTED, "ns_tree_attn: head_dim %d (a multiple of 8 up to 128)", p->head_dim);
  if (p->n_head_kv < 1 || p->n_head < 1 || p->n_head % p->n_head_kv)
    return fail(NS_ERR_INVALID, "ns_tree_attn: %d query heads over %d kv heads", p->n_head, p->n_head_kv);
  if (p->n_head > 65536 || p->B > (1 << 20))
    return fail(NS_ERR_UNSUPPORTED, "ns_tree_attn: %d heads, %d sequences", p->n_head, p->B);
  if (!(p->scale > 0.f) || p->scale > 3e38f) return fail(NS_ERR_INVALID, "ns_tree_attn: scale must be positive and finite");
  return NS_OK;
}

}  // namespace ns

extern "C" int ns_tree_attn_workspace_bytes(const ns_tree_attn_t* p, size_t* bytes) {
  using namespace ns;
  if (!bytes) return fail(NS_ERR_INVALID, "ns_tree_attn_workspace_bytes: null output");
  int st = ta_check(p);
  if (st) return st;
  return ta_dispatch(p, nullptr, nullptr, bytes);
}

extern "C" int ns_tree_attn(const ns_tree_attn_t* p, void* workspace, size_t workspace_bytes, ns_stream_t stream) {
  using namespace ns;
  int st = ta_check(p);
  if (st) return st;
  if (p->B == 0 || p->T == 0) return NS_OK;
  if (!p->lens || !p->q || !p->k_cache || !p->v_cache || !p->out || !workspace)
    return fail(NS_ERR_INVALID, "ns_tree_attn: null pointer");
  const int64_t m = p->dtype == NS_F32 ? 4 : 8;
  if (!aligned_to(p->k_cache, 16) || !aligned_to(p->v_cache, 16) || !strides_multiple(p->kc_stride, 3, m) ||
      !strides_multiple(p->vc_stride, 3, m))
    return fail(NS_ERR_INVALID, "ns_tree_attn: caches must start and step by 16 bytes");
  if (!aligned_to(workspace, 256)) return fail(NS_ERR_INVALID, "ns_tree_attn: workspace must be 256-byte aligned");
  size_t need = 0;
  st = ta_dispatch(p, nullptr, nullptr, &need);
  if (st) return st;
  if (workspace_bytes < need)
    return fail(NS_ERR_SIZE, "ns_tree_attn: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  return ta_dispatch(p, workspace, stream, nullptr);
}
