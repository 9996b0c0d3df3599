// ns_tree_attn for 16-bit types and many rows: the same list of blocks, with the products on tcgen05.
// Included by tree_attn.cu inside namespace ns.
//
// A CTA has two slots, each a 128-row tile of queries with its scores S and output O in tensor memory:
// while one slot's softmax runs on the CUDA cores, the other slot's products run on the tensor cores.
// PAIR: the slots are two tiles of rows (128 < rows) and every block of keys serves both; else they are
// the same rows and take the blocks in turn, joined at the end.  Roles (one CTA an SM):
//   warps 0-3, 4-7   softmax of slot 0 and 1, a row per thread: S from tensor memory, running maximum,
//                    P = 2^(S - m) in 16 bits back over S, and the output at an item's end
//   warps 8, 11      issue the products of slot 0 and 1: S = Q K^T (both operands in shared memory),
//                    O += P V (P in tensor memory)
//   warp 9           TMA of key and value blocks into two rings
//   warp 10          clears values that are not finite where a block is masked (see below)
// The maximum that S is taken relative to is let lag: O is rescaled only when a row's maximum has
// grown by more than 2^8 (probabilities up to 256 are as exact as those up to 1), which after the
// first blocks is hardly ever, so O stays in tensor memory from block to block.
// The 32-wide loads and stores of tensor memory are .aligned: a __syncwarp() stands before those that follow code in
// which lanes may part (rows that exist and do not, loops over a row's ancestors).  It costs nothing that shows.
// The probabilities that are masked are zero, but zero times a value that is not finite is not: warp 10
// looks through the value tile of a masked block, zeroes such rows and leaves their bits for the softmax
// warps, which add them, from the cache, to the rows that see them.
//
// Measured (device time of a call in a captured graph, bf16, 64 query and 8 kv heads):
//   5 nodes over 131,071 keys, heads of 128        93 us, 5.8 TB/s: the keys' and values' bytes
//   8 x 64-node trees over up to 16,384 keys, 128  230 us, 940 TFLOP/s; the kernel itself 207
//   8 x 27-node trees over up to 8,191 keys, 64    69 us; the kernel 56, the join 11
// (on several GPUs of the kind: 92 to 94, 226 to 236, 69)
// A slot's period (128 keys) is about 3,400 cycles: 1,900 to 2,000 of softmax (a row per thread: 110 to
// read the scores, 400 for the maximum, 1,500 for 128 exponentials at 8 cycles a warp each) and then the
// slot's own products (1,024 cycles at heads of 128, 512 at 64) with the hand-overs around them.  The two
// slots overlap, so the tensor cores are busy half of the time.  A polynomial in place of some of the
// exponentials was slower (its FMAs cost what they save); one issuing warp for both slots 3-13 % slower;
// two issuing warps without turns 25 % slower at heads of 128; scores read again from tensor memory in a
// rolled loop 20 % slower per block.

constexpr int kTcAttnThreads = 384;
constexpr int kTcAttnBlock = 128;  // keys
constexpr float kTcAttnLag = 8.f;  // log2 of how far the maximum may lag

template <int HD>
struct TcAttnCfg {
  static constexpr int kPanels = HD / 64;             // 128-byte column panels of a row
  static constexpr int kPanel = 128 * 128;            // bytes: 128 rows of 128 bytes
  static constexpr int kTile = kPanels * kPanel;      // a tile of queries, keys or values
  static constexpr int kK = HD == 64 ? 4 : 2, kV = HD == 64 ? 4 : 3;  // ring entries
  static constexpr int kTiles = (2 + kK + kV) * kTile;
};

struct TcAttnCtl {
  uint64_t kfull[4], kempty[4], vfull[4], vclean[4], vempty[4];
  uint64_t sfull[2], pready[2], pvdone[2], qready[2];
  uint64_t meet, turn[2], drain[2];
  int64_t u0, u1;              // the run, and where it starts
  TaPos first;
  uint32_t tmem;
  int abort;
  uint32_t bad[4][4];          // value rows of a ring entry that are not finite
  uint64_t anc[kTreeMax];
  int depth[kTreeMax], par[kTreeMax];
};

// K-major / MN-major operand in panels of 128-byte rows, 16-byte chunks XOR-swizzled by row % 8
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version of sm_100
  d |= (uint64_t)2 << 61;  // SWIZZLE_128B
  return d;
}
// kind::f16, fp32 accumulators; b_mn: B is MN-major
template <int DT>
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn) {
  const uint32_t fmt = DT == NS_BF16 ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, float* f) {
  uint32_t* v = reinterpret_cast<uint32_t*>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
// waits for the loads, and holds the 32 values back until then
__device__ __forceinline__ void tmem_wait_ld_x32(float* f) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3]), "+f"(f[4]), "+f"(f[5]), "+f"(f[6]), "+f"(f[7]), "+f"(f[8]),
      "+f"(f[9]), "+f"(f[10]), "+f"(f[11]), "+f"(f[12]), "+f"(f[13]), "+f"(f[14]), "+f"(f[15]), "+f"(f[16]),
      "+f"(f[17]), "+f"(f[18]), "+f"(f[19]), "+f"(f[20]), "+f"(f[21]), "+f"(f[22]), "+f"(f[23]), "+f"(f[24]),
      "+f"(f[25]), "+f"(f[26]), "+f"(f[27]), "+f"(f[28]), "+f"(f[29]), "+f"(f[30]), "+f"(f[31])
      :: "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* tmap, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar)) : "memory");
}

// Pairs of fp32 values in one 64-bit register pair.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// A starting value that the compiler does not see: it would clone a loop's body for its first turn, and
// the launch would fetch the code of both (15 us more when the bodies are as long as the softmax's).
__device__ __forceinline__ int opaque(int v) {
  int r;
  asm volatile("mov.u32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Which of 32 keys from k0 on a row sees: cached ones from klo to len, then the nodes of vis.
__device__ __forceinline__ uint32_t seen_bits(int k0, int len, int klo, uint64_t vis) {
  const int up = min(max(len - k0, 0), 32), dn = min(max(klo - k0, 0), 32), sh = k0 - len;
  const uint64_t below = ((1ull << up) - 1) & ~((1ull << dn) - 1);
  const uint64_t nodes = sh >= 64 || sh <= -32 ? 0 : sh >= 0 ? vis >> sh : vis << -sh;
  return (uint32_t)below | (uint32_t)nodes;
}

// True in one lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

struct TcAttnArgs {
  TaArgs a;
  CUtensorMap kmap, vmap;
};

// A wait looks at the clock and at the other roles only every so many polls: the loops of the roles have
// to stay in the instruction caches.
constexpr uint32_t kTcAttnPolls = 1024;

// An item's part in this CTA's run: n blocks from block blk0.
struct TcItem {
  TaPos pos;
  int n;
};

template <int DT, int HD, bool PAIR>
__global__ void __launch_bounds__(kTcAttnThreads, 1) tree_attn_tc_kernel(const __grid_constant__ TcAttnArgs args) {
  using Cfg = TcAttnCfg<HD>;
  constexpr int BN = kTcAttnBlock, MR = PAIR ? 256 : 128, NK = Cfg::kK, NV = Cfg::kV;
  extern __shared__ uint8_t tc_attn_smem[];
  const TaArgs& a = args.a;
  const ns_tree_attn_t& p = a.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_attn_smem) + 1023) & ~uintptr_t(1023));
  TcAttnCtl& S = *reinterpret_cast<TcAttnCtl*>(base + Cfg::kTiles);
  const uint32_t sq = smem_addr(base), sk = sq + 2 * Cfg::kTile, sv = sk + NK * Cfg::kTile;

  if (tid == 0) {
    constexpr int kUsers = PAIR ? 2 : 1;  // slots that use a ring entry
    prefetch_tmap(&args.kmap);
    prefetch_tmap(&args.vmap);
    for (int i = 0; i < NK; ++i) mbar_init(&S.kfull[i], 1), mbar_init(&S.kempty[i], kUsers);
    for (int i = 0; i < NV; ++i) mbar_init(&S.vfull[i], 1), mbar_init(&S.vclean[i], 1), mbar_init(&S.vempty[i], kUsers);
    for (int i = 0; i < 2; ++i)
      mbar_init(&S.sfull[i], 1), mbar_init(&S.pready[i], 4), mbar_init(&S.pvdone[i], 1), mbar_init(&S.qready[i], 4);
    mbar_init(&S.meet, 8);
    for (int i = 0; i < 2; ++i) mbar_init(&S.turn[i], 1), mbar_init(&S.drain[i], 1);
    S.abort = 0;
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(&S.tmem, 512);
  griddep_wait();
  griddep_launch_dependents();
  if (warp == 9) {  // the run
    const int64_t total = ta_total_warp(a, BN, lane);
    const int runs = ta_runs(a, total);
    const bool busy = (int)blockIdx.x < runs;
    const int64_t lo = busy ? ta_first_unit(total, runs, blockIdx.x) : 0;
    if (lane == 0) {
      S.u0 = lo;
      S.u1 = busy ? ta_first_unit(total, runs, blockIdx.x + 1) : 0;
      if (busy) S.first = ta_locate(a, BN, lo);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const int64_t u0 = S.u0, u1 = S.u1;
  const uint32_t tmem = S.tmem;
  // columns: S of slot 0, 1 at 0, 128 (P over them), O at 256, 256 + HD
  auto s_col = [&](int s) { return tmem + 128u * s; };
  auto o_col = [&](int s) { return tmem + 256u + (uint32_t)HD * s; };

  // A wait that runs out (kWaitLimitNs) ends this role; the others see the flag, or run out themselves.
  auto give_up = [&](uint64_t& since) {
    const uint64_t now = globaltimer_ns();
    if (since == 0) since = now;
    if (now - since > kWaitLimitNs) {
      raise_device_error(NS_DEVERR_COPY_WAIT);
      *(volatile int*)&S.abort = 1;
    }
    return *(volatile int*)&S.abort != 0;
  };
  auto await = [&](uint64_t* bar, uint32_t parity) {
    uint64_t since = 0;
#pragma unroll 1
    for (uint32_t i = 1;; ++i) {
      if (mbar_try_wait(bar, parity)) return true;
      if (i % kTcAttnPolls == 0 && give_up(since)) return false;
    }
  };
  // The same for a whole warp: all of its threads go on or none.  Every poll is voted on, so the loop never
  // diverges: a vote after a loop that threads may leave apart costs 200 cycles even when all are ready.
  auto await_all = [&](uint64_t* bar, uint32_t parity) {
    uint64_t since = 0;
#pragma unroll 1
    for (uint32_t i = 1;; ++i) {
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
      if (i % kTcAttnPolls == 0 && __any_sync(0xffffffffu, give_up(since))) return false;
    }
  };
  auto arrive_warp = [&](uint64_t* bar) {  // one arrival for what all of the warp's threads did
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  // the items of the run, one after another
  auto walk = [&](auto&& body) {
    if (u0 >= u1) return;
    TaPos at = S.first;
#pragma unroll 1
    for (int64_t u = u0; u < u1;) {
      const int n = (int)(u1 - u < at.nblk - at.blk ? u1 - u : at.nblk - at.blk);
      if (!body(TcItem{at, n}, u)) return;
      u += n;
      if (u >= u1) return;
      at.blk += n - 1;
      ta_next(a, BN, at);
    }
  };
  // no row of the block needs a mask (a node is at most T - 1 deep)
  auto is_masked = [&](const TaSpan& sp, int k0) {
    return k0 + BN > sp.len || (p.window > 0 && sp.len + p.T - 1 - k0 >= p.window);
  };

  // registers from the four helper warps to the softmax warps: 256 * 208 + 128 * 88 = 384 * 168
  if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");

  if (warp < 8) {
    // ------------------------------------------------------------------ softmax
    const int s = warp >> 2, row = tid & 127;
    const uint32_t lane_base = (uint32_t)(warp & 3) << 21;  // TMEM lane 32 * (warp % 4) in bits 16+
    const float sc = p.scale * 1.4426950408889634f;
    int done = opaque(0), vbase = opaque(0), cur_b = opaque(-1);  // blocks of this slot, blocks of the run
    uint32_t met = 0;
    auto meet = [&]() {  // barrier of the two warpgroups; bounded like every wait
      arrive_warp(&S.meet);
      return await_all(&S.meet, met++ & 1);
    };
    walk([&](const TcItem& it, int64_t u) {
      const TaSpan sp = ta_span(p, it.pos.b);
      const int b = it.pos.b;
      if (cur_b >= 0 && !meet()) return false;  // both slots are through with the last item
      if (PAIR || s == 0) {  // this tile's queries, zeros past the rows and dims: a warp takes its 32 rows
        constexpr int CH = HD / 8, RPI = 32 / CH;  // 16-byte chunks of a row, rows of one step
        const int ch = lane % CH;
        const uint32_t dst = sq + (PAIR ? s : 0) * Cfg::kTile + (ch >> 3) * Cfg::kPanel;
        const uint16_t* qb = static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] + ch * 8;
        auto chunk = [&](int i, auto&& put) {
          const int rr = (warp & 3) * 32 + i * RPI + lane / CH, gr = it.pos.rt * MR + (PAIR ? s * 128 : 0) + rr;
          const int qt = gr / a.rep;
          const bool ok = qt < p.T && ch * 8 < p.head_dim;
          const uint16_t* q = qb + (ok ? qt * p.q_stride[1] + (it.pos.h * a.rep + gr % a.rep) * p.q_stride[2] : 0);
          const uint32_t d = dst + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4);
          put(d, q, ok);
        };
        if (a.vec & 1) {
#pragma unroll 8
          for (int i = 0; i < 32 / RPI; ++i)
            chunk(i, [&](uint32_t d, const uint16_t* q, bool ok) { cp_async16_z(d, ok ? (const void*)q : p.q, ok); });
        } else {
#pragma unroll 1
          for (int i = 0; i < 32 / RPI; ++i)
            chunk(i, [&](uint32_t d, const uint16_t* q, bool ok) {
              uint32_t w[4] = {0, 0, 0, 0};
              if (ok)
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = (uint32_t)q[2 * j] | ((uint32_t)q[2 * j + 1] << 16);
              sts128(d, w[0], w[1], w[2], w[3]);
            });
        }
        cp_async_commit();
      }
      if (b != cur_b) {
        if (warp == 0) {  // two nodes a lane, the parents in shared memory
#pragma unroll
          for (int i = 0; i < kTreeMax; i += 32)
            if (i + lane < p.T) S.par[i + lane] = p.parents ? p.parents[(int64_t)b * p.T + i + lane] : i + lane - 1;
          __syncwarp();
#pragma unroll 1
          for (int t = lane; t < p.T; t += 32) {
            bool bad = false;
            uint64_t mk = p.parents ? tree_mask(t, [&](int i) { return S.par[i]; }, &bad) : chain_mask(t);
            if (mk && sp.len + t >= p.max_ctx) mk = 0, bad = true;
            if (bad) raise_device_error(NS_DEVERR_ROUTE);
            S.anc[t] = mk;
            S.depth[t] = __popcll(mk) - 1;
          }
        }
        cur_b = b;
        if (!meet()) return false;  // the tree is there
      }
      const int r = it.pos.rt * MR + (PAIR ? s * 128 : 0) + row, t = r / a.rep;
      const int h = it.pos.h * a.rep + r % a.rep;
      const bool has_row = r < p.T * a.rep;
      uint64_t vis = has_row ? S.anc[t] : 0;
      const bool used = vis != 0;
      int klo = used ? 0 : 0x7fffffff;
      if (used && p.window > 0) {
        const int dep = S.depth[t];
        klo = sp.len + dep - p.window + 1;
        for (uint64_t w = vis; w; w &= w - 1) {
          const int nd = __ffsll((long long)w) - 1;
          if (dep - S.depth[nd] >= p.window) vis &= ~(1ull << nd);
        }
      }
      // The tensor-memory instructions below are .aligned: the whole warp has to be at them together, and the
      // code above (rows copied and not, loops as long as a row's ancestors) lets lanes part.
      __syncwarp();
      {
        uint32_t z[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = 0;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) tmem_st_x32(o_col(s) + lane_base + 32 * c, z);
        tmem_wait_st();
      }
      cp_async_wait<0>();
      fence_proxy_async_smem();
      tc_fence_before();
      if (PAIR || s == 0) arrive_warp(&S.qready[PAIR ? s : 0]);

      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = PAIR ? 0 : s; j < it.n; j += PAIR ? 1 : 2) {
        if (!await_all(&S.sfull[s], done & 1)) return false;
        tc_fence_after();
        // The code of a block has to stay small: it is fetched anew by every launch and shares the
        // instruction caches with the other roles.  So what is rare is a rolled loop over tensor memory.
        const int k0 = sp.lo + (it.pos.blk + j) * BN;
        const bool masked = is_masked(sp, k0);
        if (masked) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float y[32];
            tmem_ld_x32(s_col(s) + lane_base + 32 * c, y);
            const uint32_t see = seen_bits(k0 + 32 * c, sp.len, klo, vis);
            tmem_wait_ld_x32(y);
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = see >> i & 1 ? y[i] : -INFINITY;
            tmem_st_x32(s_col(s) + lane_base + 32 * c, reinterpret_cast<const uint32_t*>(y));
          }
          tmem_wait_st();
        }
        float x[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_x32(s_col(s) + lane_base + 32 * c, x + 32 * c);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_ld_x32(x + 32 * c);
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 4; i + 8 <= 128; i += 8)
#pragma unroll
          for (int c = 0; c < 4; ++c) mx[c] = max3(mx[c], x[i + c], x[i + 4 + c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], x[124 + c]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
        // the reference of the exponentials: set by the first keys seen, moved when it lags too far
        const bool move = m == -INFINITY ? top != -INFINITY : top > m + kTcAttnLag;
        if (__any_sync(0xffffffffu, move && m != -INFINITY)) {
          const float f = move && m != -INFINITY ? ex2(m - top) : 1.f;
          if (!await_all(&S.pvdone[s], (done - 1) & 1)) return false;  // O holds the blocks before this one
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            float o[32];
            tmem_ld_x32(o_col(s) + lane_base + 32 * c, o);
            tmem_wait_ld_x32(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= f;
            tmem_st_x32(o_col(s) + lane_base + 32 * c, reinterpret_cast<const uint32_t*>(o));
          }
          tmem_wait_st();
          l *= f;
        }
        if (move) m = top;
        const float ref = (m == -INFINITY ? 0.f : m) + kTaShift<DT>;
        uint64_t sum[2] = {0, 0};
        const uint64_t sc2 = pair2(sc, sc), ref2 = pair2(-ref, -ref);
        // probabilities, rounded to 16 bits: half an ulp each, as large as the output's own rounding
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float e0, e1;
            unpair2(fma2(pair2(x[32 * c + 2 * i], x[32 * c + 2 * i + 1]), sc2, ref2), e0, e1);
            e0 = ex2(e0), e1 = ex2(e1);
            sum[i & 1] = add2(sum[i & 1], pair2(e0, e1));
            pk[i] = pack16<DT>(e0, e1);
          }
          tmem_st_x16(s_col(s) + lane_base + 16 * c, pk);
        }
        float sum0, sum1, sum2, sum3;
        unpair2(sum[0], sum0, sum1);
        unpair2(sum[1], sum2, sum3);
        l += (sum0 + sum1) + (sum2 + sum3);
        if (masked) {
          const int v = vbase + j, st = v % NV;
          if (!await_all(&S.vclean[st], (v / NV) & 1)) return false;
          uint32_t any = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) any |= S.bad[st][w];
          if (any) {
            if (done > 0 && !await_all(&S.pvdone[s], (done - 1) & 1)) return false;
            tc_fence_after();
            tmem_wait_st();
#pragma unroll 1
            for (int kk = 0; kk < BN; ++kk) {
              if (!(S.bad[st][kk >> 5] >> (kk & 31) & 1)) continue;
              uint32_t w;  // its probability, from the column that holds it and its neighbour
              asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;"
                           : "=r"(w) : "r"(s_col(s) + lane_base + (kk >> 1)) : "memory");
              w = kk & 1 ? w >> 16 : w & 0xFFFFu;
              const int nd = k0 + kk - sp.len;
              const bool see = nd < 0 ? k0 + kk >= klo : nd < kTreeMax && (vis >> nd & 1);
              const float pv = DT == NS_F16 ? f16_bits_to_float(w) : __uint_as_float(w << 16);
              const int64_t vrow = b * p.vc_stride[0] + it.pos.h * p.vc_stride[1] + (int64_t)(k0 + kk) * p.vc_stride[2];
#pragma unroll 1
              for (int c = 0; c < HD / 32; ++c) {
                float o[32];
                tmem_ld_x32(o_col(s) + lane_base + 32 * c, o);
                tmem_wait_ld_x32(o);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (see && 32 * c + i < p.head_dim) o[i] = fmaf(pv, load_float(p.v_cache, DT, vrow + 32 * c + i), o[i]);
                __syncwarp();  // lanes whose row does not see the key skipped the loads
                tmem_st_x32(o_col(s) + lane_base + 32 * c, reinterpret_cast<const uint32_t*>(o));
              }
              tmem_wait_st();
            }
          }
        }
        tmem_wait_st();
        tc_fence_before();
        arrive_warp(&S.pready[s]);
        ++done;
      }
      vbase += it.n;

      // the item's rows: out, or into the workspace when other runs have the rest of its keys
      if (done > 0 && !await_all(&S.pvdone[s], (done - 1) & 1)) return false;
      tc_fence_after();
      float f0 = 1.f, f1 = 0.f;
      if constexpr (!PAIR) {  // slot 0 and 1 hold alternate blocks of the same rows; each warpgroup joins half of the dims
        float* ml = reinterpret_cast<float*>(base + Cfg::kTile);  // the unused second tile of queries
        ml[s * 256 + row] = m, ml[s * 256 + 128 + row] = l;
        tc_fence_before();
        if (!meet()) return false;
        tc_fence_after();
        const float ma = ml[row], mb = ml[256 + row];
        m = fmaxf(ma, mb);
        const float ref = m == -INFINITY ? 0.f : m;
        f0 = ex2(ma - ref), f1 = ex2(mb - ref);
        l = ml[128 + row] * f0 + ml[384 + row] * f1;
      }
      const bool whole = it.n == it.pos.nblk;
      const float scale = whole && used ? ta_row_scale<DT>(m, l, p.sinks, h) : 0.f;
      const int slot = 2 * blockIdx.x + (u - it.pos.blk <= u0 ? 0 : 1);
      const int64_t pr = (int64_t)slot * MR + (PAIR ? s * 128 : 0) + row;
      const int64_t oo = b * p.o_stride[0] + t * p.o_stride[1] + h * p.o_stride[2];
      if (!whole && has_row && (PAIR || s == 0)) *reinterpret_cast<float2*>(a.part_ml + pr * 2) = make_float2(ta_part_max(used, m), l);
      constexpr int NC = HD / 32;
#pragma unroll 1
      for (int c = PAIR ? 0 : s * (NC / 2); c < (PAIR ? NC : (s + 1) * (NC / 2)); ++c) {
        __syncwarp();  // lanes without a row do not store (here and above)
        float o[32];
        tmem_ld_x32(o_col(PAIR ? s : 0) + lane_base + 32 * c, o);
        if constexpr (!PAIR) {
          float o2[32];
          tmem_ld_x32(o_col(1) + lane_base + 32 * c, o2);
          tmem_wait_ld_x32(o);
          tmem_wait_ld_x32(o2);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = o[i] * f0 + o2[i] * f1;
        } else {
          tmem_wait_ld_x32(o);
        }
        if (has_row && whole) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            if (32 * c + i < p.head_dim) {
              float y[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) y[k] = used ? o[i + k] * scale : 0.f;
              if (a.vec & 2) {
                store8(p.out, DT, oo + 32 * c + i, y);
              } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) store_float(p.out, DT, oo + 32 * c + i + k, y[k]);
              }
            }
        } else if (has_row) {
          float4* po = reinterpret_cast<float4*>(a.part_o + pr * HD + 32 * c);
#pragma unroll
          for (int i = 0; i < 8; ++i) po[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      __syncwarp();
      tc_fence_before();
      return true;
    });
  } else if (warp == 8 || warp == 11) {
    // ------------------------------------------------------------------ products of one slot
    // A warp per slot, taking turns: P V of a block and Q K^T of the slot's next one go out together, then
    // the other slot's.  In turns the slots stay half a period apart (issued side by side, both products
    // finish late and both softmaxes then compete for the ex2 unit), and what a warp waits for is hidden
    // behind the other's products.  The whole warp walks and waits, one elected lane issues, so the
    // operands stay in uniform registers.
    const int s = warp == 8 ? 0 : 1;
    int cb = opaque(0), items = opaque(0), steps = opaque(0), turns = opaque(0);  // blocks of the run before this item, items, steps of this slot
    bool ok = true;
    const uint64_t qa = sw128_desc(sq + (PAIR ? s : 0) * Cfg::kTile, 16, 1024);
    const uint64_t kd = sw128_desc(sk, 16, 1024), vd = sw128_desc(sv, Cfg::kPanel, 1024);
    const uint32_t ds = s_col(s), dof = o_col(s);
    walk([&](const TcItem& it, int64_t) {
      if (!(ok = await_all(&S.qready[PAIR ? s : 0], items & 1))) return false;
      // one turn: P V of block c_pv (of the run; -1: none), Q K^T of block c_qk
      auto issue = [&](int c_pv, int c_qk) {
        const int vst = c_pv % NV, kst = c_qk % NK;
        if (c_pv >= 0 && !await_all(&S.vclean[vst], (c_pv / NV) & 1)) return false;
        if (c_qk >= 0 && !await_all(&S.kfull[kst], (c_qk / NK) & 1)) return false;
        // slot 0's first turn is free, then each turn follows the other slot's last
        if ((s == 1 || turns > 0) && !await_all(&S.turn[s], (turns - (s == 0 ? 1 : 0)) & 1)) return false;
        ++turns;
        if (c_pv >= 0 && !await_all(&S.pready[s], steps++ & 1)) return false;
        tc_fence_after();
        const uint64_t va = vd + vst * (Cfg::kTile >> 4), ka = kd + kst * (Cfg::kTile >> 4);
        if (elect_one()) {
          if (c_pv >= 0) {
#pragma unroll
            for (int kk = 0; kk < BN / 16; ++kk)
              mma_f16_ts(dof, ds + 8 * kk, va + kk * (2048 >> 4), idesc_f16<DT>(128, HD, true), 1);
            tc_commit(&S.pvdone[s]);
            tc_commit(&S.vempty[vst]);
          }
          if (c_qk >= 0) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * Cfg::kPanel + (kk & 3) * 32) >> 4;
              mma_f16_ss(ds, qa + off, ka + off, idesc_f16<DT>(128, BN, false), kk > 0);
            }
            tc_commit(&S.sfull[s]);
            tc_commit(&S.kempty[kst]);
          }
          mbar_arrive(&S.turn[s ^ 1]);
        }
        __syncwarp();
        return true;
      };
      // both slots take the same number of turns; a slot without a block passes
      constexpr int step = PAIR ? 1 : 2;
      const int j0 = PAIR ? 0 : s, n_turns = PAIR ? it.n : (it.n + 1) / 2;
      ok = issue(-1, j0 < it.n ? cb + j0 : -1);
#pragma unroll 1
      for (int k = 0; ok && k < n_turns; ++k) {
        const int j = j0 + k * step;
        ok = issue(j < it.n ? cb + j : -1, j + step < it.n ? cb + j + step : -1);
      }
      cb += it.n, ++items;
      return ok;
    });
    if (!ok) {  // what was issued has to land before tensor memory is freed
      if (elect_one()) tc_commit(&S.drain[s]);
      mbar_wait_bounded(&S.drain[s], 0);
    }
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------------ copies, one thread
    if (lane == 0) {
      int ck = 0, cv = 0;
      bool ok = true;
      walk([&](const TcItem& it, int64_t) {
        const TaSpan sp = ta_span(p, it.pos.b);
        auto copy = [&](bool key, int j) {
          const int c = key ? ck : cv, ring = key ? NK : NV, st = c % ring;
          uint64_t* full = key ? &S.kfull[st] : &S.vfull[st];
          if (c >= ring && !await(key ? &S.kempty[st] : &S.vempty[st], (c / ring - 1) & 1)) return false;
          mbar_arrive_expect_tx(full, Cfg::kTile);
          const uint32_t dst = (key ? sk : sv) + st * Cfg::kTile;
          const int k0 = sp.lo + (it.pos.blk + j) * BN;
#pragma unroll
          for (int x = 0; x < Cfg::kPanels; ++x)
            tma_load_4d(dst + x * Cfg::kPanel, key ? &args.kmap : &args.vmap, 64 * x, k0, it.pos.h, it.pos.b, full);
          ++(key ? ck : cv);
          return true;
        };
#pragma unroll 1
        for (int j = 0; ok && j < it.n; ++j) {
          ok = copy(true, j);
          if (PAIR) ok = ok && copy(false, j);
          else if (j > 0) ok = ok && copy(false, j - 1);
        }
        if (!PAIR) ok = ok && copy(false, it.n - 1);
        return ok;
      });
      if (!ok) {  // copies in flight land before the CTA leaves
        for (int c = max(0, ck - NK); c < ck; ++c) mbar_wait_bounded(&S.kfull[c % NK], (c / NK) & 1);
        for (int c = max(0, cv - NV); c < cv; ++c) mbar_wait_bounded(&S.vfull[c % NV], (c / NV) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 10) {
    // ------------------------------------------------------------------ values that are not finite
    int cv = 0;
    walk([&](const TcItem& it, int64_t) {
      const TaSpan sp = ta_span(p, it.pos.b);
#pragma unroll 1
      for (int j = 0; j < it.n; ++j, ++cv) {
        const int st = cv % NV;
        if (!await_all(&S.vfull[st], (cv / NV) & 1)) return false;
        if (is_masked(sp, sp.lo + (it.pos.blk + j) * BN)) {
          // a lane looks at one 16-byte chunk of one of four rows at a time; bit i: a bad row of group i
          const uint32_t va = sv + st * Cfg::kTile;
          uint32_t mine = 0;
#pragma unroll 8
          for (int i = 0; i < BN / 4; ++i) {
            uint32_t acc = 0;
#pragma unroll
            for (int x = 0; x < Cfg::kPanels; ++x) acc |= not_finite<DT>(va + x * Cfg::kPanel + i * 512 + lane * 16);
            mine |= acc ? 1u << i : 0u;
          }
          if (lane < 4) S.bad[st][lane] = 0;
          __syncwarp();
          if (__any_sync(0xffffffffu, mine != 0)) {
#pragma unroll 1
            for (int i = 0; i < BN / 4; ++i)
              if (mine >> i & 1) atomicOr(&S.bad[st][i >> 3], 1u << (4 * (i & 7) + (lane >> 3)));
            __syncwarp();
#pragma unroll 1
            for (int i = 0; i < BN / 4; ++i)
              if (S.bad[st][i >> 3] >> (4 * (i & 7) + (lane >> 3)) & 1)
#pragma unroll
                for (int x = 0; x < Cfg::kPanels; ++x) sts128(va + x * Cfg::kPanel + i * 512 + lane * 16, 0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        if (lane == 0) mbar_arrive(&S.vclean[st]);
      }
      return true;
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// Whether the tensor-core kernel takes a 16-bit call: caches that a tensor map describes, and more than 8
// rows or wide heads.  Measured (us, this kernel / the
// mma.sync one, 8 kv heads): 8 rows, 8 x 8192 keys, head_dim 64: 37.0 / 34.6; head_dim 128: 47.1 / 51.6;
// 16 rows: 39.7 / 39.5 and 50.5 / 57.3; 32 rows: 42.0 / 50.7 and 53.1 / 69.6; 128 rows: 44.4 / 95.2 and
// 59.4 / 133.2.
static bool ta_takes_tc(const ns_tree_attn_t* p) {
  const int rows = p->T * (p->n_head / p->n_head_kv);
  if (rows <= 8 && p->head_dim <= 64) return false;
  const int64_t dims[3] = {p->B, p->n_head_kv, p->max_ctx};
  for (int i = 0; i < 3; ++i)
    for (const int64_t* s : {p->kc_stride, p->vc_stride})
      if (dims[i] > 1 && (s[i] <= 0 || s[i] >= (1ll << 38))) return false;
  return true;
}

template <int DT>
static int ta_cache_map(CUtensorMap* m, const ns_tree_attn_t* p, const void* base, const int64_t* stride) {
  EncodeTiledFn fn;
  int st = get_encode_fn(&fn);
  if (st) return st;
  const cuuint64_t dims[4] = {(cuuint64_t)p->head_dim, (cuuint64_t)p->max_ctx, (cuuint64_t)p->n_head_kv, (cuuint64_t)p->B};
  cuuint64_t strides[3];
  const int64_t n[3] = {p->max_ctx, p->n_head_kv, p->B}, el[3] = {stride[2], stride[1], stride[0]};
  for (int i = 0; i < 3; ++i) strides[i] = n[i] > 1 ? (cuuint64_t)el[i] * 2 : 256;  // unused where there is one of them
  const cuuint32_t box[4] = {64, kTcAttnBlock, 1, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, DT == NS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NS_ERR_CUDA, "cuTensorMapEncodeTiled (cache) failed (%d)", (int)r);
  return NS_OK;
}

template <int DT, int HD>
static int ta_run_tc(const ns_tree_attn_t* p, void* ws, ns_stream_t stream, size_t* bytes) {
  const int rep = p->n_head / p->n_head_kv, rows = p->T * rep;
  const bool pair = rows > 128;
  const int MR = pair ? 256 : 128;
  const size_t o_bytes = (size_t)2 * kTaMaxSms * MR * HD * sizeof(float);
  if (bytes) {
    *bytes = o_bytes + (size_t)2 * kTaMaxSms * MR * 2 * sizeof(float);
    return NS_OK;
  }
  TcAttnArgs t;
  t.a.p = *p;
  t.a.rep = rep;
  t.a.tile_rows = MR;
  t.a.row_tiles = (rows + MR - 1) / MR;
  t.a.block = kTcAttnBlock;
  t.a.vec = (aligned_to(p->q, 16) && strides_multiple(p->q_stride, 3, 8) ? 1 : 0) |
            (aligned_to(p->out, 16) && strides_multiple(p->o_stride, 3, 8) ? 2 : 0);
  t.a.part_o = static_cast<float*>(ws);
  t.a.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + o_bytes);
  int sms = 0;
  int st = num_sms(&sms);
  if (st) return st;
  t.a.grid = std::min(sms, kTaMaxSms);
  if ((st = ta_cache_map<DT>(&t.kmap, p, p->k_cache, p->kc_stride))) return st;
  if ((st = ta_cache_map<DT>(&t.vmap, p, p->v_cache, p->vc_stride))) return st;
  constexpr size_t smem = TcAttnCfg<HD>::kTiles + sizeof(TcAttnCtl) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of one SM");
  auto kernel = pair ? tree_attn_tc_kernel<DT, HD, true> : tree_attn_tc_kernel<DT, HD, false>;
  NS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  NS_CUDA_TRY(launch_pdl(kernel, dim3(t.a.grid), kTcAttnThreads, smem, stream, 1, t));
  return ta_join<DT, HD>(t.a, stream);
}
