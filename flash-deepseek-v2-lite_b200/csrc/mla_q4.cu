// Latent attention over the paged 4-bit cache (latent4.cuh):
//   score[h, s] = scale * (q_abs[h] . latent[s] + q_pe[h] . rope[s]),  s = 0 .. position
//   o_lat[h]    = sum_s softmax(score)[h, s] * latent[s]
// for the 16 heads of every query row; the tokens of a row come from the pages of its
// block-table row.
#include "latent4.cuh"
#include "params.cuh"

namespace dsv2 {

constexpr int kQ4Pos = 128;                                  // positions of a tile: 8 blocks
constexpr int kQ4TileBlocks = kQ4Pos / kL4Tokens;
constexpr int kQ4Stages = 3;
constexpr int kQ4StageBytes = kQ4TileBlocks * kL4BlockBytes; // 51200
// per-row cost in blocks, for the work balance: 4 / 8 / 16 / 32 give 17.3 / 16.1 / 16.0 / 16.9 us for 32
// rows of 512, 41.9 / 40.9 / 42.1 / 45.1 for 256 ragged ones, 41.3 / 36.9 / 36.4 / 37.8 for 9 x 3 long ones,
// 57.8 / 55.7 / 58.1 / 62.7 for 100 x 2 of 50 .. 2500
constexpr int kQ4SegUnits = 8;
constexpr int kQ4ScoreWarps = 8;                             // a block of a tile each
constexpr int kQ4PvWarps = 8;                                // 64 latent dims each
constexpr int kQ4Compute = (kQ4ScoreWarps + kQ4PvWarps) * 32;
constexpr int kQ4ProducerWarp = kQ4ScoreWarps + kQ4PvWarps;  // warp 16: copies
constexpr int kQ4Threads = kQ4Compute + 128;                 // a whole warpgroup of which one warp works
// registers a thread: the launch gives 20 warps 96 each; the copy warpgroup hands most of its own on
constexpr int kQ4LaunchRegs = 96, kQ4CopyRegs = 24, kQ4ScoreRegs = 120, kQ4PvRegs = 104;
static_assert(4 * kQ4CopyRegs + kQ4ScoreWarps * kQ4ScoreRegs + kQ4PvWarps * kQ4PvRegs <= kQ4Threads / 32 * kQ4LaunchRegs,
              "register shares exceed the launch's");
constexpr int kQ4QBytes = kHeads * (1024 + 128);             // a query row: q_abs, then q_pe
constexpr int kQ4Steps = 32;                                 // k-steps of 16 latent dims; 4 roped ones follow
constexpr int kQ4PRow = kQ4Pos + 8;                          // row of P
constexpr float kQ4VUp = 256.f;                              // the P V product's values are v / 256
constexpr float kQ4Slack = 8.f;                              // log2 growth of a row's maximum left unscaled

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// (not volatile, unlike mma_bf16_16816: the compiler may move loads and conversions between them)
__device__ __forceinline__ void q4_mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int kRegs>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
__device__ __forceinline__ void q4_bar(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// barrier 1 over the score warps that also says whether any thread's predicate holds
__device__ __forceinline__ bool q4_bar_any(bool pred) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(r)
               : "r"(static_cast<uint32_t>(pred)), "n"(kQ4ScoreWarps * 32)
               : "memory");
  return r != 0;
}
__device__ __forceinline__ uint32_t h2fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t h2mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t b2fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t b2mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {   // 2^x to 2 ulp, results below 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Nibble pairs to the fp16 pairs of the score product (queries scaled into fp16's range).  A
// nibble q at bits 3..0 of a half, under the bits of 1024, is the fp16 number 1024 + q; one at
// bits 7..4, under the bits of 64, is 64 + q: one shift serves four nibbles.  (1024 + q) s - 1032 s
// = (q - 8) s in one fma, exactly: s has 4 significant bits and is at most 60, so 1032 s (12 bits,
// the last 0) and the result (8 bits) are fp16 numbers and the fma rounds once.
struct Q4Scale {
  uint32_t s, b0, b4;   // scale pair, -1032 s, -72 s
};
__device__ __forceinline__ Q4Scale q4_scale(uint32_t codes /* code of each half in its low byte */) {
  Q4Scale r;
  r.s = codes << 7;
  r.b0 = h2mul(r.s, 0xe408e408u);   // -1032
  r.b4 = h2mul(r.s, 0xd480d480u);   // -72
  return r;
}
// (w & mask) | bits in one instruction: it takes one immediate, so the bits are kept in a register
// that the compiler cannot see through (else it splits the two constants over two instructions)
template <uint32_t kMask>
__device__ __forceinline__ uint32_t q4_under(uint32_t w, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(kMask), "r"(bits));
  return r;
}
__device__ __forceinline__ uint32_t q4_opaque(uint32_t bits) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(bits));
  return r;
}
__device__ __forceinline__ uint32_t q4_lo(uint32_t w, const Q4Scale& c, uint32_t m1024) { return h2fma(q4_under<0x000f000fu>(w, m1024), c.s, c.b0); }
__device__ __forceinline__ uint32_t q4_hi(uint32_t w, const Q4Scale& c, uint32_t m64) { return h2fma(q4_under<0x00f000f0u>(w, m64), c.s, c.b4); }

// Nibble pairs to the bf16 pairs of the P V product: P spans more binades than fp16 has (a
// probability far below the row's largest still decides a dim in which that token is 0).  A nibble q
// at bits 3..0 of a half, under the bits of 128, is the bf16 number 128 + q.  One at bits 7..4 alone
// is q 2^-129: bit 7 is the lowest exponent bit, and subnormals and the first binade have the same
// spacing.  So one shift serves four nibbles here too.  To keep the factor of the second kind finite
// all values come out as v 2^-8, made up for at the end.  A code in bits 11..4 of a bf16 number is the
// scale times 2^-112 (subnormals included); every product and fma below is exact (at most 8 bits).
struct Q4ScaleB {
  uint32_t m0, b0;      // scale 2^-8 and -136 times it
  uint32_t m1, b1;      // scale 2^121 and -8 scale 2^-8
};
__device__ __forceinline__ Q4ScaleB q4_scale_b(uint32_t codes) {
  Q4ScaleB r;
  const uint32_t raw = codes << 4;
  r.m0 = b2mul(raw, 0x73807380u);                        // 2^104
  r.b0 = b2mul(raw, 0xf708f708u);                        // -136 * 2^104
  r.m1 = b2mul(b2mul(raw, 0x7f007f00u), 0x74807480u);    // 2^127, then 2^106
  r.b1 = b2mul(raw, 0xf500f500u);                        // -2^107
  return r;
}
__device__ __forceinline__ uint32_t q4_b_lo(uint32_t w, const Q4ScaleB& c, uint32_t m128) { return b2fma(q4_under<0x000f000fu>(w, m128), c.m0, c.b0); }
__device__ __forceinline__ uint32_t q4_b_hi(uint32_t w, const Q4ScaleB& c) { return b2fma(w & 0x00f000f0u, c.m1, c.b1); }

// Bounded mbarrier wait, a loop of four instructions: the waiting warps share the issue slots with
// the working ones.  It gives up after 2^24 polls (seconds), and at once when this CTA already has.
__device__ __forceinline__ bool q4_wait(uint64_t* bar, uint32_t parity, volatile int* s_abort) {
  if (mbar_try_wait(bar, parity)) return true;
  if (*s_abort != 0) return false;
  uint32_t left;
  asm volatile(
      "{\n .reg .pred p;\n mov.u32 %0, 16777216;\n"
      "POLL:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra DONE;\n"
      " sub.u32 %0, %0, 1;\n setp.ne.u32 p, %0, 0;\n @p bra POLL;\n"
      "DONE:\n}\n"
      : "=&r"(left)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (left != 0) return true;
  *s_abort = 1;
  set_device_error(kErrMbarTimeout);
  return false;
}

// Attended length of query row r: 0 .. the positions its table row can hold.
__device__ __forceinline__ int q4_len(const MlaQ4Params& p, int r) {
  const long long pos = p.positions[r];
  const int seq = p.seq_rows ? p.seq_rows[r] : r;
  if (pos < 0 || seq < 0) return 0;
  if (seq >= p.seqs || pos >= static_cast<long long>(p.width) * p.page_blocks * kL4Tokens) {
    set_device_error(kErrIndex);
    return 0;
  }
  return static_cast<int>(pos + 1);
}
// blocks of a row (a row with nothing to attend owns one, fully masked) and its units of work
__device__ __forceinline__ int q4_blocks(int len) { return len > 0 ? (len + kL4Tokens - 1) / kL4Tokens : 1; }
__device__ __forceinline__ int q4_units(int len) { return q4_blocks(len) + kQ4SegUnits; }

// place of a lane's fragment of a step in its row of 32
__device__ __forceinline__ int q4_frag_slot(int step, int lane) { return lane ^ ((step & 6) >> 1); }

struct Q4Smem {
  unsigned char ring[kQ4Stages][kQ4StageBytes];
  unsigned char q[2][kQ4QBytes];            // query rows as they lie in memory
  uint4 qf[kQ4Steps + 4][32];               // the row's A fragments, one per lane: fp16 latent, bf16 roped steps
  bf16 p[2][kHeads][kQ4PRow];               // P, columns in the order the fragments want
  float qinv[kHeads];                       // softmax scale over the power of two that scaled the query
  float smax[kHeads][kQ4ScoreWarps];
  float alpha[2][kHeads];
  float lsum[kQ4ScoreWarps][kHeads];
  float fin[2][kHeads];
  uint64_t full[kQ4Stages], empty[kQ4Stages];
  uint64_t p_full[2], p_empty[2], q_full[2], q_empty[2], fin_full[2], fin_empty[2];
  long long first_S;                        // stream position of the CTA's first row
  int wsum[32];
  int rescale[2];
  int first_row, abort;
};
static_assert(sizeof(Q4Smem) <= 232448, "4-bit latent attention: shared memory exceeds 227 KB");

// One launch, persistent: the rows form one stream of units (kQ4SegUnits of per-row cost, then
// the row's 16-token blocks), cut into equal ranges, one CTA (20 warps, of which 17 work) per SM.  A row inside
// one range writes o_lat; a row cut by a boundary leaves (o, m, l) partials, two slots per CTA
// (slot 0: a row that began before the range), which mla_q4_merge_kernel joins.
//  - warps 0-7, scores: one block (16 positions) of a tile each, all dims; the row's query
//    fragments are made once per row, in shared memory, as fp16 scaled by a power of two per head;
//  - warps 8-15, P V: 64 latent dims each;
//  - warp 16: copies blocks (looked up 32 at a time) and query rows, and notes each row's partials.
// The maximum that P is taken against is kept until a score exceeds it by 2^kQ4Slack: the score
// warps then agree on a new one and the P V warps rescale.
//
// With the merge launch: 64 rows of 8192 tokens 90 us (212 MB, 2.4 TB/s), 64 x 2048 36 us, 256 ragged rows
// of 1 .. 1900 58 us, one row of 512 12 us.  The copies alone take 49 us of the 90, scores without P V 66,
// P V without scores 56: about 33 us of products and as much of conversions on each side (34.8 kFLOP and
// 1024 nibble conversions a token, for 400 bytes) overlap with each other and with the copies only in
// part.  Tiles of 64 positions (7 stages) and conversions taken out on one side changed nothing.
__global__ __launch_bounds__(kQ4Threads, 1) void mla_q4_kernel(const MlaQ4Params p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Q4Smem& sm = *reinterpret_cast<Q4Smem*>(smem_raw);
  volatile int* s_abort = &sm.abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = p.rows;
  if (tid == 0) {
    for (int i = 0; i < kQ4Stages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], kQ4ScoreWarps + kQ4PvWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.p_full[i], kQ4ScoreWarps);
      mbar_init(&sm.p_empty[i], kQ4PvWarps);
      mbar_init(&sm.q_full[i], 1);
      mbar_init(&sm.q_empty[i], kQ4ScoreWarps);
      mbar_init(&sm.fin_full[i], 1);
      mbar_init(&sm.fin_empty[i], kQ4PvWarps);
    }
    sm.abort = 0;
    fence_mbar_init();
  }
  pdl_enter();

  // --- prefix sum of the rows' units; this CTA's range [start, end) and its first row
  long long T = 0;
  int mine0 = 0, incl0 = 0;
  for (int base = 0; base < R; base += kQ4Threads) {
    const int r = base + tid;
    const int u = r < R ? q4_units(q4_len(p, r)) : 0;
    int v = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += w;
    }
    if (lane == 31) sm.wsum[warp] = v;
    if (base == 0) {
      mine0 = u;
      incl0 = v;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQ4Threads / 32; ++w) T += sm.wsum[w];
    if (base + kQ4Threads < R) __syncthreads();
  }
  const long long c = blockIdx.x;
  const long long n_cta = min(static_cast<long long>(gridDim.x), (T + p.min_units - 1) / p.min_units);
  if (c >= n_cta) {
    if (tid == 0) p.cuts[c] = make_int4(-1, 0, 0, 0);
    return;
  }
  const long long start = mla_range_start(c, T, n_cta), end = mla_range_start(c + 1, T, n_cta);
  if (R <= kQ4Threads) {
    long long off = 0;
#pragma unroll
    for (int w = 0; w < kQ4Threads / 32; ++w)
      if (w < warp) off += sm.wsum[w];
    const long long S = off + incl0 - mine0;
    if (tid < R && S <= start && start < S + mine0) {
      sm.first_S = S;
      sm.first_row = tid;
    }
  } else {
    long long run = 0;
    for (int base = 0; base < R && run <= start; base += kQ4Threads) {
      __syncthreads();
      const int r = base + tid;
      const int u = r < R ? q4_units(q4_len(p, r)) : 0;
      int v = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
      }
      if (lane == 31) sm.wsum[warp] = v;
      __syncthreads();
      long long off = run, total = 0;
#pragma unroll
      for (int w = 0; w < kQ4Threads / 32; ++w) {
        if (w < warp) off += sm.wsum[w];
        total += sm.wsum[w];
      }
      const long long S = off + v - u;
      if (r < R && S <= start && start < S + u) {
        sm.first_S = S;
        sm.first_row = r;
      }
      run += total;
    }
  }
  __syncthreads();
  const long long S0 = sm.first_S;
  const int r0 = sm.first_row;

  // the row at stream position S: its blocks [j0, j1) in this CTA's range
  auto segment = [&](long long S, int nblk, int& j0, int& j1) {
    const long long St = S + kQ4SegUnits;
    j0 = static_cast<int>(max(0LL, start - St));
    j1 = static_cast<int>(min(static_cast<long long>(nblk), end - St));
    return St >= start && St + nblk <= end;   // wholly in the range
  };

  if (warp >= kQ4ProducerWarp) {
    // ================= producer warp
    regs_dec<kQ4CopyRegs>();
    if (warp > kQ4ProducerWarp) return;
    if (lane == 0) {
      // the second CTA of a cut row notes the row, its first partial slot and their number; every
      // CTA writes its entry, also one whose range holds no block (per-row units alone)
      const long long St = S0 + kQ4SegUnits;
      int4 cut = make_int4(-1, 0, 0, 0);
      if (St < start && mla_owner(St, T, n_cta) == c - 1) {
        const int nblk = q4_blocks(q4_len(p, r0));
        cut = make_int4(r0, static_cast<int>(2 * (c - 1)) + mla_slot(S0, mla_range_start(c - 1, T, n_cta)),
                        static_cast<int>(mla_owner(St + nblk - 1, T, n_cta) - c + 2), 0);
      }
      p.cuts[c] = cut;
    }
    bool ok = true;
    int seg = 0, st = 0;
    uint32_t round = 0;   // times the ring has been filled
    long long S = S0;
    for (int r = r0; S + kQ4SegUnits < end && r < R; ++r, ++seg) {
      const int len = q4_len(p, r), nblk = q4_blocks(len);
      int j0, j1;
      segment(S, nblk, j0, j1);
      // query block into buffer seg & 1
      if (seg >= 2 && ok) ok = q4_wait(&sm.q_empty[seg & 1], static_cast<uint32_t>(((seg >> 1) - 1) & 1), s_abort);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        unsigned char* dq = sm.q[seg & 1];
        uint64_t* bar = &sm.q_full[seg & 1];
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, kQ4QBytes);
          bulk_load(smem_u32(dq), p.q_abs + static_cast<long long>(r) * kHeads * 512, kHeads * 1024, bar);
          bulk_load(smem_u32(dq + kHeads * 1024), p.q_pe + static_cast<long long>(r) * kHeads * 64, kHeads * 128, bar);
        }
        __syncwarp();
      }
      const int* table = len > 0 ? p.table + (p.seq_rows ? p.seq_rows[r] : r) * p.table_stride : nullptr;
      for (int jb = j0; jb < j1; jb += 32) {
        // 32 blocks' addresses, one per lane
        long long blk = 0;
        if (table && jb + lane < j1) {
          const int j = jb + lane;
          blk = static_cast<long long>(table[j / p.page_blocks]) * p.page_blocks + j % p.page_blocks;
          if (blk < 0 || blk >= p.n_blocks) {
            set_device_error(kErrIndex);
            blk = 0;
          }
        }
        for (int t = 0; t < 32 && jb + t < j1; t += kQ4TileBlocks) {
          if (round > 0 && ok) ok = q4_wait(&sm.empty[st], (round - 1) & 1, s_abort);
          ok = __all_sync(0xffffffffu, ok);
          const int nb = min(kQ4TileBlocks, j1 - jb - t);
          if (ok && lane == 0) mbar_arrive_expect_tx(&sm.full[st], nb * kL4BlockBytes);
          __syncwarp();
          if (ok && lane >= t && lane < t + nb)
            bulk_load(smem_u32(sm.ring[st] + (lane - t) * kL4BlockBytes), p.cache + blk * kL4BlockBytes, kL4BlockBytes, &sm.full[st]);
          if (++st == kQ4Stages) {
            st = 0;
            ++round;
          }
        }
      }
      S += nblk + kQ4SegUnits;
    }
    // every copy has landed before the CTA may exit (consumed ones at once; after a failed wait,
    // the ones nobody consumed)
    for (int i = 0; i < kQ4Stages; ++i) {
      if (i >= st && round == 0) break;   // never filled
      const uint32_t last = i < st ? round : round - 1;
      for (uint32_t n = 0; n < (1u << 20) && !mbar_try_wait(&sm.full[i], last & 1); ++n) {
      }
    }
    for (int k = max(0, seg - 2); k < seg; ++k)
      for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(&sm.q_full[k & 1], static_cast<uint32_t>((k >> 1) & 1)); ++i) {
      }
    return;
  }

  const int gq = lane >> 2, tq = lane & 3;
  int seg = 0, st = 0;
  uint32_t ring_phase = 0, g = 0;   // parity of the ring's round; tiles of this CTA so far
  long long S = S0;
  auto next_tile = [&]() {
    ++g;
    if (++st == kQ4Stages) {
      st = 0;
      ring_phase ^= 1;
    }
  };

  if (warp < kQ4ScoreWarps) {
    // ================= score warps
    regs_inc<kQ4ScoreRegs>();
    const uint32_t m1024 = q4_opaque(0x64006400u), m64 = q4_opaque(0x54005400u);
    // B fragment column gq of the 8 positions of half i of a block: token 8 i + (gq >> 1) + 4 (gq & 1);
    // lane tq takes groups 4 gi + tq
    const int tok = (gq >> 1) + 4 * (gq & 1);
    const int fx = l4_group_xor(tok);
    const int base = warp * kL4BlockBytes;
    const int off_w = base + tok * 256 + ((tq ^ (fx & 3)) << 4);   // group gi: + 64 (gi ^ (fx >> 2))
    const int off_s = base + kL4ScaleOff + 16 * tq + 4 * (gq >> 1);
    const int off_r = base + kL4RopeOff + tok * 128 + (tq << 4);   // chunk 4 h + tq: + 64 (h ^ (tok >> 2))
    // bytes (gq & 1) and (gq & 1) + 2 of the scale word, into both halves
    const uint32_t sel0 = (gq & 1) ? 0x4141u : 0x4040u, sel1 = (gq & 1) ? 0x4343u : 0x4242u;
    for (int r = r0; S + kQ4SegUnits < end && r < R; ++r, ++seg) {
      const int len = q4_len(p, r), nblk = q4_blocks(len);
      int j0, j1;
      const bool complete = segment(S, nblk, j0, j1);
      // --- query fragments: thread (heads h and h + 8, part e) takes pieces e + 16 i of 8 dims (words
      // 4 (e & 3) .. of group 4 i + e / 4), and parts 0 .. 7 a piece of 8 roped dims.  Every score warp is
      // past the previous row's products (row-end barrier)
      q4_wait(&sm.q_full[seg & 1], static_cast<uint32_t>((seg >> 1) & 1), s_abort);
      if (warp < 4) {
        const int h = tid >> 4, e = tid & 15;
        const unsigned char* sq = sm.q[seg & 1];
        uint4 u[2][5];
        float up[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
          for (int i = 0; i < 4; ++i) u[hh][i] = *reinterpret_cast<const uint4*>(sq + (h + 8 * hh) * 1024 + e * 16 + 256 * i);
          u[hh][4] = *reinterpret_cast<const uint4*>(sq + kHeads * 1024 + (h + 8 * hh) * 128 + (e & 7) * 16);
          float amax = 0.f;
#pragma unroll
          for (int i = 0; i < 5; ++i) {
            const uint4 v = u[hh][i];
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(bf16lo(v.x)), fabsf(bf16hi(v.x))), fmaxf(fabsf(bf16lo(v.y)), fabsf(bf16hi(v.y)))));
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(bf16lo(v.z)), fabsf(bf16hi(v.z))), fmaxf(fabsf(bf16lo(v.w)), fabsf(bf16hi(v.w)))));
          }
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          // 2^k brings the head's largest element into [2^13, 2^14): bf16 elements down to 2^-27 of it
          // stay exact in fp16.  k is kept in -100 .. 100 so that 2^k and 2^-k are normal
          int k = 13 - (static_cast<int>(__float_as_uint(amax) >> 23) - 127);
          k = max(-100, min(100, k));
          up[hh] = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
          if (e == 0) sm.qinv[h + 8 * hh] = __uint_as_float(static_cast<uint32_t>(127 - k) << 23) * p.scale_log2;
        }
        // word j of group c holds its dims (2 j, 2 j + 1): step 8 (c / 4) + j / 2, registers 2 (j & 1) and
        // 2 (j & 1) + 1 (the two heads) of lane (h, c & 3)
        auto f16 = [&](int hh, uint32_t w) { return pack_f16x2(bf16lo(w) * up[hh], bf16hi(w) * up[hh]); };
        auto b16 = [&](int hh, uint32_t w) { return pack_bf16x2(bf16lo(w) * up[hh], bf16hi(w) * up[hh]); };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int step = 8 * i + 2 * (e & 3), ln = h * 4 + (e >> 2);
          const uint4 v0 = u[0][i], v1 = u[1][i];
          sm.qf[step][q4_frag_slot(step, ln)] = make_uint4(f16(0, v0.x), f16(1, v1.x), f16(0, v0.y), f16(1, v1.y));
          sm.qf[step + 1][q4_frag_slot(step + 1, ln)] = make_uint4(f16(0, v0.z), f16(1, v1.z), f16(0, v0.w), f16(1, v1.w));
        }
        if (e < 8) {
          const int step = kQ4Steps + 2 * (e >> 2), ln = h * 4 + (e & 3);
          const uint4 v0 = u[0][4], v1 = u[1][4];
          sm.qf[step][q4_frag_slot(step, ln)] = make_uint4(b16(0, v0.x), b16(1, v1.x), b16(0, v0.y), b16(1, v1.y));
          sm.qf[step + 1][q4_frag_slot(step + 1, ln)] = make_uint4(b16(0, v0.z), b16(1, v1.z), b16(0, v0.w), b16(1, v1.w));
        }
      }
      q4_bar(1, kQ4ScoreWarps * 32);
      if (lane == 0) mbar_arrive(&sm.q_empty[seg & 1]);
      const float inv0 = sm.qinv[gq], inv1 = sm.qinv[gq + 8];
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;   // heads gq, gq + 8

      for (int jt = j0; jt < j1; jt += kQ4TileBlocks, next_tile()) {
        const int buf = static_cast<int>(g & 1);
        q4_wait(&sm.full[st], ring_phase, s_abort);
        float s[2][4];
        if (jt + warp < j1) {
          const unsigned char* kv = sm.ring[st];
#pragma unroll
          for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
          for (int gi = 0; gi < 4; ++gi) {
            const uint32_t sw = *reinterpret_cast<const uint32_t*>(kv + off_s + 64 * gi);
            const Q4Scale sc[2] = {q4_scale(__byte_perm(sw, 0, sel0)), q4_scale(__byte_perm(sw, 0, sel1))};
            const uint4 u[2] = {*reinterpret_cast<const uint4*>(kv + off_w + 64 * (gi ^ (fx >> 2))),
                                *reinterpret_cast<const uint4*>(kv + off_w + 2048 + 64 * (gi ^ (fx >> 2)))};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int ks = 8 * gi + 2 * i;
              const uint4 q0 = sm.qf[ks][q4_frag_slot(ks, lane)], q1 = sm.qf[ks + 1][q4_frag_slot(ks + 1, lane)];
              const uint32_t a0[4] = {q0.x, q0.y, q0.z, q0.w}, a1[4] = {q1.x, q1.y, q1.z, q1.w};
              uint32_t w[2];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                w[j] = i == 0 ? u[j].x : i == 1 ? u[j].y : i == 2 ? u[j].z : u[j].w;
                mma_f16_16816(s[j], a0, q4_lo(w[j], sc[j], m1024), q4_hi(w[j], sc[j], m64));
              }
#pragma unroll
              for (int j = 0; j < 2; ++j)
                mma_f16_16816(s[j], a1, q4_lo(w[j] >> 8, sc[j], m1024), q4_hi(w[j] >> 8, sc[j], m64));
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int ks = kQ4Steps + 2 * h;
            const uint4 q0 = sm.qf[ks][q4_frag_slot(ks, lane)], q1 = sm.qf[ks + 1][q4_frag_slot(ks + 1, lane)];
            const uint32_t a0[4] = {q0.x, q0.y, q0.z, q0.w}, a1[4] = {q1.x, q1.y, q1.z, q1.w};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint4 u = *reinterpret_cast<const uint4*>(kv + off_r + 1024 * j + 64 * (h ^ (tok >> 2)));
              q4_mma_bf16(s[j], a0, u.x, u.y);
              q4_mma_bf16(s[j], a1, u.z, u.w);
            }
          }
          const int t0 = (jt + warp) * kL4Tokens + tq;   // columns 2 tq, 2 tq + 1: tokens t0 + 8 j, + 4
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[j][0] *= inv0;
            s[j][1] *= inv0;
            s[j][2] *= inv1;
            s[j][3] *= inv1;
            if (t0 + 8 * j >= len) s[j][0] = s[j][2] = -INFINITY;
            if (t0 + 8 * j + 4 >= len) s[j][1] = s[j][3] = -INFINITY;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = -INFINITY;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[st]);   // done with the tile
        const float x0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        const float x1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
        const bool grow = q4_bar_any(x0 > m0 + kQ4Slack || x1 > m1 + kQ4Slack);
        float a0 = 1.f, a1 = 1.f;
        if (grow) {
          float y0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1)), y1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
          y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, 2));
          y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, 2));
          if (tq == 0) {
            sm.smax[gq][warp] = y0;
            sm.smax[gq + 8][warp] = y1;
          }
          q4_bar(1, kQ4ScoreWarps * 32);
          float n0 = m0, n1 = m1;
#pragma unroll
          for (int w = 0; w < kQ4ScoreWarps; ++w) {
            n0 = fmaxf(n0, sm.smax[gq][w]);
            n1 = fmaxf(n1, sm.smax[gq + 8][w]);
          }
          a0 = ex2(m0 - (n0 == -INFINITY ? 0.f : n0));
          a1 = ex2(m1 - (n1 == -INFINITY ? 0.f : n1));
          l0 *= a0;
          l1 *= a1;
          m0 = n0;
          m1 = n1;
        }
        const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
        if (g >= 2) q4_wait(&sm.p_empty[buf], ((g >> 1) - 1) & 1, s_abort);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // P is bf16 (2^-8; another bf16 part of it would double the P V product, which bounds long rows).  l sums
          // what is stored: the weights that are used add up to 1, and a token that decides the row alone comes out
          // as it is in the cache
          const uint32_t w0 = pack_bf16x2(ex2(s[j][0] - u0), ex2(s[j][1] - u0));
          const uint32_t w1 = pack_bf16x2(ex2(s[j][2] - u1), ex2(s[j][3] - u1));
          l0 += bf16lo(w0) + bf16hi(w0);
          l1 += bf16lo(w1) + bf16hi(w1);
          const int col = 16 * warp + 8 * j + 2 * tq;
          *reinterpret_cast<uint32_t*>(&sm.p[buf][gq][col]) = w0;
          *reinterpret_cast<uint32_t*>(&sm.p[buf][gq + 8][col]) = w1;
        }
        if (warp == 0) {
          if (tq == 0) {
            sm.alpha[buf][gq] = a0;
            sm.alpha[buf][gq + 8] = a1;
          }
          if (lane == 0) sm.rescale[buf] = grow;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[buf]);
      }

      // --- row end: l over the quad and the score warps; warp 0 publishes 1 / l
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      if (tq == 0) {
        sm.lsum[warp][gq] = l0;
        sm.lsum[warp][gq + 8] = l1;
      }
      q4_bar(1, kQ4ScoreWarps * 32);
      if (warp == 0) {
        const int fb = seg & 1;
        if (seg >= 2) q4_wait(&sm.fin_empty[fb], static_cast<uint32_t>(((seg >> 1) - 1) & 1), s_abort);
        if (tq == 0) {
          float L0 = 0.f, L1 = 0.f;
#pragma unroll
          for (int w = 0; w < kQ4ScoreWarps; ++w) {
            L0 += sm.lsum[w][gq];
            L1 += sm.lsum[w][gq + 8];
          }
          sm.fin[fb][gq] = L0 > 0.f ? kQ4VUp / L0 : (L0 == 0.f ? 0.f : L0);   // NaN stays NaN
          sm.fin[fb][gq + 8] = L1 > 0.f ? kQ4VUp / L1 : (L1 == 0.f ? 0.f : L1);
          if (!complete) {
            float* ml = p.ml_part + (c * 2 + mla_slot(S, start)) * kHeads * 2;
            ml[gq * 2] = m0;
            ml[gq * 2 + 1] = L0;
            ml[(gq + 8) * 2] = m1;
            ml[(gq + 8) * 2 + 1] = L1;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.fin_full[fb]);
      }
      // lsum is written again only after the next row's tile barriers
      S += nblk + kQ4SegUnits;
    }
  } else {
    // ================= P V warps: latent dims [64 pv, 64 pv + 64); lane gq owns dims 64 pv + 8 gq
    // .. + 8, one word, whose dim t is column gq of n-tile t; lane tq takes tokens tq + 4 i
    regs_inc<kQ4PvRegs>();
    const uint32_t m128 = q4_opaque(0x43004300u);
    const int pv = warp - kQ4ScoreWarps;
    const int grp = 2 * pv + (gq >> 2);
    const int off0 = tq * 256 + ((grp ^ l4_group_xor(tq)) << 4) + 4 * (gq & 3);
    const int off1 = (tq + 4) * 256 + ((grp ^ l4_group_xor(tq + 4)) << 4) + 4 * (gq & 3);
    const int off_s = kL4ScaleOff + 16 * grp + 4 * tq;
    const int mi = lane >> 3, ri = lane & 7;
    for (int r = r0; S + kQ4SegUnits < end && r < R; ++r, ++seg) {
      const int len = q4_len(p, r), nblk = q4_blocks(len);
      int j0, j1;
      const bool complete = segment(S, nblk, j0, j1);
      float o[8][4];
#pragma unroll
      for (int t = 0; t < 8; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
      for (int jt = j0; jt < j1; jt += kQ4TileBlocks, next_tile()) {
        const int buf = static_cast<int>(g & 1);
        q4_wait(&sm.p_full[buf], (g >> 1) & 1, s_abort);
        q4_wait(&sm.full[st], ring_phase, s_abort);
        if (sm.rescale[buf]) {
          const float a0 = sm.alpha[buf][gq], a1 = sm.alpha[buf][gq + 8];
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            o[t][0] *= a0;
            o[t][1] *= a0;
            o[t][2] *= a1;
            o[t][3] *= a1;
          }
        }
        const int nb = min(kQ4TileBlocks, j1 - jt);
        const unsigned char* tile = sm.ring[st];
        const uint32_t p_row = smem_u32(&sm.p[buf][(mi & 1) * 8 + ri][(mi >> 1) * 8]);
        // what a lane needs of a block; the next block's is on its way while one is computed
        struct Part {
          uint32_t pa[4], w0, w1, w2, w3, sw;
        };
        auto load = [&](int b) {
          const unsigned char* kv = tile + b * kL4BlockBytes;
          Part q;
          ldmatrix_x4(p_row + 32 * b, q.pa[0], q.pa[1], q.pa[2], q.pa[3]);
          q.w0 = *reinterpret_cast<const uint32_t*>(kv + off0);
          q.w1 = *reinterpret_cast<const uint32_t*>(kv + off1);
          q.w2 = *reinterpret_cast<const uint32_t*>(kv + off0 + 2048);
          q.w3 = *reinterpret_cast<const uint32_t*>(kv + off1 + 2048);
          q.sw = *reinterpret_cast<const uint32_t*>(kv + off_s);
          return q;
        };
        auto block = [&](const Part& q) {
          const Q4ScaleB c01 = q4_scale_b(__byte_perm(q.sw, 0, 0x4140)), c23 = q4_scale_b(__byte_perm(q.sw, 0, 0x4342));
          // even dims of the word are its low half's nibbles, odd ones the high half's
          const uint32_t e01 = __byte_perm(q.w0, q.w1, 0x5410), d01 = __byte_perm(q.w0, q.w1, 0x7632);
          const uint32_t e23 = __byte_perm(q.w2, q.w3, 0x5410), d23 = __byte_perm(q.w2, q.w3, 0x7632);
          q4_mma_bf16(o[0], q.pa, q4_b_lo(e01, c01, m128), q4_b_lo(e23, c23, m128));
          q4_mma_bf16(o[1], q.pa, q4_b_lo(d01, c01, m128), q4_b_lo(d23, c23, m128));
          q4_mma_bf16(o[2], q.pa, q4_b_hi(e01, c01), q4_b_hi(e23, c23));
          q4_mma_bf16(o[3], q.pa, q4_b_hi(d01, c01), q4_b_hi(d23, c23));
          const uint32_t f01 = e01 >> 8, g01 = d01 >> 8, f23 = e23 >> 8, g23 = d23 >> 8;
          q4_mma_bf16(o[4], q.pa, q4_b_lo(f01, c01, m128), q4_b_lo(f23, c23, m128));
          q4_mma_bf16(o[5], q.pa, q4_b_lo(g01, c01, m128), q4_b_lo(g23, c23, m128));
          q4_mma_bf16(o[6], q.pa, q4_b_hi(f01, c01), q4_b_hi(f23, c23));
          q4_mma_bf16(o[7], q.pa, q4_b_hi(g01, c01), q4_b_hi(g23, c23));
        };
        if (jt + kQ4TileBlocks < nblk && nb == kQ4TileBlocks) {   // whole blocks only: no branch between them
          Part cur = load(0);
#pragma unroll
          for (int b = 0; b < kQ4TileBlocks; ++b) {
            Part nxt = cur;
            if (b + 1 < kQ4TileBlocks) nxt = load(b + 1);
            block(cur);
            cur = nxt;
          }
        } else {
#pragma unroll 1
          for (int b = 0; b < nb; ++b) {
            Part q = load(b);
            if (jt + b == nblk - 1) {
              // tokens past the row's length may hold anything, and P = 0 does not cancel an infinity:
              // give them a finite scale
              const int rem = len - (jt + b) * kL4Tokens;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (tq + 4 * i >= rem) q.sw &= ~(0xffu << (8 * i));
            }
            block(q);
          }
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm.empty[st]);
          mbar_arrive(&sm.p_empty[buf]);
        }
      }
      const int fb = seg & 1;
      q4_wait(&sm.fin_full[fb], static_cast<uint32_t>((seg >> 1) & 1), s_abort);
      // columns 2 tq and 2 tq + 1 of the 8 n-tiles: 16 consecutive dims from 64 pv + 16 tq
      if (complete) {
        const float inv[2] = {sm.fin[fb][gq], sm.fin[fb][gq + 8]};
        bf16* ob = p.o_lat + (static_cast<long long>(r) * kHeads + gq) * 512 + 64 * pv + 16 * tq;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          const float i = inv[cc >> 1];
          uint4 v;
          v.x = pack_bf16x2(o[0][cc] * i, o[1][cc] * i);
          v.y = pack_bf16x2(o[2][cc] * i, o[3][cc] * i);
          v.z = pack_bf16x2(o[4][cc] * i, o[5][cc] * i);
          v.w = pack_bf16x2(o[6][cc] * i, o[7][cc] * i);
          *reinterpret_cast<uint4*>(ob + (cc >> 1) * 8 * 512 + 8 * (cc & 1)) = v;
        }
      } else {
        float* op = p.o_part + ((c * 2 + mla_slot(S, start)) * kHeads + gq) * 512 + 64 * pv + 16 * tq;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          float* oc = op + (cc >> 1) * 8 * 512 + 8 * (cc & 1);
          *reinterpret_cast<float4*>(oc) = make_float4(o[0][cc], o[1][cc], o[2][cc], o[3][cc]);
          *reinterpret_cast<float4*>(oc + 4) = make_float4(o[4][cc], o[5][cc], o[6][cc], o[7][cc]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.fin_empty[fb]);
      S += nblk + kQ4SegUnits;
    }
  }
}

// o_lat[r, h] = sum_k 2^(m_k - M) o_k / sum_k 2^(m_k - M) l_k over the partials of a row that was cut.
// A CTA per cut and head: 4 groups of 64 threads take every fourth partial (a long row alone has one
// per SM), then meet in shared memory.  A launch of its own: with the merge in the last CTA of a row, 148
// partials of 32 KB went through one SM, and a row of 8192 took 88 us instead of 21.
__global__ __launch_bounds__(256) void mla_q4_merge_kernel(const MlaQ4Params p) {
  pdl_enter();
  const int h = blockIdx.y, tid = threadIdx.x;
  const int4 cut = __ldcg(p.cuts + blockIdx.x);
  const int r = cut.x, first = cut.y, n = cut.z;
  if (r < 0) return;
  if (r >= p.rows || first < 0 || n < 2 || 2 * (first / 2 + n) > p.part_slots || n > kMlaMaxCtas) {
    if (tid == 0) set_device_error(kErrIndex);   // not what the attention kernel writes
    return;
  }
  __shared__ float s_w[kMlaMaxCtas];
  __shared__ float s_inv;
  __shared__ float4 s_o[4][2][64];
  auto slot = [&](int k) -> long long { return k == 0 ? first : 2LL * (first / 2 + k); };
  if (tid < 32) {
    float M = -INFINITY, den = 0.f;
    for (int k = tid; k < n; k += 32) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.ml_part + (slot(k) * kHeads + h) * 2));
      s_w[k] = ml.x;
      if (ml.y != 0.f) M = fmaxf(M, ml.x);
    }
    M = warp_max(M);
    for (int k = tid; k < n; k += 32) {
      const float l = __ldcg(p.ml_part + (slot(k) * kHeads + h) * 2 + 1);
      const float w = l != 0.f ? ex2(s_w[k] - M) : 0.f;
      s_w[k] = w;
      den += w * l;
    }
    den = warp_sum(den);
    if (tid == 0) s_inv = den != 0.f ? kQ4VUp / den : 0.f;
  }
  __syncthreads();
  const int g = tid >> 6, d = tid & 63;
  float4 acc[2];
  acc[0] = acc[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = g; k < n; k += 4) {
    const float4* o = reinterpret_cast<const float4*>(p.o_part + (slot(k) * kHeads + h) * 512) + d;
    const float4 v = __ldcg(o), u = __ldcg(o + 64);
    const float w = s_w[k];
    acc[0].x += w * v.x;
    acc[0].y += w * v.y;
    acc[0].z += w * v.z;
    acc[0].w += w * v.w;
    acc[1].x += w * u.x;
    acc[1].y += w * u.y;
    acc[1].z += w * u.z;
    acc[1].w += w * u.w;
  }
  s_o[g][0][d] = acc[0];
  s_o[g][1][d] = acc[1];
  __syncthreads();
  if (tid < 128) {
    const float4* o = &s_o[0][0][0] + tid;   // [group][128]
    const float inv = s_inv;
    const float4 a = o[0], b = o[128], c = o[256], e = o[384];
    *reinterpret_cast<uint2*>(p.o_lat + (static_cast<long long>(r) * kHeads + h) * 512 + 4 * tid) =
        make_uint2(pack_bf16x2((a.x + b.x + c.x + e.x) * inv, (a.y + b.y + c.y + e.y) * inv),
                   pack_bf16x2((a.z + b.z + c.z + e.z) * inv, (a.w + b.w + c.w + e.w) * inv));
  }
}

cudaError_t mla_q4_init() {
  return cudaFuncSetAttribute(mla_q4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(Q4Smem)));
}

// One CTA per SM, at most kMlaMaxCtas and at most one per two partial slots; the kernel itself
// uses no more CTAs than the stream has min_units pieces.
cudaError_t launch_mla_q4(const MlaQ4Params& p, int num_sms, cudaStream_t st) {
  const int grid = std::min(std::min(num_sms, kMlaMaxCtas), p.part_slots / 2);
  launch_kernel(mla_q4_kernel, grid, kQ4Threads, sizeof(Q4Smem), st, p);
  launch_kernel(mla_q4_merge_kernel, dim3(grid, kHeads), 256, 0, st, p);
  return cudaGetLastError();
}

}  // namespace dsv2
