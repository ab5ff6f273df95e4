// Paged attention for many query rows of a kv head (a tree of drafts, a run of tokens): the arithmetic of
// sage_paged_attn.cu on tcgen05.
//
// A CTA (one per SM) owns QT row tiles of 128 query rows of one kv head and walks its stretch of the list:
//   softmax warps   one warpgroup per row tile, one thread per row: q to TMEM (fp16), then per key tile S from TMEM,
//                   weights (fp16) back over S, O rescaled in TMEM when the references move, epilogue
//   producer warp   TMA of the raw codes and scales into a ring
//   MMA warps       one per row tile: S_t = Q_t K^T, O_t += P_t V (A from TMEM); two score tiles a row tile, so that the
//                   scores of the next key tile are there when the softmax of this one ends
//   4 converter warps   int8 and e4m3 codes to fp16 operand tiles in shared memory, once for all QT * 128 rows, and what
//                   the rows need of each key (factor of its score, its V scale, the log2 of that)
// Codes convert exactly, so there is nothing to choose there.
// TMEM (512 columns): O_t at t D, the score tiles of t at QT D + 128 t, P over the first half of its scores; Q_t behind
// them where it fits (D 64 and 256), else in shared memory (D 96 and 128).
//
// 8 trees of 64 drafts (256 rows a kv head) over up to 8190 keys, 8 kv heads, D 128: 89 us on B200, 578 TFLOP/s (8190 keys
// each: 107, where the few-rows kernel took 373).  48 us with up to 2048 keys, so a good 30 us do not grow with the keys: the start
// of each CTA's stretch, partial rows and their join.  No unit is full: tensor pipe 34 %, issue 47 %.  A key tile passes through
// conversion, scores, softmax and values in about 2000 cycles, and leaving out the exponentials, the loads of what a key needs, or
// most of either product changes the time by less than 10 % each.
#include "sage_paged_attn.cuh"

namespace sage {

template <int D>
struct Wide {
  static constexpr int QT = D == 256 ? 1 : 2;
  static constexpr int kSoftmaxWarps = 4 * QT, kConverters = 4;
  // QT 2: 16 warps (one idle), so that the two warpgroups of the other roles hand registers to the two of softmax: 512
  // threads of 128 at launch, then 256 of 176 and 256 of 80
  static constexpr int kThreads = QT == 2 ? 512 : 32 * (kSoftmaxWarps + 1 + QT + kConverters);
  static constexpr int kLaunchRegs = 128, kSoftmaxRegs = 176, kOtherRegs = 80;
  static_assert(QT != 2 || 256 * (kSoftmaxRegs + kOtherRegs) <= 512 * kLaunchRegs, "register split");
  static constexpr int kRows = 128 * QT;
  static constexpr int kPanels = (D + 63) / 64;            // of 64 channels: 128 bytes a key
  static constexpr int kPanel = kTileKeys * 128;
  static constexpr int kOperand = kPanels * kPanel;        // K or V of a tile in fp16
  static constexpr int kRaw = D == 256 ? 2 : 3;            // ring of raw stages
  static constexpr int kBufs = D == 256 ? 2 : 3;           // ring of operand tiles
  // Q as fp16: in TMEM where there is room beside O and two score tiles a row tile, else in shared memory
  static constexpr bool kQShared = QT * (D + 2 * kTileKeys + D / 2) > 512;
  static constexpr int kO = 0, kS = QT * D, kQ = kS + QT * 2 * kTileKeys;
  static_assert(kQ + (kQShared ? 0 : QT * D / 2) <= 512, "TMEM columns");
  static constexpr int kQPanel = 128 * 128, kQTile = kPanels * kQPanel;   // bytes in shared memory: 64 channels, a row tile
  static constexpr int kParams = 3 * kTileKeys;            // floats of a tile: factor, V scale, its log2
  static constexpr int kSmem = 1024 + kBufs * 2 * kOperand + kRaw * (Tile<D>::kStage + 2 * kTileKeys * 4) +
                               kBufs * kParams * 4 + (kQShared ? QT * kQTile : 0);
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// D(tmem) (+)= A(tmem) * B(smem), fp16 operands, fp32 accumulator.  The whole warp calls; one lane, always the same, issues.
// (With a branch to one lane around the loop the addresses are moved to uniform registers one by one: 87 us for 8 x 64 rows
// over 8190 keys, D 128, 80 us this way.)
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, e;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The same with A in shared memory.
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, e;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 16 (8) consecutive 32-bit columns.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Bit i: byte i of the word is not zero.
__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t w) {
  return ((__vcmpne4(w, 0) & 0x01010101u) * 0x10204080u) >> 28;
}

// tc_commit of the lane that issues.
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred e;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(smem_u32(bar))
      : "memory");
}

// Instruction descriptor, kind::f16: fp16 A and B, fp32 D; b_mn: B is stored with N contiguous.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Descriptor of an operand stored with N contiguous, 128-byte swizzle: panels of 64 columns `panel` bytes apart, groups of
// 8 rows (of K) 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_nmajor(uint32_t smem_addr, uint32_t panel) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// Byte of 16-byte chunk `ch` (8 fp16 channels) of key `row` in an operand tile.
__device__ __forceinline__ int operand_at(int row, int ch) {
  return ch / 8 * (kTileKeys * 128) + row * 128 + (((ch % 8) ^ (row & 7)) << 4);
}

template <typename T, int D>
__global__ void __launch_bounds__(Wide<D>::kThreads, 1)
    paged_wide_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map) {
  using W = Wide<D>;
  using S = Tile<D>;
  constexpr int QT = W::QT;
  extern __shared__ unsigned char smem_raw[];
  __shared__ int64_t warp_sums[W::kThreads / 32], found[2];
  __shared__ uint64_t raw_full[W::kRaw], raw_empty[W::kRaw], k_full[W::kBufs], v_full[W::kBufs], buf_empty[W::kBufs];
  __shared__ uint64_t s_full[QT][2], p_full[QT][2], q_full[QT], o_full[QT], pv_done[QT], all_done[QT];
  __shared__ uint32_t tmem_base;
  __shared__ int given_up;
  __shared__ float q_scale[QT][128];
  unsigned char* operands = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* queries = operands + W::kBufs * 2 * W::kOperand;   // kQShared
  unsigned char* stages = queries + (W::kQShared ? QT * W::kQTile : 0);
  float* scales = reinterpret_cast<float*>(stages + W::kRaw * S::kStage);
  float* params = scales + W::kRaw * 2 * kTileKeys;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    given_up = 0;
    for (int i = 0; i < W::kRaw; ++i) mbar_init(raw_full + i, 1), mbar_init(raw_empty + i, W::kConverters);
    for (int i = 0; i < W::kBufs; ++i) {
      mbar_init(k_full + i, W::kConverters);
      mbar_init(v_full + i, W::kConverters);
      mbar_init(buf_empty + i, QT);
    }
    for (int t = 0; t < QT; ++t) {
      for (int i = 0; i < 2; ++i) mbar_init(s_full[t] + i, 1), mbar_init(p_full[t] + i, 4);
      mbar_init(q_full + t, 4);
      mbar_init(o_full + t, 1);
      mbar_init(pv_done + t, 1);
      mbar_init(all_done + t, 1);
    }
    fence_barrier_init();
  }
  // Nothing of the stream's earlier work is read before it is done; only then may the join start, which reads the lengths
  // before it waits for this kernel.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0) {
    tmem_alloc(&tmem_base, 512);
    tmem_relinquish();
  }
  Cursor now;
  tc_fence_before();
  int64_t todo = locate<W::kThreads>(a, warp_sums, found, now);
  tc_fence_after();
  if (todo == 0) {   // no barrier since the allocation: the scan's lie behind it
    if (warp == 0) tmem_dealloc(tmem_base, 512);
    return;
  }
  const uint32_t tmem = tmem_base;
  // whether row tile t of the unit holds a live row
  auto active = [&](const Cursor& c, int t) { return c.unit % a.row_tiles * W::kRows + t * 128 < c.fresh * a.group; };

  if (warp == W::kSoftmaxWarps) {
    if constexpr (QT == 2) regs_decrease<W::kOtherRegs>();
    load_tiles<D>(a, &k_map, &v_map, now, todo, stages, scales, raw_full, raw_empty, W::kRaw, &given_up);
  } else if (warp > W::kSoftmaxWarps && warp <= W::kSoftmaxWarps + QT) {
    // ------------------------------------------------------------------------------------------------ products
    if constexpr (QT == 2) regs_decrease<W::kOtherRegs>();
    constexpr uint32_t kScores = idesc_f16(128, kTileKeys, false), kValues = idesc_f16(128, D, true);
    const int t = __shfl_sync(0xffffffffu, warp - W::kSoftmaxWarps - 1, 0);
    const uint64_t k_desc = smem_desc_kmajor(smem_u32(operands), 128);
    const uint64_t v_desc = smem_desc_nmajor(smem_u32(operands) + W::kOperand, W::kPanel);
    const uint64_t q_desc = smem_desc_kmajor(smem_u32(queries) + t * W::kQTile, 128);
    const uint32_t s_at = tmem + W::kS + t * 2 * kTileKeys, q_at = tmem + W::kQ + t * (D / 2), o_at = tmem + W::kO + t * D;
    int buf = 0;               // of the tile whose values are next, and of the one whose scores are next
    int ahead = 0;
    uint32_t phase = 0, ahead_phase = 0, p_phase = 0, q_phase = 0;   // p_phase: a bit per score tile
    // scores of the next tile into score tile i
    auto scores = [&](int i) {
      wait_stage(k_full + ahead, ahead_phase, &given_up, a.p.status);
      tc_fence_after();
      const uint64_t k = k_desc + ahead * (2 * W::kOperand / 16);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const uint64_t ks = k + (s / 4 * W::kPanel + s % 4 * 32) / 16;
        if constexpr (W::kQShared)
          mma_f16_ss(s_at + i * kTileKeys, q_desc + (s / 4 * W::kQPanel + s % 4 * 32) / 16, ks, kScores, s > 0);
        else
          mma_f16_ts(s_at + i * kTileKeys, q_at + s * 8, ks, kScores, s > 0);
      }
      commit(s_full[t] + i);
    };
    auto next = [](int& b, uint32_t& p) {
      if (++b == W::kBufs) b = 0, p ^= 1;
    };
    while (todo > 0) {
      const int tiles = __shfl_sync(0xffffffffu, (int)min((int64_t)(now.tiles - now.tile), todo), 0);   // known to be uniform
      if (active(now, t)) {
        wait_stage(q_full + t, q_phase, &given_up, a.p.status);
        q_phase ^= 1;
        scores(0), next(ahead, ahead_phase);
        if (tiles > 1) scores(1), next(ahead, ahead_phase);
#pragma unroll 1
        for (int j = 0; j < tiles; ++j) {
          const int i = j & 1;
          wait_stage(v_full + buf, phase, &given_up, a.p.status);
          wait_stage(p_full[t] + i, p_phase >> i & 1, &given_up, a.p.status);
          p_phase ^= 1u << i;
          tc_fence_after();
          const uint64_t v = v_desc + buf * (2 * W::kOperand / 16);
#pragma unroll
          for (int s = 0; s < kTileKeys / 16; ++s)
            mma_f16_ts(o_at, s_at + i * kTileKeys + s * 8, v + s * (2048 / 16), kValues, j > 0 || s > 0);
          commit(pv_done + t);
          commit(buf_empty + buf);
          next(buf, phase);
          if (j + 2 < tiles) scores(i), next(ahead, ahead_phase);
        }
        commit(o_full + t);
      } else {   // no row of this row tile is live
#pragma unroll 1
        for (int j = 0; j < tiles; ++j) {
          wait_stage(v_full + buf, phase, &given_up, a.p.status);
          if (lane == 0) arrive(buf_empty + buf);
          next(buf, phase);
        }
        ahead = buf, ahead_phase = phase;
      }
      todo -= tiles;
      now.tile += tiles - 1;
      if (todo > 0) advance(a, now);
    }
    commit(all_done + t);   // nothing is in flight when the CTA ends
    wait_stage(all_done + t, 0, &given_up, a.p.status);
    __syncwarp();
  } else if (warp > W::kSoftmaxWarps + QT + W::kConverters) {
    if constexpr (QT == 2) regs_decrease<W::kOtherRegs>();   // idle
  } else if (warp > W::kSoftmaxWarps) {
    // ------------------------------------------------------------------------------------------------ converters
    if constexpr (QT == 2) regs_decrease<W::kOtherRegs>();
    const int ct = tid - 32 * (W::kSoftmaxWarps + 1 + QT);
    int raw = 0, buf = 0;
    uint32_t raw_phase = 0, phase = 0;
    // The eight lanes of a phase of a 16-byte access take four neighbouring chunks of a raw row and of the row that
    // differs in bits 0 and 2: different banks in the raw tile (bit 2) and in the operand tile (bit 0), whose rows are
    // twice as long.
    constexpr int kItems = kTileKeys * (D / 16) / (32 * W::kConverters);
    auto place = [&](int i, int& row, int& ch) {
      const int item = ct + i * 32 * W::kConverters;
      if constexpr (D == 96) {
        row = item / 6, ch = item % 6;
      } else {
        constexpr int kQuads = D / 64;
        const int g = item / 8, pair = g / kQuads;
        ch = g % kQuads * 4 + item % 4;
        row = (pair / 4 * 8 + pair % 4) ^ (item / 4 % 2 * 5);
      }
    };
    constexpr int kTogether = kItems < 4 ? kItems : 4;   // chunks of a thread under way at once
    auto fetch = [&](const unsigned char* from, int i0, uint4 (&v)[kTogether]) {
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        int row, ch;
        place(i0 + i, row, ch);
        v[i] = *reinterpret_cast<const uint4*>(from + S::at(row, ch * 16));
      }
    };
    auto put = [&](unsigned char* to, int i, const uint4& x, const uint4& y) {
      int row, ch;
      place(i, row, ch);
      *reinterpret_cast<uint4*>(to + operand_at(row, 2 * ch)) = x;
      *reinterpret_cast<uint4*>(to + operand_at(row, 2 * ch + 1)) = y;
    };
    for (; todo > 0; --todo) {
      const int key0 = now.tile * kTileKeys, total = now.len + now.fresh;
      wait_stage(raw_full + raw, raw_phase, &given_up, a.p.status);
      wait_stage(buf_empty + buf, phase ^ 1, &given_up, a.p.status);
      const unsigned char* kt = stages + raw * S::kStage;
      unsigned char* to = operands + buf * 2 * W::kOperand;
      if (ct < kTileKeys) {
        const float* sc = scales + raw * 2 * kTileKeys;
        float* out = params + buf * W::kParams;
        const float vs = sc[kTileKeys + ct];
        const bool there = key0 + ct < total;   // no row sees the others
        out[ct] = there ? sc[ct] * a.scale : 0.0f;
        out[kTileKeys + ct] = there ? vs : 0.0f;
        out[2 * kTileKeys + ct] = __log2f(there ? vs : 0.0f);   // of a zero row -infinity
      }
#pragma unroll
      for (int i0 = 0; i0 < kItems; i0 += kTogether) {
        uint4 v[kTogether];
        fetch(kt, i0, v);
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
          uint4 x, y;
          int8_to_f16(v[i].x, x.x, x.y), int8_to_f16(v[i].y, x.z, x.w);
          int8_to_f16(v[i].z, y.x, y.y), int8_to_f16(v[i].w, y.z, y.w);
          put(to, i0 + i, x, y);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) arrive(k_full + buf);
      const bool drafts = key0 + kTileKeys > now.len;
#pragma unroll
      for (int i0 = 0; i0 < kItems; i0 += kTogether) {
        uint4 v[kTogether];
        fetch(kt + S::kBytes, i0, v);
        if (drafts) {
          // codes behind the last key are anything, and a NaN code of a draft that its reader does not see must not
          // reach it through 0 * NaN: both are cleared
#pragma unroll
          for (int i = 0; i < kTogether; ++i) {
            int row, ch;
            place(i0 + i, row, ch);
            if (key0 + row >= total) v[i] = make_uint4(0, 0, 0, 0);
            if (key0 + row >= now.len) {
              v[i].x &= ~__vcmpeq4(v[i].x & 0x7f7f7f7fu, 0x7f7f7f7fu);
              v[i].y &= ~__vcmpeq4(v[i].y & 0x7f7f7f7fu, 0x7f7f7f7fu);
              v[i].z &= ~__vcmpeq4(v[i].z & 0x7f7f7f7fu, 0x7f7f7f7fu);
              v[i].w &= ~__vcmpeq4(v[i].w & 0x7f7f7f7fu, 0x7f7f7f7fu);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
          const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
          uint32_t x[8];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            x[2 * k] = e4m3_to_f16((uint16_t)w[k]), x[2 * k + 1] = e4m3_to_f16((uint16_t)(w[k] >> 16));
          put(to + W::kOperand, i0 + i, make_uint4(x[0], x[1], x[2], x[3]), make_uint4(x[4], x[5], x[6], x[7]));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) arrive(v_full + buf), arrive(raw_empty + raw);
      if (++raw == W::kRaw) raw = 0, raw_phase ^= 1;
      if (++buf == W::kBufs) buf = 0, phase ^= 1;
      if (todo > 1) advance(a, now);
    }
  } else {
    // ------------------------------------------------------------------------------------------------ softmax
    if constexpr (QT == 2) regs_increase<W::kSoftmaxRegs>();
    const int t = warp / 4;
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;   // of TMEM
    const uint32_t s_tiles = tmem + lanes + W::kS + t * 2 * kTileKeys, o_at = tmem + lanes + W::kO + t * D;
    const bool mask_vectors = a.T % 16 == 0 && (reinterpret_cast<uintptr_t>(a.mask) & 15) == 0 && a.mask_i % 16 == 0 &&
                              a.mask_b % 16 == 0;
    int buf = 0, segment = 0;
    uint32_t phase = 0, s_phase = 0, o_phase = 0;   // s_phase: a bit per score tile
    uint32_t pv_phase = 1;                          // of the row tile's last product
    while (todo > 0) {
      // ---- a row tile, or this CTA's part of it: key tiles first_tile ... last - 1
      const int first_tile = now.tile, last = (int)min((int64_t)now.tiles, now.tile + todo);
      const bool act = active(now, t);
      const int row = now.unit % a.row_tiles * W::kRows + t * 128 + warp % 4 * 32 + lane, token = row / a.group;
      const int head = now.unit / a.row_tiles * a.group + row % a.group;
      const bool warp_live = act && row - lane < now.fresh * a.group, live = token < now.fresh;
      Softmax sm;
      sm.clear();
      float row_scale = 1.0f;
      if (act) {
        if (warp_live) {
          if constexpr (D == 128) {
            // 16 lanes a row, two rows at a time: whole lines (a row a lane touches each line eight times over).  Not taken
            // for D 64 and 256, whose rows go to TMEM, where a lane holds its own row, nor for D 96, whose 12 chunks do not
            // divide a warp: they load a row a lane.
            const int tile_row = now.unit % a.row_tiles * W::kRows + t * 128, base = warp % 4 * 32 + lane / 16, ch = lane % 16;
            int tok = (tile_row + base) / a.group, in_group = (tile_row + base) - tok * a.group;
            const T* heads = static_cast<const T*>(a.q) + now.b * a.q_st.b + (int64_t)(now.unit / a.row_tiles) * a.group * a.q_st.h;
            // a small loop with the next rows under way: unrolled, fetching the code would take longer than the rows
            uint4 v[4];
            auto fetch = [&] {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                v[i] = tok < now.fresh ? *reinterpret_cast<const uint4*>(heads + tok * a.q_st.s + in_group * a.q_st.h + ch * 8)
                                       : make_uint4(0, 0, 0, 0);
                in_group += 2;
                if (in_group >= a.group) in_group -= a.group, ++tok;
                if (in_group >= a.group) in_group -= a.group, ++tok;
              }
            };
            fetch();
#pragma unroll 1
            for (int i0 = 0; i0 < 16; i0 += 4) {
              uint4 w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = v[i];
              if (i0 < 12) fetch();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r128 = base + 2 * (i0 + i);
                if constexpr (!std::is_same<T, __half>::value) {
                  uint32_t top = __vmaxu2(__vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu),
                                          __vmaxu2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
#pragma unroll
                  for (int o = 1; o < 16; o *= 2) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
                  top = max(top & 0xffffu, top >> 16);
                  const int e = row_exponent(top);
                  const float inverse = __int_as_float((254 - e) << 23);
                  if (ch == 0) q_scale[t][r128] = __int_as_float(e << 23);
                  float x[8];
                  unpack8(w[i], x, T());
                  w[i] = make_uint4(pack2(x[0] * inverse, x[1] * inverse, __half()), pack2(x[2] * inverse, x[3] * inverse, __half()),
                                    pack2(x[4] * inverse, x[5] * inverse, __half()), pack2(x[6] * inverse, x[7] * inverse, __half()));
                }
                *reinterpret_cast<uint4*>(queries + t * W::kQTile + ch / 8 * W::kQPanel + r128 * 128 +
                                          (((ch % 8) ^ (r128 & 7)) << 4)) = w[i];
              }
            }
            __syncwarp();
            if constexpr (!std::is_same<T, __half>::value) row_scale = q_scale[t][warp % 4 * 32 + lane];
          } else {
            // the row in fp16, scaled by a power of two of its largest value, as D / 2 TMEM columns
            const T* src = static_cast<const T*>(a.q) + now.b * a.q_st.b + token * a.q_st.s + head * a.q_st.h;
            constexpr int kPart = D == 256 ? 128 : D;   // channels held in registers at once
            uint4 v[kPart / 8];
            auto fetch = [&](int c0) {
#pragma unroll
              for (int i = 0; i < kPart / 8; ++i)
                v[i] = live ? *reinterpret_cast<const uint4*>(src + c0 + 8 * i) : make_uint4(0, 0, 0, 0);
            };
            fetch(0);
            float inverse = 1.0f;
            if constexpr (!std::is_same<T, __half>::value) {
              uint32_t top = 0;
#pragma unroll
              for (int c0 = D - kPart; c0 >= 0; c0 -= kPart) {
                if (D > kPart) fetch(c0);
#pragma unroll
                for (int i = 0; i < kPart / 8; ++i)
                  top = __vmaxu2(top, __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu),
                                               __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu)));
              }
              top = max(top & 0xffffu, top >> 16);
              const int e = row_exponent(top);
              row_scale = __int_as_float(e << 23);
              inverse = __int_as_float((254 - e) << 23);
            }
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += kPart) {
              if (c0 > 0) fetch(c0);
#pragma unroll
              for (int i = 0; i < kPart / 32; ++i) {   // 32 channels: 16 columns
                uint32_t w[16];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const uint4 y = v[4 * i + k];
                  if constexpr (std::is_same<T, __half>::value) {
                    w[4 * k] = y.x, w[4 * k + 1] = y.y, w[4 * k + 2] = y.z, w[4 * k + 3] = y.w;
                  } else {
                    float x[8];
                    unpack8(y, x, T());
#pragma unroll
                    for (int z = 0; z < 4; ++z) w[4 * k + z] = pack2(x[2 * z] * inverse, x[2 * z + 1] * inverse, __half());
                  }
                }
                if constexpr (W::kQShared) {
                  const int r128 = warp % 4 * 32 + lane;
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const int ch = (c0 + 32 * i) / 8 + k;
                    *reinterpret_cast<uint4*>(queries + t * W::kQTile + ch / 8 * W::kQPanel + r128 * 128 +
                                              (((ch % 8) ^ (r128 & 7)) << 4)) =
                        make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                  }
                } else {
                  tmem_st16(tmem + lanes + W::kQ + t * (D / 2) + c0 / 2 + i * 16, w);
                }
              }
            }
          }
          if constexpr (W::kQShared) {
            fence_proxy_async_smem();
          } else {
            tmem_wait_st();
            tc_fence_before();
          }
        }
        __syncwarp();
        if (lane == 0) arrive(q_full + t);
      }
#pragma unroll 1
      for (int tile = first_tile; tile < last; ++tile) {
        if (act) {
          const int si = (tile - first_tile) & 1;
          const uint32_t s_at = s_tiles + si * kTileKeys;
          wait_stage(s_full[t] + si, s_phase >> si & 1, &given_up, a.p.status);
          s_phase ^= 1u << si;
          if (warp_live) {
            wait_stage(k_full + buf, phase, &given_up, a.p.status);   // long there: orders the reads of params
            tc_fence_after();
            const float* factor = params + buf * W::kParams;
            const int key0 = tile * kTileKeys;
            const bool drafts = key0 + kTileKeys > now.len;
            uint32_t packed[32];
            bool again = true;
            // Most tiles: every row sees every key and no reference moves.  The weights are computed on that assumption in
            // one straight run and looked over afterwards; where it did not hold the scores are still in TMEM, and the tile
            // is done over.  (What a key needs is read by every lane of eight warps, and the words returned are what shared
            // memory is busy with: two a key here, not three.)
            if (tile != first_tile && !drafts) {
              const uint64_t scale2 = f2_pack(row_scale, row_scale), minus_t = f2_pack(-sm.t, -sm.t);
              uint64_t sum[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
              float top[2] = {0.0f, 0.0f};
#pragma unroll
              for (int part = 0; part < 2; ++part) {
                uint32_t r[32];
                tmem_ld32(s_at + 32 * part, r);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const int k = 32 * part + 4 * i;
                  const float4 f = *reinterpret_cast<const float4*>(factor + k);
                  const float4 w = *reinterpret_cast<const float4*>(factor + kTileKeys + k);
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const int c = 4 * i + 2 * h;
                    const uint64_t score = f2_pack(__uint_as_float(r[c]), __uint_as_float(r[c + 1]));
                    const uint64_t by = h ? f2_pack(f.z, f.w) : f2_pack(f.x, f.y);
                    float p, q;
                    // the factor of the key first: a row's scale may be as large as 2^126
                    if constexpr (std::is_same<T, __half>::value)
                      f2_unpack(f2_fma(score, by, minus_t), p, q);
                    else
                      f2_unpack(f2_fma(f2_mul(score, by), scale2, minus_t), p, q);
                    const uint64_t u = f2_pack(fast_exp2(p), fast_exp2(q));
                    sum[h] = f2_add(u, sum[h]);
                    f2_unpack(f2_mul(u, h ? f2_pack(w.z, w.w) : f2_pack(w.x, w.y)), p, q);
                    top[h] = fmaxf(fmaxf(top[h], p), q);
                    packed[16 * part + c / 2] = pack_weights(p, q);
                  }
                }
              }
              float p, q;
              f2_unpack(f2_add(sum[0], sum[1]), p, q);
              p = (p + q) * sm.ratio();
              again = __any_sync(0xffffffffu, !(fmaxf(top[0], top[1]) <= kMostWeight) || bits(p) > bits(kTileKeys * kMostSum));
              if (!again) sm.l += p;
            }
            if (!again) {
              tmem_st32(s_at, packed);
            } else {
              // which keys the row sees: bit j is key key0 + j (what is behind the last key has a factor that hides it)
              uint64_t seen = ~uint64_t(0);
              if (drafts) {
                const int t0 = key0 - now.len;   // number of the first key as a draft
                seen = t0 >= 0 ? 0 : (uint64_t(1) << -t0) - 1;
                if (live) {
                  const int from = max(t0, 0);
                  if (a.mask != nullptr) {
                    const uint8_t* mask = a.mask + now.b * a.mask_b + token * a.mask_i;
                    const int to = min(t0 + kTileKeys, now.fresh);
                    if (mask_vectors) {   // rows of whole 16-byte vectors
#pragma unroll 5
                      for (int d = from & ~15; d < to; d += 16) {
                        const uint4 v = *reinterpret_cast<const uint4*>(mask + d);
                        const uint64_t bits = nonzero_bytes(v.x) | nonzero_bytes(v.y) << 4 | nonzero_bytes(v.z) << 8 |
                                              nonzero_bytes(v.w) << 12;
                        seen |= d >= t0 ? bits << (d - t0) : bits >> (t0 - d);
                      }
                    } else {
#pragma unroll 8
                      for (int d = from; d < to; ++d) seen |= (uint64_t)(mask[d] != 0) << (d - t0);
                    }
                    if (now.fresh - t0 < kTileKeys) seen &= (uint64_t(1) << (now.fresh - t0)) - 1;
                  } else if (token >= from) {
                    const int count = min(token - t0 + 1, kTileKeys);
                    seen |= count == kTileKeys ? ~uint64_t(0) : (uint64_t(1) << count) - 1;
                  }
                }
              }
              // 16 keys at a time, once for the references and once for the weights; one small loop on purpose: this code runs
              // once or twice a row tile, and what it costs is fetching it
              float most = -INFINITY, most_t = -INFINITY, m = 0.0f, unit = 0.0f;
              uint64_t sum = f2_pack(0.0f, 0.0f);
#pragma unroll 1
              for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
                for (int k = 0; k < kTileKeys / 16; ++k) {
                  const float* by = factor + 16 * k;
                  float x[16];
                  uint32_t r[16];
                  tmem_ld16(s_at + 16 * k, r);
                  tmem_wait_ld();
                  const uint32_t see = (uint32_t)(seen >> (16 * k));
#pragma unroll
                  for (int i = 0; i < 16; i += 2) {
                    const float2 f = *reinterpret_cast<const float2*>(by + i);
                    uint64_t v = f2_mul(f2_pack(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2_pack(f.x, f.y));
                    if constexpr (!std::is_same<T, __half>::value) v = f2_mul(v, f2_pack(row_scale, row_scale));
                    f2_unpack(v, x[i], x[i + 1]);
                    if (!(see >> i & 1)) x[i] = -INFINITY;
                    if (!(see >> (i + 1) & 1)) x[i + 1] = -INFINITY;
                  }
                  if (pass == 0) {
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                      const float2 log_v = *reinterpret_cast<const float2*>(by + 2 * kTileKeys + i);
                      float p, q;
                      f2_unpack(f2_add(f2_pack(x[i], x[i + 1]), f2_pack(log_v.x, log_v.y)), p, q);
                      most = fmaxf(fmaxf(most, x[i]), x[i + 1]);
                      most_t = fmaxf(fmaxf(most_t, p), q);
                    }
                  } else {
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                      const float2 vs = *reinterpret_cast<const float2*>(by + kTileKeys + i);
                      const uint64_t u = f2_pack(fast_exp2(x[i] - m), fast_exp2(x[i + 1] - m));
                      sum = f2_add(sum, u);
                      float p, q;
                      f2_unpack(f2_mul(f2_mul(u, f2_pack(vs.x, vs.y)), f2_pack(unit, unit)), p, q);
                      // the scale of a key not seen may be anything
                      w[i / 2] = pack_weights(x[i] == -INFINITY ? 0.0f : p, x[i + 1] == -INFINITY ? 0.0f : q);
                    }
                    tmem_st8(s_at + 8 * k, w);   // over 8 columns of scores, all read by then
                  }
                }
                if (pass > 0) break;
                const bool moves = sm.exceeded(most, most_t);
                if (__any_sync(0xffffffffu, moves)) {
                  float keep = 1.0f;
                  if (moves) keep = sm.move(most, most_t);
                  if (tile != first_tile) {   // the first product of a row tile overwrites O
                    // the products of the tile before must be done (older ones are: this tile's scores came after them)
                    wait_stage(pv_done + t, pv_phase, &given_up, a.p.status);
                    tc_fence_after();
#pragma unroll 1
                    for (int i = 0; i < D / 16; ++i) {
                      uint32_t r[16];
                      tmem_ld16(o_at + 16 * i, r);
                      tmem_wait_ld();
#pragma unroll
                      for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * keep);
                      tmem_st16(o_at + 16 * i, r);
                    }
                  }
                }
                m = sm.m(), unit = sm.score_unit();
              }
              float p, q;
              f2_unpack(sum, p, q);
              sm.l += p + q;
            }
            tmem_wait_st();
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0) arrive(p_full[t] + si);
          pv_phase ^= 1;
        }
        if (++buf == W::kBufs) buf = 0, phase ^= 1;
      }
      // ---- its end
      const bool whole = last == now.tiles && first_tile == 0, mine = row < a.T * a.group;
      if (act) {
        wait_stage(o_full + t, o_phase, &given_up, a.p.status);
        o_phase ^= 1;
        tc_fence_after();
      }
      T* dst = static_cast<T*>(a.out) + now.b * a.out_st.b + token * a.out_st.s + head * a.out_st.h;
      // partial rows: four channels of all rows, then the next four, so that the lanes' stores are whole lines
      const int64_t first_row = (2 * (int64_t)blockIdx.x + (segment > 0)) * W::kRows;
      const int in_tile = t * 128 + warp % 4 * 32 + lane;
      float* part = a.part_o + first_row * D + in_tile * 4;
      const float inverse = sm.l == 0.0f ? 0.0f : 1.0f / sm.l;
      if (warp_live) {
#pragma unroll 1
        for (int i = 0; i < D / 32; ++i) {
          uint32_t r[32];
          tmem_ld32(o_at + 32 * i, r);
          tmem_wait_ld();
          if (mine && whole) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              float x[8];
#pragma unroll
              for (int z = 0; z < 8; ++z) x[z] = live && sm.l != 0.0f ? __uint_as_float(r[k + z]) * inverse * sm.v_unit() : 0.0f;
              store8(dst + 32 * i + k, x);
            }
          } else if (mine && live) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<uint4*>(part + (32 * i + k) * W::kRows) = make_uint4(r[k], r[k + 1], r[k + 2], r[k + 3]);
          }
        }
        tc_fence_before();
      } else if (mine && whole) {
        for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint4*>(dst + 8 * i) = make_uint4(0, 0, 0, 0);
      }
      if (mine && whole) {
        if (a.lse != nullptr)
          a.lse[((int64_t)now.b * a.H + head) * a.T + token] =
              !live || sm.l == 0.0f ? -INFINITY : (sm.m() + log2f(sm.l)) * 0.69314718055994531f;
      } else if (mine && live) {
        a.part_state[first_row + in_tile] = sm.state();
      }
      ++segment;
      todo -= last - first_tile;
      now.tile = last - 1;
      if (todo > 0) advance(a, now);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

int wide_ctas() { return sm_count(); }
int wide_rows(int D) { return D == 256 ? 128 : 256; }

template <typename T, int D>
static int launch_wide(const PagedAttnArgs& a, cudaStream_t st) {
  using W = Wide<D>;
  CUtensorMap k_map, v_map;
  const uint64_t rows = (uint64_t)a.p.num_pages * a.p.Hkv << a.p.page_shift;
  if (!code_map<D>(&k_map, a.p.k8, rows, 1 << a.p.page_shift) || !code_map<D>(&v_map, a.p.v8, rows, 1 << a.p.page_shift))
    return SAGE_ERR_LAUNCH;
  static std::atomic<uint64_t> prepared{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(prepared.load() >> dev & 1))) {
    // setmaxnreg moves registers inside what the CTA was launched with: a build with fewer would wait forever
    cudaFuncAttributes fa{};
    e = cudaFuncGetAttributes(&fa, paged_wide_kernel<T, D>);
    if (e == cudaSuccess && W::QT == 2 && fa.numRegs != W::kLaunchRegs) {
      set_error("paged attention built with %d registers per thread; its setmaxnreg split needs %d", fa.numRegs,
                W::kLaunchRegs);
      return SAGE_ERR_LAUNCH;
    }
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(paged_wide_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, W::kSmem);
    if (e == cudaSuccess && dev < 64) prepared.fetch_or(uint64_t(1) << dev);
  }
  if (e == cudaSuccess) {
    e = launch_early(paged_wide_kernel<T, D>, dim3(a.ctas), W::kThreads, W::kSmem, st, a, k_map, v_map);
  }
  if (e == cudaSuccess) return SAGE_OK;
  set_error("paged attention: %s", cudaGetErrorString(e));
  return SAGE_ERR_LAUNCH;
}

int launch_paged_wide(const PagedAttnArgs& a, int dtype, cudaStream_t st) {
  return by_head_dim(a.p.D, [&](auto d) {
    constexpr int kD = decltype(d)::value;
    return dtype == SAGE_BF16 ? launch_wide<__nv_bfloat16, kD>(a, st) : launch_wide<__half, kD>(a, st);
  });
}

}  // namespace sage
