// Attention over the paged K/V cache for the tokens of one step: single tokens, a run of tokens, or a tree of drafts.
//
// Row (b, i, h) sees the keys j < lens[b] and the drafted keys lens[b] + t with t <= i (no mask) or mask[b, i, t]:
//   s_j = sm_scale * ks_j * (q . k8_j),   p_j = exp(s_j - m),   o = sum_j p_j vs_j v8_j / sum_j p_j
//
// One pass over the keys with two running references, of the scores and of the scores with the V scale in them:
//   x_j = log2(e) s_j,               m ~ max x_j,    l = sum 2^(x_j - m)
//   t_j = x_j + log2(vs_j),      m' ~ max t_j - 8,   p'_j = 2^(t_j - m'),   O = sum p'_j v8_j
//   o = 2^(m' - m) O / l,   lse = ln 2 (m + log2 l)
// The products with V take weights p' in fp16, which are placed high in its range, the row's largest (with its scale) at 2^7
// to 2^15: p' keeps 11 bits down to 2^-21 of that one, and below it is off by 2^-32 of it (with the largest at 1, 2^-14 and
// 2^-25: hundreds of thousands of keys at 2^-24 of a dominating one came out 1 % off).  l knows nothing of V: a scale of
// 2^-109 or 2^119, the ends of what append writes, takes nothing from it, and a NaN row of V leaves the log-sum-exp as it is.
// One exponential serves both: p'_j = 2^(x_j - m') vs_j and l in units of 2^m' with one factor 2^(m' - m) a group; where that
// may leave the range of fp32 (V scales above 2^72) p'_j = 2^(x_j - m) vs_j 2^(m - m'), in this order, in the code for rare groups.
// m and m' are whole numbers, so the factors and all rescaling are exact powers of two; log2 vs serves only to place m'.  They
// move, both, when a score exceeds m by more than 8, as in the dense kernel, or a weight 2^15, and O is rescaled then.
// Both products run on fp16 operands with fp32 accumulators: int8 and e4m3 codes are exact in fp16, bf16 queries are
// scaled by a power of two of their row (what is below 2^-24 of the row's largest value is rounded).  The references
// and l are fp32.  The tensor cores cut O towards zero at its last place every four keys: up to 2^-25 of it a key of the warp.
//
// The query rows of a kv head (T tokens of H / Hkv heads) are cut into row tiles, the keys into tiles of 64.  All
// (sequence, kv head, row tile, key tile) of a call form one list that the CTAs share evenly, whatever the lengths are: a
// CTA walks a contiguous stretch of it with one load pipeline (a producer warp that issues TMA boxes and prefetches page
// numbers, and consumer warps that wait for nothing but their stage).  A row tile that falls to several CTAs is joined
// from their partial (O, l, m') by a second small kernel, in the order of the keys.
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T: keys and channels fill the 16 rows of an mma tile
// and the query rows its 8 columns, so that the 1 to 8 rows of a single token's group cost one column tile.
//
// Bound by memory: one token (4 query rows a kv head) over 16 sequences of 16 to 32 thousand keys, 8 kv heads, D 128, takes
// 149 to 157 us on B200 (by the GPU), 85 to 89 % of the measured copy rate; issue slots are 58 % taken.  D 64, 96 and 256
// reach 72, 84 and 91 %.  Steps on the way, us: one CTA a row 11122; shared list, rows times keys, cp.async 257; transposed
// products, TMA 175; no logarithm and no comparison a key where no maximum moves 156; warps joining all at once 147; two
// references 149.  One token over 1024 keys takes 11.3 us with the join, most of it start-up and dependent loads.  With more
// than 16 rows (D 256: 8) each key is converted twice, since more column tiles a warp do not fit the registers: 8 drafts of 8
// sequences over 8190 keys, D 128, take 55 us, 29 % of the rate.
#include "sage_paged_attn.cuh"

namespace sage {

constexpr int kWarps = 4;                              // consumer warps
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kJoinThreads = 128;

// What the join of a CTA's warps needs of a query row: the factor of each warp's O, 1 / l and 2^(m' - m).
struct alignas(16) JoinRow {
  float factor[4];
  float inverse, unit;
};

template <int D, int NR, int WM>
struct Config {
  // CTAs of an SM: as the registers of a thread allow (96 for four CTAs, 128 for three, 168 for two)
  static constexpr int kCtas = NR == 1 && D <= 128 ? 4 : D == 64 ? 3 : 2;
  static constexpr int kRows = 8 * NR * WM;               // of a row tile
  static constexpr int kPerStage = Tile<D>::kStage + 2 * kTileKeys * 4 + 16;
  static constexpr int kFit = (232448 / kCtas - 2048 - 1024) / kPerStage;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kSmem = 1024 + kStages * kPerStage;
  static_assert(kStages >= 2, "two stages at the least");
};

// The rows of a kv head are one row tile of 8 NR WM rows: WM groups of 4 / WM warps that share its keys, NR column tiles of 8
// rows a warp.
template <typename T, int D, int NR, int WM>
__global__ void __launch_bounds__(kThreads, Config<D, NR, WM>::kCtas)
    paged_attn_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map) {
  using C = Config<D, NR, WM>;
  using S = Tile<D>;
  constexpr int WK = kWarps / WM, NS = D / 16, NT = D / 16, kStages = C::kStages;
  extern __shared__ unsigned char smem_raw[];
  __shared__ int64_t warp_sums[kThreads / 32], found[2];
  __shared__ RowState join_state[kWarps][8 * NR];
  __shared__ JoinRow join_row[C::kRows];
  __shared__ int given_up;
  unsigned char* stages = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float* scales = reinterpret_cast<float*>(stages + kStages * S::kStage);               // [stage][ks, vs][64]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + kStages * 2 * kTileKeys);
  uint64_t* empty = full + kStages;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    given_up = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, kWarps);
    }
    fence_barrier_init();
  }
  // Nothing of the stream's earlier work is read before it is done; only then may the join start, which reads the lengths
  // before it waits for this kernel.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  Cursor now;
  int64_t todo = locate<kThreads>(a, warp_sums, found, now);
  if (todo == 0) return;
  int slot = 0;
  uint32_t phase = 0;

  if (warp == kWarps) {
    load_tiles<D>(a, &k_map, &v_map, now, todo, stages, scales, full, empty, kStages, &given_up);
    return;
  }

  // -------------------------------------------------------------------- consumers
  const int n = lane / 4, c = lane % 4, wm = warp % WM, wk = warp / WM;
  uint32_t qf[NR][NS][2];
  float o[NR][NT][4];
  Softmax sm[NR][2];
  bool fresh_unit = true;
  int segment = 0;                    // row tiles that this CTA has finished
  int first_tile = now.tile;          // of the row tile, by this CTA
  const int row0 = wm * 8 * NR;       // first query row of this warp
  int head0 = 0;                      // first query head of the kv head
  for (; todo > 0; --todo) {
    if (fresh_unit) {
      head0 = now.unit * a.group;
      fresh_unit = false;
      first_tile = now.tile;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int t = 0; t < NT; ++t) o[r][t][0] = o[r][t][1] = o[r][t][2] = o[r][t][3] = 0.0f;
        sm[r][0].clear(), sm[r][1].clear();
        const int row = row0 + 8 * r + n, token = row / a.group;
        const bool live = token < now.fresh;
        const T* src = static_cast<const T*>(a.q) + now.b * a.q_st.b + token * a.q_st.s + (head0 + row % a.group) * a.q_st.h;
        // channels of step s: four consecutive ones, as a word of four codes holds them
        uint2 w[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const int d = D % 64 == 0 ? (c + 4 * (s / 4)) * 16 + s % 4 * 4 : (c + 4 * (s / 2)) * 8 + s % 2 * 4;
          w[s] = live ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0, 0);
        }
        if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
          for (int s = 0; s < NS; ++s) qf[r][s][0] = w[s].x, qf[r][s][1] = w[s].y;
        } else {
          uint32_t top = 0;
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, (e < 2 ? w[s].x : w[s].y) >> (16 * (e & 1)) & 0x7fffu);
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = row_exponent(top);
          const float inverse = __int_as_float((254 - e) << 23);
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            qf[r][s][0] = pack2(__uint_as_float(w[s].x << 16) * inverse, __uint_as_float(w[s].x & 0xffff0000u) * inverse,
                                __half());
            qf[r][s][1] = pack2(__uint_as_float(w[s].y << 16) * inverse, __uint_as_float(w[s].y & 0xffff0000u) * inverse,
                                __half());
          }
          sm[r][0].set_row_exponent(__shfl_sync(0xffffffffu, e, 8 * c));
          sm[r][1].set_row_exponent(__shfl_sync(0xffffffffu, e, 8 * c + 4));
        }
      }
    }

    wait_stage(full + slot, phase, &given_up, a.p.status);   // after a timeout the rest runs through on what is there
    const unsigned char* kt = stages + slot * S::kStage;
    unsigned char* vt = stages + slot * S::kStage + S::kBytes;
    const float* ks = scales + slot * 2 * kTileKeys;
    const int key0 = now.tile * kTileKeys, total = now.len + now.fresh;

#pragma unroll 1
    for (int g = wk * 16; g < kTileKeys; g += WK * 16) {
      const bool drafts = key0 + g + 16 > now.len;   // the group holds keys that some rows do not see
      if (drafts) {
        // codes behind the last key are anything, and a NaN code of a draft that its reader does not see must not reach
        // it through 0 * NaN: both are cleared (by each warp that reads the group)
        for (int i = lane; i < D; i += 32) {
          const int row = g + i % 16;
          uint4* at = reinterpret_cast<uint4*>(vt + S::at(row, i / 16 * 16));
          if (key0 + row >= total) {
            *at = make_uint4(0, 0, 0, 0);
          } else if (key0 + row >= now.len) {
            uint4 v = *at;
            v.x &= ~__vcmpeq4(v.x & 0x7f7f7f7fu, 0x7f7f7f7fu);
            v.y &= ~__vcmpeq4(v.y & 0x7f7f7f7fu, 0x7f7f7f7fu);
            v.z &= ~__vcmpeq4(v.z & 0x7f7f7f7fu, 0x7f7f7f7fu);
            v.w &= ~__vcmpeq4(v.w & 0x7f7f7f7fu, 0x7f7f7f7fu);
            *at = v;
          }
        }
        fence_proxy_async_smem();   // before the stage's next load
        __syncwarp();
      }
      float s[NR][4] = {};          // [2 h + e]: key in slot n + 8 h, row 2c + e of the column tile
      const int keys[2] = {g + S::slot_key(n), g + S::slot_key(n + 8)};
      auto step = [&](int i, uint32_t w0, uint32_t w1) {
        uint32_t x[4];
        int8_to_f16(w0, x[0], x[2]);
        int8_to_f16(w1, x[1], x[3]);
#pragma unroll
        for (int r = 0; r < NR; ++r) mma_f16(s[r], x, qf[r][i][0], qf[r][i][1]);
      };
      if constexpr (D % 64 == 0) {
#pragma unroll
        for (int i = 0; i < NS / 4; ++i) {
          const uint4 u = *reinterpret_cast<const uint4*>(kt + S::at(keys[0], (c + 4 * i) * 16));
          const uint4 v = *reinterpret_cast<const uint4*>(kt + S::at(keys[1], (c + 4 * i) * 16));
          step(4 * i, u.x, v.x), step(4 * i + 1, u.y, v.y), step(4 * i + 2, u.z, v.z), step(4 * i + 3, u.w, v.w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) {
          const uint2 u = *reinterpret_cast<const uint2*>(kt + S::at(keys[0], (c + 4 * i) * 8));
          const uint2 v = *reinterpret_cast<const uint2*>(kt + S::at(keys[1], (c + 4 * i) * 8));
          step(2 * i, u.x, v.x), step(2 * i + 1, u.y, v.y);
        }
      }
      // Most groups: every row sees every key and no reference moves.  The weights are computed on that assumption and
      // looked over afterwards; where it did not hold the group is done over from its scores.
      const float factor[2] = {ks[keys[0]] * a.scale, ks[keys[1]] * a.scale};
      const float v_scale[2] = {ks[kTileKeys + keys[0]], ks[kTileKeys + keys[1]]};
      uint32_t pf[NR][2];
      bool again = true;
      // x - t of the lane's two rows.  The factor of the key comes first: a row's scale may be as large as 2^126.
      auto less = [&](int r, uint64_t score, uint64_t by, uint64_t minus_t) {
        if constexpr (std::is_same<T, __half>::value)
          return f2_fma(score, by, minus_t);
        else
          return f2_fma(f2_mul(score, by), f2_pack(sm[r][0].row_scale(), sm[r][1].row_scale()), minus_t);
      };
      if (!drafts) {
        uint64_t l[NR];   // the lane's two rows as a pair
        float top = 0.0f;
        uint32_t most = 0;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const uint64_t minus_t = f2_pack(-sm[r][0].t, -sm[r][1].t);
          float x, y;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            f2_unpack(less(r, f2_pack(s[r][2 * h], s[r][2 * h + 1]), f2_pack(factor[h], factor[h]), minus_t), x, y);
            const uint64_t u = f2_pack(fast_exp2(x), fast_exp2(y));
            l[r] = h == 0 ? u : f2_add(l[r], u);
            f2_unpack(f2_mul(u, f2_pack(v_scale[h], v_scale[h])), x, y);
            top = fmaxf(fmaxf(top, x), y);
            pf[r][h] = pack_weights(x, y);
          }
          l[r] = f2_mul(l[r], f2_pack(sm[r][0].ratio(), sm[r][1].ratio()));
          f2_unpack(l[r], x, y);
          most = max(max(most, bits(x)), bits(y));
        }
        again = __any_sync(0xffffffffu, !(top <= kMostWeight) || most > bits(2 * kMostSum));
        if (!again) {
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            f2_unpack(f2_add(f2_pack(sm[r][0].l, sm[r][1].l), l[r]), sm[r][0].l, sm[r][1].l);
            pf[r][0] = transposed(pf[r][0]), pf[r][1] = transposed(pf[r][1]);
          }
        }
      }
      if (again) {
        const float log_v[2] = {__log2f(v_scale[0]), __log2f(v_scale[1])};   // of a zero row -infinity
        // what the lane's rows do not see, bit 4 r + 2 e + h; a loop, since fetching this code is what it costs
        uint32_t hidden = 0;
        if (drafts) {
#pragma unroll 1
          for (int i = 0; i < 4 * NR; ++i) {
            const int row = row0 + 8 * (i / 4) + 2 * c + i / 2 % 2, key = g + S::slot_key(n + i % 2 * 8);
            const int t = key0 + key - now.len;   // number of the key as a draft
            const bool seen = t < 0 || (t < now.fresh && row < now.fresh * a.group &&
                                        (a.mask != nullptr ? a.mask[now.b * a.mask_b + row / a.group * a.mask_i + t] != 0
                                                           : t * a.group <= row));
            hidden |= (uint32_t)!seen << i;
          }
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float keep[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float& x = s[r][2 * h + e];
              x *= factor[h];
              if constexpr (!std::is_same<T, __half>::value) x *= sm[r][e].row_scale();
              if (hidden >> (4 * r + 2 * e + h) & 1) x = -INFINITY;
            }
            float top = fmaxf(s[r][e], s[r][2 + e]), top_v = fmaxf(s[r][e] + log_v[0], s[r][2 + e] + log_v[1]);
#pragma unroll
            for (int z = 4; z < 32; z *= 2) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, z));
              top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, z));
            }
            keep[e] = sm[r][e].move(top, top_v);   // by less than they wait for too: here it costs nothing
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) o[r][t][0] *= keep[0], o[r][t][1] *= keep[1], o[r][t][2] *= keep[0], o[r][t][3] *= keep[1];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float p[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = s[r][2 * h + e], u = fast_exp2(x - sm[r][e].m());
              sm[r][e].l += u;
              p[e] = x == -INFINITY ? 0.0f : u * v_scale[h] * sm[r][e].score_unit();   // an unseen key's scale may be anything
            }
            pf[r][h] = transposed(pack_weights(p[0], p[1]));
          }
        }
      }
      // four keys a lane; a word of four channels of each is two output tiles
      auto product = [&](int i, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t u = __byte_perm(w0, w1, x ? 0x7362 : 0x5140), v = __byte_perm(w2, w3, x ? 0x7362 : 0x5140);
          const uint32_t f[4] = {e4m3_to_f16((uint16_t)u), e4m3_to_f16((uint16_t)(u >> 16)), e4m3_to_f16((uint16_t)v),
                                 e4m3_to_f16((uint16_t)(v >> 16))};
#pragma unroll
          for (int r = 0; r < NR; ++r) mma_f16(o[r][2 * i + x], f, pf[r][0], pf[r][1]);
        }
      };
      int vkeys[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) vkeys[k] = g + S::slot_key(2 * c + k % 2 + k / 2 * 8);
      if constexpr (S::kWide) {
#pragma unroll
        for (int i = 0; i < S::kHalves; ++i) {
          uint4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = *reinterpret_cast<const uint4*>(vt + S::at(vkeys[k], i * 128 + S::first_channel(n)));
          product(4 * i, v[0].x, v[1].x, v[2].x, v[3].x), product(4 * i + 1, v[0].y, v[1].y, v[2].y, v[3].y);
          product(4 * i + 2, v[0].z, v[1].z, v[2].z, v[3].z), product(4 * i + 3, v[0].w, v[1].w, v[2].w, v[3].w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = *reinterpret_cast<const uint32_t*>(vt + S::at(vkeys[k], S::first_channel(n) + 4 * i));
          product(i, v[0], v[1], v[2], v[3]);
        }
      }
    }
    const bool last_tile = now.tile + 1 == now.tiles, ends = last_tile || todo == 1;
    if (!ends) {
      __syncwarp();
      if (lane == 0) arrive(empty + slot);
    }
    if (ends) {
      // the row tile ends here, or this CTA's part of it does
      const bool whole = last_tile && first_tile == 0;
      const int64_t part = (2 * (int64_t)blockIdx.x + (segment > 0)) * C::kRows;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sm[r][e].l += __shfl_xor_sync(0xffffffffu, sm[r][e].l, 4);
          sm[r][e].l += __shfl_xor_sync(0xffffffffu, sm[r][e].l, 8);
          sm[r][e].l += __shfl_xor_sync(0xffffffffu, sm[r][e].l, 16);
        }
      // The warps of a row tile join through the stage that all of them have read by then, eight rows of each at a time:
      // every warp leaves its part, every thread adds up eight channels of a row in the order of the warps.
      auto consumers_sync = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
      float* area = reinterpret_cast<float*>(stages + slot * S::kStage);   // [warp][8 rows][D]
      static_assert(kWarps * 8 * D * 4 <= S::kStage, "the parts must fit a stage");
      auto place = [](int row, int quad) {   // four channels; permuted against bank conflicts
        return (row * (D / 4) + (quad ^ (row >> 1 & 3) ^ (S::kWide ? (quad >> 4 & 1) << 2 : 0))) * 4;
      };
      // A barrier stands between each thing written here and its readers, and between those and the next row tile's writers,
      // whichever warp is ahead: states are read before the second barrier, the rows' factors are written after the first.
      if (n == 0) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) join_state[warp][8 * r + 2 * c + e] = sm[r][e].state();
      }
      consumers_sync();
      if (tid < C::kRows) {   // a thread a row: the warps' factors, the sum of the weights
        const int g = tid / (8 * NR);
        RowState all{kLowest, 0.0f, kLowest};
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const RowState& state = join_state[w * WM + g][tid % (8 * NR)];
          all.m = fmaxf(all.m, state.m), all.t = fmaxf(all.t, state.t);
        }
        JoinRow& to = join_row[tid];
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const RowState& state = join_state[w * WM + g][tid % (8 * NR)];
          all.l = fmaf(fast_exp2(state.m - all.m), state.l, all.l);
          to.factor[w] = fast_exp2(state.t - all.t);
        }
        if (tid < a.T * a.group) {
          const int token = tid / a.group, head = head0 + tid % a.group;
          const bool seen = token < now.fresh && all.l != 0.0f;
          to.inverse = seen ? 1.0f / all.l : 0.0f;
          to.unit = fast_exp2(all.t - all.m);
          if (!whole)
            a.part_state[part + tid] = all;
          else if (a.lse != nullptr)
            a.lse[((int64_t)now.b * a.H + head) * a.T + token] =
                seen ? (all.m + log2f(all.l)) * 0.69314718055994531f : -INFINITY;
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if (r > 0) consumers_sync();
#pragma unroll
        for (int t = 0; t < NT; t += 2)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float4*>(area + warp * (8 * D) + place(2 * c + e, S::channel(n, t, 0) / 4)) =
                make_float4(o[r][t][e], o[r][t][2 + e], o[r][t + 1][e], o[r][t + 1][2 + e]);
        consumers_sync();
#pragma unroll 1
        for (int item = tid; item < WM * D; item += 32 * kWarps) {
          const int of = item / (D / 8), g = of / 8, rr = of % 8, d = item % (D / 8) * 8;
          const int row = g * 8 * NR + 8 * r + rr;
          if (row >= a.T * a.group) continue;
          const JoinRow& by = join_row[row];
          float x[8] = {};
#pragma unroll
          for (int w = 0; w < WK; ++w) {
            const float f = by.factor[w];
            const float* from = area + (w * WM + g) * (8 * D);
            const float4 u = *reinterpret_cast<const float4*>(from + place(rr, d / 4));
            const float4 v = *reinterpret_cast<const float4*>(from + place(rr, d / 4 + 1));
            x[0] = fmaf(f, u.x, x[0]), x[1] = fmaf(f, u.y, x[1]), x[2] = fmaf(f, u.z, x[2]), x[3] = fmaf(f, u.w, x[3]);
            x[4] = fmaf(f, v.x, x[4]), x[5] = fmaf(f, v.y, x[5]), x[6] = fmaf(f, v.z, x[6]), x[7] = fmaf(f, v.w, x[7]);
          }
          if (whole) {
            const float inverse = by.inverse, unit = by.unit;
#pragma unroll
            for (int z = 0; z < 8; ++z) x[z] = inverse != 0.0f ? x[z] * inverse * unit : 0.0f;   // 0: sees nothing
            const int token = row / a.group, head = head0 + row % a.group;
            store8(static_cast<T*>(a.out) + now.b * a.out_st.b + token * a.out_st.s + head * a.out_st.h + d, x);
          } else {
            float* to = a.part_o + (part + row) * D + d;
            *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
          }
        }
      }
      fence_proxy_async_smem();   // before the stage's next load
      __syncwarp();
      if (lane == 0) arrive(empty + slot);
      ++segment;
      fresh_unit = true;
    }
    if (++slot == kStages) slot = 0, phase ^= 1;
    if (todo > 1) advance(a, now);
  }
}

// Which CTAs share row tile `unit` of sequence b, found by all threads of a join block: CTAs c0 .. c1, c0 with its partial
// slot `slot`, the others with slot 0.  Returns its key tiles.
__device__ __forceinline__ int sharing(const PagedAttnArgs& a, int b, int unit, int64_t* warp_sums, int& fresh, int& c0,
                                       int& c1, int& slot) {
  const int per = a.p.Hkv * a.row_tiles;
  int len;
  int64_t mine = 0, before = 0, list, start;
  for (int s = threadIdx.x; s < a.B; s += kJoinThreads) {
    const int t = sequence(a, s, len, fresh);
    mine += t;
    if (s < b) before += t;
  }
  {   // both sums over the block with one pair of barriers
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (threadIdx.x % 32 == 0) warp_sums[threadIdx.x / 32] = mine, warp_sums[kJoinThreads / 32 + threadIdx.x / 32] = before;
    __syncthreads();
    list = start = 0;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) list += warp_sums[w], start += warp_sums[kJoinThreads / 32 + w];
  }
  const int tiles = sequence(a, b, len, fresh);
  list *= per;
  start = start * per + (int64_t)unit * tiles;
  c0 = c1 = slot = 0;
  if (tiles > 0) {
    const int share = sharers(a, list);
    c0 = (int)(((start + 1) * share - 1) / list);
    c1 = (int)(((start + tiles) * share - 1) / list);
    slot = (int64_t)c0 * list / share < start ? 1 : 0;   // not the first row tile of CTA c0
  }
  return tiles;
}

// Joins the partial rows of the row tiles that fell to several CTAs, and writes the rows that see nothing at all; the CTAs
// of a row tile are joined in the order of its keys.  A warp takes a row.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads, 8) paged_join_kernel(const PagedAttnArgs a, int tile_rows, int blocks_per_unit) {
  __shared__ int64_t warp_sums[2 * kJoinThreads / 32];
  const int64_t id = blockIdx.x / blocks_per_unit;
  const int b = (int)(id / a.p.Hkv), unit = (int)(id - (int64_t)b * a.p.Hkv);   // a row tile holds all rows of a kv head
  int fresh, c0, c1, slot;
  const int tiles = sharing(a, b, unit, warp_sums, fresh, c0, c1, slot);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tiles > 0 && c0 == c1) return;   // the CTA wrote the rows itself
  const int lane = threadIdx.x % 32;
  const int row = blockIdx.x % blocks_per_unit * (kJoinThreads / 32) + threadIdx.x / 32;
  if (row >= a.T * a.group) return;
  const int token = row / a.group, head = unit * a.group + row % a.group;
  const bool live = tiles > 0 && token < fresh;
  float top = kLowest, top_t = kLowest, sum = 0.0f, o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = 0.0f;
  if (live) {
    for (int x = c0 + lane; x <= c1; x += 32) {
      const RowState state = a.part_state[(2 * (int64_t)x + (x == c0 ? slot : 0)) * tile_rows + row];
      top = fmaxf(top, state.m), top_t = fmaxf(top_t, state.t);
    }
#pragma unroll
    for (int x = 16; x > 0; x /= 2) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      top_t = fmaxf(top_t, __shfl_xor_sync(0xffffffffu, top_t, x));
    }
    constexpr int kAtOnce = 4;   // parts under way at once: the loads are what this kernel waits for
#pragma unroll 1
    for (int x0 = c0; x0 <= c1; x0 += kAtOnce) {
      RowState state[kAtOnce];
      float v[kAtOnce][D / 32];
#pragma unroll
      for (int z = 0; z < kAtOnce; ++z) {
        const int x = min(x0 + z, c1);   // the last one again, left out below
        const int64_t at = (2 * (int64_t)x + (x == c0 ? slot : 0)) * tile_rows + row;
        state[z] = a.part_state[at];
#pragma unroll
        for (int i = 0; i < D / 32; i += D % 64 ? 1 : 2) {
          if constexpr (D % 64 == 0) {
            const float2 w = *reinterpret_cast<const float2*>(a.part_o + at * D + i * 32 + lane * 2);
            v[z][i] = w.x, v[z][i + 1] = w.y;
          } else {
            v[z][i] = a.part_o[at * D + i * 32 + lane];
          }
        }
      }
#pragma unroll
      for (int z = 0; z < kAtOnce; ++z) {
        if (x0 + z > c1) break;
        const float f = fast_exp2(state[z].t - top_t);
        sum = fmaf(fast_exp2(state[z].m - top), state[z].l, sum);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = fmaf(f, v[z][i], o[i]);
      }
    }
  }
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum, unit_v = fast_exp2(top_t - top);
  T* dst = static_cast<T*>(a.out) + b * a.out_st.b + token * a.out_st.s + head * a.out_st.h;
#pragma unroll
  for (int i = 0; i < D / 32; i += D % 64 ? 1 : 2) {
    if constexpr (D % 64 == 0)
      *reinterpret_cast<uint32_t*>(dst + i * 32 + lane * 2) = pack2(o[i] * inverse * unit_v, o[i + 1] * inverse * unit_v, T());
    else
      dst[i * 32 + lane] = T(o[i] * inverse * unit_v);
  }
  if (a.lse != nullptr && lane == 0)
    a.lse[((int64_t)b * a.H + head) * a.T + token] =
        sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

// The same for the partial rows of the kernel for many rows (four channels of all rows, then the next four): a block takes
// 32 rows, a lane a row, a warp a quarter of its channels.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) wide_join_kernel(const PagedAttnArgs a, int tile_rows, int blocks_per_unit) {
  __shared__ int64_t warp_sums[2 * kJoinThreads / 32];
  const int64_t id = blockIdx.x / blocks_per_unit;
  const int per = a.p.Hkv * a.row_tiles, b = (int)(id / per), unit = (int)(id - (int64_t)b * per);
  int fresh, c0, c1, slot;
  const int tiles = sharing(a, b, unit, warp_sums, fresh, c0, c1, slot);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tiles > 0 && c0 == c1) return;   // the CTA wrote the rows itself
  constexpr int kChannels = D / 4;     // of a warp
  const int lane = threadIdx.x % 32, d0 = threadIdx.x / 32 * kChannels;
  const int row = blockIdx.x % blocks_per_unit * 32 + lane, r = unit % a.row_tiles * tile_rows + row;
  if (r >= a.T * a.group) return;
  const int token = r / a.group, head = unit / a.row_tiles * a.group + r % a.group;
  const bool live = tiles > 0 && token < fresh;
  float top = kLowest, top_t = kLowest, sum = 0.0f, o[kChannels];
#pragma unroll
  for (int i = 0; i < kChannels; ++i) o[i] = 0.0f;
  if (live) {
    for (int x = c0; x <= c1; ++x) {
      const RowState state = a.part_state[(2 * (int64_t)x + (x == c0 ? slot : 0)) * tile_rows + row];
      top = fmaxf(top, state.m), top_t = fmaxf(top_t, state.t);
    }
    for (int x = c0; x <= c1; ++x) {
      const int64_t first = (2 * (int64_t)x + (x == c0 ? slot : 0)) * tile_rows;
      const RowState state = a.part_state[first + row];
      const float f = fast_exp2(state.t - top_t);
      sum = fmaf(fast_exp2(state.m - top), state.l, sum);
      const float* part = a.part_o + first * D + (int64_t)d0 * tile_rows + row * 4;
#pragma unroll
      for (int i = 0; i < kChannels; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(part + i * tile_rows);
        o[i] = fmaf(f, v.x, o[i]), o[i + 1] = fmaf(f, v.y, o[i + 1]);
        o[i + 2] = fmaf(f, v.z, o[i + 2]), o[i + 3] = fmaf(f, v.w, o[i + 3]);
      }
    }
  }
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum, unit_v = fast_exp2(top_t - top);
#pragma unroll
  for (int i = 0; i < kChannels; ++i) o[i] *= inverse, o[i] *= unit_v;
  T* dst = static_cast<T*>(a.out) + b * a.out_st.b + token * a.out_st.s + head * a.out_st.h + d0;
#pragma unroll
  for (int i = 0; i < kChannels; i += 8) store8(dst + i, o + i);
  if (a.lse != nullptr && d0 == 0)
    a.lse[((int64_t)b * a.H + head) * a.T + token] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

// The row tile that holds the rows of a kv head (32 at the most, D 256: 16; more go to the kernel for many rows).  Columns
// come in eights, so a single token of up to eight heads a group takes one column tile; two a warp share the converted
// codes, D 256 has registers for one.
struct Shape {
  int nr, wm;
};
static Shape row_tile(int64_t rows, int D) {
  if (rows <= 8) return {1, 1};
  if (D == 256) return {1, 2};
  return {2, rows <= 16 ? 1 : 2};
}

// From which rows of a kv head on the kernel for many rows is taken: when they do not fit this kernel's row tile.  Up to there it
// is the faster one whatever the batch and the context are.  Measured on B200 on the device, 32 rows (D 256: 16) of 8 kv heads, us,
// few / many:
//   sequences x keys   1 x 500    1 x 4000   8 x 250    8 x 1000   64 x 250   8 x 8190   64 x 2000
//   D 64               12 / 15    22 / 31    15 / 18    18 / 24    32 / 44    39 / 55    78 / 112
//   D 96               12 / 17    25 / 40    16 / 20    20 / 27    38 / 48    47 / 61    97 / 126
//   D 128              14 / 19    26 / 47    19 / 24    24 / 32    44 / 58    57 / 67    118 / 140
//   D 256              14 / 24    26 / 63    17 / 25    24 / 39    41 / 69    65 / 95    125 / 197
// Two row tiles here took 108 us for 36 rows of 8 x 8190 keys, D 128, where the other kernel took 78 (D 64: 70 / 67, D 96: 86 / 75).
static bool wide(int64_t rows, int D) { return rows > (D == 256 ? 16 : 32); }

static int shared_ctas(int D, Shape s) { return sm_count() * (s.nr == 1 && D <= 128 ? 4 : D == 64 ? 3 : 2); }

template <typename T, int D, int NR, int WM>
static int launch_paged_attn(const PagedAttnArgs& a, cudaStream_t st) {
  using C = Config<D, NR, WM>;
  CUtensorMap k_map, v_map;
  const uint64_t rows = (uint64_t)a.p.num_pages * a.p.Hkv << a.p.page_shift;
  if (!code_map<D>(&k_map, a.p.k8, rows, 1 << a.p.page_shift) || !code_map<D>(&v_map, a.p.v8, rows, 1 << a.p.page_shift))
    return SAGE_ERR_LAUNCH;
  static std::atomic<uint64_t> prepared{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(prepared.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(paged_attn_kernel<T, D, NR, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e == cudaSuccess && dev < 64) prepared.fetch_or(uint64_t(1) << dev);
  }
  if (e == cudaSuccess) {
    e = launch_early(paged_attn_kernel<T, D, NR, WM>, dim3(a.ctas), kThreads, C::kSmem, st, a, k_map, v_map);
  }
  if (e == cudaSuccess) return SAGE_OK;
  set_error("paged attention: %s", cudaGetErrorString(e));
  return SAGE_ERR_LAUNCH;
}

template <typename T, int D>
static int launch_join(const PagedAttnArgs& a, int tile_rows, bool many, cudaStream_t st) {
  const int used = std::min(tile_rows, a.T * a.group), per_block = many ? 32 : kJoinThreads / 32;
  const int blocks = (used + per_block - 1) / per_block;
  const dim3 grid((unsigned)(a.B * a.p.Hkv * a.row_tiles * blocks));
  const cudaError_t e = launch_early(many ? wide_join_kernel<T, D> : paged_join_kernel<T, D>, grid, kJoinThreads, 0, st, a,
                                     tile_rows, blocks);
  if (e == cudaSuccess) return SAGE_OK;
  set_error("paged attention: %s", cudaGetErrorString(e));
  return SAGE_ERR_LAUNCH;
}

template <typename T, int D>
static int launch_paged_attn(const PagedAttnArgs& a, Shape s, cudaStream_t st) {
  if constexpr (D == 256)
    return s.wm == 1 ? launch_paged_attn<T, D, 1, 1>(a, st) : launch_paged_attn<T, D, 1, 2>(a, st);
  else
    return s.nr == 1   ? launch_paged_attn<T, D, 1, 1>(a, st)
           : s.wm == 1 ? launch_paged_attn<T, D, 2, 1>(a, st)
                       : launch_paged_attn<T, D, 2, 2>(a, st);
}

}  // namespace sage

using namespace sage;

extern "C" size_t sage_paged_attention_workspace_bytes(int B, int T, int H, int Hkv, int D) {
  if (B <= 0 || T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || sage_qk_row_bytes(D) == 0) return 0;
  const int64_t rows = (int64_t)T * (H / Hkv);
  const Shape s = row_tile(rows, D);
  const size_t slots = wide(rows, D) ? (size_t)2 * wide_ctas() * wide_rows(D) : (size_t)2 * shared_ctas(D, s) * 8 * s.nr * s.wm;
  return slots * (D * sizeof(float) + sizeof(RowState));
}

extern "C" int sage_paged_attention(const sage_paged_attention_args* args, void* stream) {
  NvtxRange nvtx("sage_paged_attention");
  set_error("%s", "");
  if (args == nullptr) {
    set_error("paged attention: no arguments");
    return SAGE_ERR_INVALID;
  }
  const sage_paged_kv& kv = args->kv;
  const int dtype = args->dtype, B = kv.B, T = args->T, H = args->H, Hkv = kv.Hkv, D = kv.D;
  int rc = check_rows(dtype, B, T, H, D);
  if (rc == SAGE_OK && (Hkv <= 0 || H % Hkv != 0)) {
    set_error("heads %d must be a multiple of kv heads %d", H, Hkv);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  if (rc == SAGE_OK) rc = check_rows_pointer(args->q, args->q_st, "q");
  if (rc == SAGE_OK) rc = check_rows_pointer(args->out, args->out_st, "out");
  PagedAttnArgs a{};
  if (rc == SAGE_OK) rc = paged_args(&a.p, kv);
  if (rc == SAGE_OK && (int64_t)kv.max_pages * kv.page_size > (int64_t)INT_MAX - T - kTileKeys) {
    set_error("%d pages of %d keys: positions must fit 32 bits", kv.max_pages, kv.page_size);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  if (rc == SAGE_OK && (int64_t)kv.num_pages * kv.page_size > (int64_t)INT_MAX / Hkv) {
    set_error("%d pages of %d keys and %d heads: cache rows must fit 32 bits", kv.num_pages, kv.page_size, Hkv);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  if (rc == SAGE_OK && (int64_t)B * T * H > INT_MAX / 64) {
    set_error("%d sequences of %d tokens and %d heads are too many for one call", B, T, H);
    rc = SAGE_ERR_UNSUPPORTED;
  }
  const size_t need = rc == SAGE_OK ? sage_paged_attention_workspace_bytes(B, T, H, Hkv, D) : 0;
  if (rc == SAGE_OK && (args->workspace == nullptr || args->workspace_bytes < (int64_t)need ||
                        (reinterpret_cast<uintptr_t>(args->workspace) & 15u))) {
    set_error("workspace of %zu bytes (16-byte aligned) required, got %lld", need, (long long)args->workspace_bytes);
    rc = SAGE_ERR_INVALID;
  }
  if (rc != SAGE_OK) return rc;
  a.q = args->q, a.q_st = strides3(args->q_st);
  a.out = args->out, a.out_st = strides3(args->out_st);
  a.lse = args->lse, a.counts = kv.counts;
  a.mask = args->mask, a.mask_b = args->mask_st[0], a.mask_i = args->mask_st[1];
  a.B = B, a.T = T, a.H = H, a.group = H / Hkv;
  const bool many = wide((int64_t)T * a.group, D);
  const Shape shape = row_tile((int64_t)T * a.group, D);
  const int tile_rows = many ? wide_rows(D) : 8 * shape.nr * shape.wm;
  a.row_tiles = (T * a.group + tile_rows - 1) / tile_rows;
  if (!many && a.row_tiles != 1) {   // its kernel holds all rows of a kv head
    set_error("paged attention: %d rows in tiles of %d", T * a.group, tile_rows);
    return SAGE_ERR_UNSUPPORTED;
  }
  if (((int64_t)kv.max_pages * kv.page_size / kTileKeys + 1) * a.row_tiles * Hkv > (int64_t)UINT_MAX) {
    set_error("%d tokens of %d heads over %d pages of %d keys are too many for one call", T, H, kv.max_pages, kv.page_size);
    return SAGE_ERR_UNSUPPORTED;
  }
  a.ctas = many ? wide_ctas() : shared_ctas(D, shape);
  a.scale = (float)((args->sm_scale > 0.0 ? args->sm_scale : 1.0 / std::sqrt((double)D)) * 1.4426950408889634);
  a.part_o = static_cast<float*>(args->workspace);
  a.part_state = reinterpret_cast<RowState*>(a.part_o + (size_t)2 * a.ctas * tile_rows * D);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_head_dim(D, [&](auto d) {
    constexpr int kD = decltype(d)::value;
    int rc2;
    if (many)
      rc2 = launch_paged_wide(a, dtype, st);
    else
      rc2 = dtype == SAGE_BF16 ? launch_paged_attn<__nv_bfloat16, kD>(a, shape, st) : launch_paged_attn<__half, kD>(a, shape, st);
    if (rc2 != SAGE_OK) return rc2;
    return dtype == SAGE_BF16 ? launch_join<__nv_bfloat16, kD>(a, tile_rows, many, st)
                              : launch_join<__half, kD>(a, tile_rows, many, st);
  });
}
