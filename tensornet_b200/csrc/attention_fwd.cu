// Attention within sequences, forward, on the tensor cores.
//
//   s = scores of 128 queries with 128 keys;  m = the largest so far;  p = 2^(s - m);  l += sum p;  o += p v;  out = o / l
//
// One pass over the keys.  A block has one or two tiles of 128 queries: a warp loads tiles of keys and values by TMA into a ring, a
// warp issues the products, and a warpgroup per tile has a query per thread, or two, where scores are capped, half of a query's keys
// per thread.  Scores are read from tensor memory into registers, and the weights go back into the columns that the scores had, as
// the left operand of the product with the values.
//
// The order of products is  s0(0) s1(0) | o0(0) s0(1) | o1(0) s1(1) | ...: while one tile's weights are made, the other's products
// run.  Products of one thread run in the order of their issue, so the next scores may overwrite the weights that the
// product before them reads, and a barrier behind s(j + 1) also says that o(j) is there.
//
// The reference m of a row moves only when its maximum has grown by more than 2^8: weights then stay below 2^8, and what has been
// added up is brought to the new reference by the threads that own the row.  Sums are fp32, weights bf16 for the product (their sum
// takes them unrounded).
//
// What bounds it is the exponentials, 2048 cycles of the special function unit per step of two tiles, and the latency around them:
// a step takes 3300 at 64 columns and 3700 at 128, where its products take 1024 and 2048.  A quarter of the exponentials is a
// polynomial (ex2_poly); with a third the instructions cost more than that saves.  2 x 4096 x 16 heads, us at 64 and 128 columns:
//   a query per thread 261, 281; and a quarter polynomial 238, 270; a third 256, 274
//   half a query per thread 244, 283; and a quarter polynomial 248, 286 (capped, 8192 causal: 498; a query per thread 550)
//   weights in columns of their own, scores ahead, a warp of products per tile: 246, 297; weights ahead of the maximum: 250, 322
//   steps of 64 keys with two buffers of scores: 283, 356
// In the order of their work, 8192 tokens x 16 heads x 128 columns causal: 264 us (1040 TFLOP/s of what is seen), capped 400 us.  Short
// sequences of up to 64 columns have three blocks of one tile and steps of 64 keys per SM, which hide each other's latency: 64 x 512 x 8
// heads x 64 columns 81 us.
#include <cuda_bf16.h>
#include <mutex>
#include "attention_tc.cuh"

namespace tn {

namespace {

using namespace attn;

constexpr int kRows = 128;
constexpr float kGrowth = 8.f;

template <int kD, int kTiles, int kHalves>
struct FwdShape {
  static constexpr int chunks = kD / 64;
  static constexpr bool small = kD == 64 && kTiles == 1;      // three blocks per SM
  static constexpr int keys = small ? 64 : 128;                // of a step
  static constexpr int q_bytes = kRows * 128 * chunks, slot_bytes = keys * 128 * chunks;
  static constexpr int slots = kTiles == 2 ? (kD == 128 ? 4 : 6) : (kD == 128 ? 2 : 4);
  static constexpr int softmax_warps = 4 * kHalves * kTiles;
  static constexpr int threads = 32 * (softmax_warps + 2);
  static constexpr int blocks = kTiles == 2 ? 1 : small && kHalves == 1 ? 3 : 2;      // per SM
  static constexpr int smem = q_bytes * kTiles + slot_bytes * slots + 1024;
  static constexpr int tmem_cols = kTiles == 2 ? 512 : small ? 128 : 256;
  static constexpr int o_col = keys * kTiles;
};

// The two warps that have half of the same queries' keys each
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool any_of_pair(int id, bool p) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "bar.red.or.pred q, %1, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(id), "r"((uint32_t)p)
      : "memory");
  return any != 0;
}

struct FwdMaps {
  CUtensorMap q, k, v;
};

template <int kD, int kTiles, Cap kCap, bool kBias>
__global__ void __launch_bounds__(FwdShape<kD, kTiles, kCap ? 2 : 1>::threads, FwdShape<kD, kTiles, kCap ? 2 : 1>::blocks)
attention_fwd_tc_kernel(const __grid_constant__ FwdMaps maps, const __grid_constant__ AttnArgs a, int tiles, int heads_first) {
  constexpr int kHalves = kCap ? 2 : 1;      // threads per query
  using Shape = FwdShape<kD, kTiles, kHalves>;
  constexpr int kKeys = Shape::keys, kHalf = kKeys / kHalves;      // of a step; of a thread
  constexpr int kSlots = Shape::slots;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_q, s_full[kSlots], s_empty[kSlots], s_score[kTiles], s_weight[kTiles], s_out[kTiles];
  __shared__ float s_pass[kTiles][2][kRows];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort_i;
  volatile int* s_abort = &s_abort_i;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int h = heads_first ? blockIdx.x % a.H : blockIdx.x / tiles;

  asm volatile("griddepcontrol.wait;" ::: "memory");
  // The last tiles of causal sequences have the most keys: they go first, those of all heads (8192 tokens x 16 heads, capped: 498 -> 404
  // us); where sequences are short, blocks of one head follow each other (780 of 256 x 4 heads: 263 -> 233).
  const Tile tile = tile_of<true>(a.rq, a.B, kRows * kTiles, tiles - 1 - (int)(heads_first ? blockIdx.x / a.H : blockIdx.x % tiles));
  if (!tile.any) return;
  const int tile_rows = min(kRows * kTiles, tile.rows.n - tile.first);      // of the output that are this block's
  Span qs{tile.rows.b, tile.rows.first, 0}, ks{0, 0, 0};
  if (tile.seq >= 0) {
    qs = span_of(a.rq, tile.seq);
    ks = span_of(a.rk, tile.seq);
  }
  // keys that tile t sees, none where it has no queries; keys_seen grows with the query
  int vis[kTiles], most = 0;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int i0 = tile.first + t * kRows;
    vis[t] = i0 < qs.n ? keys_seen(a, tile.seq, min(i0 + kRows, qs.n) - 1, qs.n, ks.n) : 0;
    most = max(most, vis[t]);
  }
  if (most == 0) {
    const int per = a.D / 8;
    for (int i = threadIdx.x; i < tile_rows * per; i += Shape::threads)
      for (const AttnOperand* to : {&a.o, &a.rest})
        if (to->p != nullptr)
          *reinterpret_cast<uint4*>(at_out(*to, tile.rows.b, tile.rows.first + tile.first + i / per, h) + i % per * 8) = make_uint4(0, 0, 0, 0);
    if (a.lse != nullptr && tile.seq >= 0)
      for (int i = threadIdx.x; i < tile_rows; i += Shape::threads)
        a.lse[(long long)h * (a.rq.off ? a.rq.T : (long long)a.B * a.rq.T) + (a.rq.off ? 0 : (long long)tile.rows.b * a.rq.T) + tile.rows.first +
              tile.first + i] = CUDART_INF_F;
    return;
  }
  // what one lane's loads and products are addressed with is known to be the same for the warp
#pragma unroll
  for (int t = 0; t < kTiles; ++t) vis[t] = one_of_warp(vis[t]);
  const int steps = one_of_warp((most + kKeys - 1) / kKeys);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t ring = base + kTiles * Shape::q_bytes;

  if (threadIdx.x == 0) {
    *s_abort = 0;
    mbar_init(smem_u32(&s_q), 1);
    for (int s = 0; s < kSlots; ++s) { mbar_init(smem_u32(&s_full[s]), 1); mbar_init(smem_u32(&s_empty[s]), 1); }
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(smem_u32(&s_score[t]), 1);
      mbar_init(smem_u32(&s_weight[t]), kHalves * kRows);
      mbar_init(smem_u32(&s_out[t]), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc<Shape::tmem_cols>(&s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // The kernel behind this one may start now, and not before: it may want tensor memory ahead of its own wait, and a block of this kernel
  // that had none yet would then wait for a block that waits for this kernel.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = s_tmem;
  const int d16 = round16(a.D);

  if (warp == Shape::softmax_warps) {
    // ---- loads: the queries, then k(0) v(0) k(1) v(1) ... through the ring
    const int g = h / (a.H / a.G), k_first = one_of_warp(ks.first), k_b = one_of_warp(ks.b), q_first = one_of_warp(qs.first + tile.first);
    const bool lead = elect_one();
    if (lead) {
      int n = 0;
      for (int t = 0; t < kTiles; ++t) n += vis[t] > 0;
      mbar_expect_tx(smem_u32(&s_q), n * Shape::q_bytes);
      for (int t = 0; t < kTiles; ++t)
        if (vis[t] > 0)
          for (int c = 0; c < Shape::chunks; ++c)
            tma_load_4d(base + t * Shape::q_bytes + c * (kRows * 128), &maps.q, 64 * c, q_first + t * kRows, h, qs.b, smem_u32(&s_q));
    }
    __syncwarp();
    for (int i = 0; i < 2 * steps; ++i) {
      const int s = i % kSlots;
      if (i >= kSlots && !mbar_wait_warp(smem_u32(&s_empty[s]), ((i / kSlots) & 1) ^ 1, s_abort)) { *s_abort = 1; break; }
      if (lead) {
        const uint32_t bar = smem_u32(&s_full[s]);
        mbar_expect_tx(bar, Shape::slot_bytes);
        for (int c = 0; c < Shape::chunks; ++c)
          tma_load_4d(ring + s * Shape::slot_bytes + c * (kKeys * 128), (i & 1) ? &maps.v : &maps.k, 64 * c, k_first + (i >> 1) * kKeys, g, k_b, bar);
      }
      __syncwarp();
    }
  } else if (warp == Shape::softmax_warps + 1) {
    // ---- products
    const bool lead = elect_one();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    bool ok = mbar_wait_warp(smem_u32(&s_q), 0, s_abort);
    auto full = [&](int i) {           // load i of the ring has landed
      ok = ok && mbar_wait_warp(smem_u32(&s_full[i % kSlots]), (i / kSlots) & 1, s_abort);
      tc_fence_after();
    };
    auto scores = [&](int t, int j) {
      const uint32_t q = base + t * Shape::q_bytes, k = ring + (2 * j % kSlots) * Shape::slot_bytes;
      const uint32_t id = idesc_of(round16(min(kKeys, vis[t] - j * kKeys)), false);
      if (lead) {
        const uint64_t qd = make_smem_desc(q, 16u, 1024u), kd = make_smem_desc(k, 16u, 1024u);
#pragma unroll
        for (int s = 0; s < kD / 16; ++s)
          if (s * 16 < d16) umma_f16(tm + t * kKeys, qd + step_k<kRows>(s), kd + step_k<kKeys>(s), id, s > 0);
        umma_commit(smem_u32(&s_score[t]));
      }
      __syncwarp();
    };
    auto values = [&](int t, int j) {
      const uint32_t v = ring + ((2 * j + 1) % kSlots) * Shape::slot_bytes;
      const int n = round16(min(kKeys, vis[t] - j * kKeys)) / 16;
      const uint32_t id = idesc_of(d16, true);
      if (lead) {
        const uint64_t vd = make_smem_desc(v, kKeys * 128, 1024u);
#pragma unroll
        for (int s = 0; s < kKeys / 16; ++s)
          if (s < n) umma_f16_ts(tm + Shape::o_col + t * kD, tm + t * kKeys + s * 8, vd + step_mn(s), id, j > 0 || s > 0);
      }
      __syncwarp();
    };
    auto free_slot = [&](int i) {
      if (lead && i + kSlots < 2 * steps) umma_commit(smem_u32(&s_empty[i % kSlots]));
      __syncwarp();
    };
    full(0);
    if (ok) {
      for (int t = 0; t < kTiles; ++t)
        if (vis[t] > 0) scores(t, 0);
      free_slot(0);
    }
    for (int j = 0; j < steps && ok; ++j) {
      full(2 * j + 1);
      if (!ok) break;
      const int end = ks.n - j * kKeys;            // rows of this tile of values that the sequence has
      if (end < kKeys && (end & 15)) zero_rows<kKeys>(smem_gen + (ring - base) + ((2 * j + 1) % kSlots) * Shape::slot_bytes, Shape::chunks, end, round16(end), lane);
      bool next = false;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        if (j * kKeys >= vis[t]) continue;
        ok = ok && mbar_wait_warp(smem_u32(&s_weight[t]), j & 1, s_abort);
        if (!ok) break;
        tc_fence_after();
        values(t, j);
        if ((j + 1) * kKeys < vis[t]) {
          if (!next) full(2 * j + 2);
          if (!ok) break;
          next = true;
          scores(t, j + 1);
        } else {
          if (lead) umma_commit(smem_u32(&s_out[t]));
          __syncwarp();
        }
      }
      free_slot(2 * j + 1);
      if (next) free_slot(2 * j + 2);
    }
    if (!ok) *s_abort = 1;
  } else {
    // ---- softmax
    const int t = warp / (4 * kHalves), half = kHalves == 2 ? (warp >> 2) & 1 : 0, r = (warp & 3) * 32 + lane;
    const int pair = 1 + t * 4 + (warp & 3);           // the barrier of the two warps that share 32 queries
    const int i = tile.first + t * kRows + r;
    const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tm_s = tm + t * kKeys + half * kHalf, tm_p = tm + t * kKeys + half * (kHalf / 2), tm_o = tm + Shape::o_col + t * kD;
    const int my_vis = t == 0 ? vis[0] : vis[kTiles - 1];
    const int lim = i < qs.n ? keys_seen(a, tile.seq, i, qs.n, ks.n) : my_vis;
    const int least = keys_seen(a, tile.seq, tile.first + t * kRows, qs.n, ks.n);      // of the tile's queries
    const float c = kCap ? a.scale / a.cap : a.scale * kLog2e;
    const float cap2 = a.cap * kLog2e;
    const float slope2 = kBias ? a.slopes[h] * kLog2e : 0.f;
    const int place0 = place_of(a, tile.first + t * kRows, qs.n, ks.n);          // of the tile's first query
    const int place = place_of(a, i, qs.n, ks.n);
    float m = kNone, l = 0.f;
    const int d_half = kHalves == 2 ? round16(d16 / 2) : d16;
    bool ok = true;
    for (int j = 0; j * kKeys < my_vis; ++j) {
      ok = ok && mbar_wait_warp(smem_u32(&s_score[t]), j & 1, s_abort);
      if (!ok) *s_abort = 1;         // (the pair's barriers are passed all the same)
      tc_fence_after();
      const int j0 = j * kKeys + half * kHalf, wide = min(kHalf, my_vis - j0);              // columns of scores
      const bool masked = j0 + kHalf > least;
      float2 s[kHalf / 2];
#pragma unroll
      for (int c0 = 0; c0 < kHalf; c0 += 32)
        if (ok && c0 < wide) tmem_ld32_nowait(tm_s + c0, reinterpret_cast<uint32_t*>(s + c0 / 2));
      tmem_ld_wait();
      // all keys on one side of all queries: the distance is linear in the key
      const float side = kBias ? (j0 + kHalf <= place0 ? 1.f : (j0 >= place0 + kRows ? -1.f : 0.f)) : 0.f;
      float tops[4] = {kNone, kNone, kNone, kNone};
#pragma unroll
      for (int c0 = 0; c0 < kHalf; c0 += 32) {
        if (c0 >= wide) continue;
        float2* x = s + c0 / 2;
        if (kCap) {
          // which tanh it is goes by scores that are seen, not by what else the columns hold
          float far[2] = {0.f, 0.f};
          if (masked) {
            const int there = lim - j0 - c0;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = make_float2(2 * e < there ? x[e].x : 0.f, 2 * e + 1 < there ? x[e].y : 0.f);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            x[e] = mul2(x[e], both(c));
            far[e & 1] = max3(far[e & 1], fabsf(x[e].x), fabsf(x[e].y));
          }
          if (__all_sync(0xffffffffu, i >= qs.n || fmaxf(far[0], far[1]) <= 1.f)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = mul2(tanh_small(x[e]), both(cap2));
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = mul2(tanh_any<kCap>(x[e]), both(cap2));
          }
        }
        if (kBias) {
          if (side != 0.f) {
            const float2 from = both(slope2 * side * (float)(j0 + c0 - place)), by = both(slope2 * side);
            float2 n = make_float2(0.f, 1.f);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 bias = fma2(n, by, from);
              x[e] = kCap ? add2(x[e], bias) : fma2(x[e], both(c), bias);
              n = add2(n, both(2.f));
            }
          } else {
            const float away = (float)(place - j0 - c0);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (!kCap) x[e] = mul2(x[e], both(c));
              x[e].x = fmaf(-slope2, fabsf(away - (float)(2 * e)), x[e].x);
              x[e].y = fmaf(-slope2, fabsf(away - (float)(2 * e + 1)), x[e].y);
            }
          }
        }
        if (masked) {
          const int there = lim - j0 - c0;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            x[e].x = 2 * e < there ? x[e].x : kNone;
            x[e].y = 2 * e + 1 < there ? x[e].y : kNone;
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) tops[e & 3] = max3(tops[e & 3], x[e].x, x[e].y);
      }
      float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      if (!kCap && !kBias) top *= c;
      // (behind the barrier both warps have their scores in registers, and weights may take their place)
      if (kHalves == 2 ? any_of_pair(pair, top > m + kGrowth) : __any_sync(0xffffffffu, top > m + kGrowth) != 0) {
        if (kHalves == 2) {
          s_pass[t][half][r] = top;
          pair_sync(pair);
          top = fmaxf(top, s_pass[t][half ^ 1][r]);
        }
        const float to = top > m + kGrowth ? top : m;
        const float by = to == kNone ? 1.f : ex2(m - to);
        m = to;
        l *= by;
        if (j > 0) {
          for (int c0 = half * d_half; c0 < (half ? d16 : d_half); c0 += 16) {
            float o[16];
            tmem_ld16_nowait(tm_o + c0, reinterpret_cast<uint32_t*>(o));
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= by;
            tmem_st16(tm_o + c0, reinterpret_cast<const uint32_t*>(o));
          }
        }
        if (kHalves == 2) pair_sync(pair);             // s_pass is free again
      }
      const float2 ref = both(m == kNone ? 0.f : -m);
      float2 sums[2] = {make_float2(l, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c0 = 0; c0 < kHalf; c0 += 32) {
        if (c0 >= wide) continue;
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float2 x = s[c0 / 2 + e];
          x = (kCap || kBias) ? add2(x, ref) : fma2(x, both(c), ref);
          x = !kCap && e % 4 == 3 ? ex2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
          sums[e & 1] = add2(sums[e & 1], x);
          w[e] = pack_bf16(x.x, x.y);
        }
        tmem_st16(tm_p + c0 / 2, w);
      }
      sums[0] = add2(sums[0], sums[1]);
      l = sums[0].x + sums[0].y;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(smem_u32(&s_weight[t]));
    }
    if (kHalves == 2) {
      s_pass[t][half][r] = l;
      pair_sync(pair);
      l += s_pass[t][half ^ 1][r];
    }
    if (ok && my_vis > 0) {
      ok = mbar_wait_warp(smem_u32(&s_out[t]), 0, s_abort);
      if (!ok) *s_abort = 1;
      tc_fence_after();
    }
    if (ok) {
      const float w = l > 0.f && i < qs.n ? 1.f / l : 0.f;
      const bool mine = t * kRows + r < tile_rows;
      const long long row = tile.rows.first + i;
      __nv_bfloat16* out = at_out(a.o, tile.rows.b, row, h);
      for (int c0 = half * d_half; c0 < (half ? a.D : min(a.D, d_half)); c0 += 16) {
        float o[16];
        if (my_vis > 0) {
          tmem_ld16_nowait(tm_o + c0, reinterpret_cast<uint32_t*>(o));
          tmem_ld_wait();
        }
        if (mine) {
          const bool some = w != 0.f;         // (what a row without weights holds may be anything)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = some ? o[e] : 0.f;
          __nv_bfloat16* rest = a.rest.p ? at_out(a.rest, tile.rows.b, row, h) : nullptr;
#pragma unroll
          for (int e = 0; e < 16; e += 8)
            if (c0 + e < a.D) {
              const uint4 v = pack8(o + e, w);
              *reinterpret_cast<uint4*>(out + c0 + e) = v;
              if (rest) *reinterpret_cast<uint4*>(rest + c0 + e) = rest8(o + e, w, v);
            }
        }
        __syncwarp();
      }
      if (a.lse != nullptr && mine && half == 0)
        a.lse[(long long)h * (a.rq.off ? a.rq.T : (long long)a.B * a.rq.T) + (a.rq.off ? 0 : (long long)tile.rows.b * a.rq.T) + row] =
            w != 0.f ? m + log2f(l) : CUDART_INF_F;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*s_abort) {
    if (threadIdx.x == 0) set_status(a.status, kMbarTimeout, 40, (int)blockIdx.x);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);        // copies in flight land
    __syncthreads();
  }
  if (warp == 0) tmem_dealloc<Shape::tmem_cols>(tmem);
}

template <int kD, int kTiles, Cap kCap, bool kBias>
cudaError_t launch(const FwdMaps& maps, const AttnArgs& a, cudaStream_t st) {
  using Shape = FwdShape<kD, kTiles, kCap ? 2 : 1>;
  auto* k = attention_fwd_tc_kernel<kD, kTiles, kCap, kBias>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::smem);      // of the current device
  if (e != cudaSuccess) return e;
  const long long tiles = tile_count(a.rq, a.B, kRows * kTiles), blocks = tiles * a.H;
  if (blocks >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  return launch_pdl(k, dim3((unsigned)blocks), dim3(Shape::threads), Shape::smem, st, maps, a, (int)tiles, mean_length(a.rq, a.B) > 512);
}
template <int kD, int kTiles>
cudaError_t launch(const FwdMaps& maps, const AttnArgs& a, cudaStream_t st) {
  return with_cap(a, [&](auto cap) {
    return a.slopes ? launch<kD, kTiles, decltype(cap)::value, true>(maps, a, st) : launch<kD, kTiles, decltype(cap)::value, false>(maps, a, st);
  });
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

}  // namespace

namespace attn {
bool operand_map(const AttnOperand& o, int D, const AttnRows& r, int B, int heads, int box_rows, CUtensorMap* out) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  // A thread that has made no call of the runtime yet, as one of torch's graph, has no context for the driver's call.
  thread_local int bound = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (bound != dev) {
    if (cudaSetDevice(dev) != cudaSuccess) return false;
    bound = dev;
  }
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)r.T, (cuuint64_t)heads, (cuuint64_t)(r.off ? 1 : B)};
  const cuuint64_t strides[3] = {(cuuint64_t)o.st * 2, (cuuint64_t)o.sh * 2, r.off ? (cuuint64_t)16 : (cuuint64_t)o.sb * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
  return enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, o.p, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
}  // namespace attn

const char* launch_attention_fwd(const AttnArgs& a, cudaStream_t st) {
  // Two tiles share what is loaded; one leaves room for another block, whose set-up and end it hides.  us with two and with one:
  // documents of 60 to 8000 (mean 1650) x 8 heads 341 and 364, 8192 tokens x 16 heads 404 and 418; 64 x 512 x 8 heads 103 and 98, 500
  // sequences of 400 x 4 heads 340 and 320, 6 of 333 to 1999 x 6 heads, which is 288 blocks of two, 72 and 66.
  const bool two = mean_length(a.rq, a.B) > 1024 && tile_count(a.rq, a.B, 2 * kRows) * a.H >= 2 * 148;
  const int keys = two || a.D > 64 ? FwdShape<128, 1, 1>::keys : FwdShape<64, 1, 1>::keys;
  FwdMaps maps;
  if (!operand_map(a.q, a.D, a.rq, a.B, a.H, kRows, &maps.q) || !operand_map(a.k, a.D, a.rk, a.B, a.G, keys, &maps.k) ||
      !operand_map(a.v, a.D, a.rk, a.B, a.G, keys, &maps.v))
    return "attention: cuTensorMapEncodeTiled failed";
  cudaError_t e = a.D > 64 ? (two ? launch<128, 2>(maps, a, st) : launch<128, 1>(maps, a, st))
                           : (two ? launch<64, 2>(maps, a, st) : launch<64, 1>(maps, a, st));
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace tn
