// Attention within sequences, backward, on the tensor cores.
//
//   p = 2^(s - lse);  dp = do v^T;  ds = p (dp - delta) ds/dx  with delta = sum(do o)
// (o with what rounding it to bf16 took off: without, gradients of sequences of 40 were off by 0.0030 of their norm, now by 0.0024,
// where rounding them in the end alone takes 0.0017)
//   dv = p^T do;  dk = scale ds^T q;  dq = scale ds k
//
// Every result has one owner, so no sums meet in memory and their order is fixed: a block owns 128 keys and walks over the queries
// of all heads that share them (dk, dv), or owns 128 queries and walks over their keys (dq).  That costs the scores and dp twice,
// seven products in place of five; sums of dq in memory would need a pass of their own over fp32 rows, and an order.
//
// Both kinds of block are one program.  X are the two operands of the 128 rows that it owns, Y those of the 128 or 64 rows at a time
// that it walks over: (K, V) and (Q, dO), or (Q, dO) and (K, V).
//   s = X1 Y1^T, dp = X2 Y2^T;   acc1 += ds Y1;   acc2 += p Y2 (keys' owners only)
// A thread has 32 columns of a row.  p and ds are made in registers and go back into the columns of tensor memory that the thread's s
// and dp had, as left operands; the tiles of Y serve as right operands of both kinds of product.  Where keys own the rows, queries
// are columns, and the loading warp brings their lse and delta to shared memory.
//
// The products of a step are issued in the order  acc2(i) s(i + 1) | acc1(i) dp(i + 1):  p(i) is made while dp(i) is, ds(i) while acc2
// and the next scores are.
//
// ds goes into its product as a sum of two bf16, the second in the columns that the first leaves free, where sequences are short or
// columns few.  sum ds k loses the part of k that the weights agree on, as sum ds = 0, and a rounding of ds does not: with 8 columns
// dq was off by 0.0030 of its norm so, with 128 columns of sequences of 2 by 0.0029, now by 0.0017.  Sequences of up to 128 take 3 % more
// time, up to 24 columns 10 to 17 % (8 of 4000 x 4 heads, us: 297 and 338); with more columns and keys 0.0025 is left as it is
// (128 columns: 479 and 530).
//
// What bounds it above 64 columns: a step of 128 x 128 takes 3300 cycles where keys are owned, of which its four products take 2300 and
// p and ds 2400, partly beside them; and 2800 where queries are.  A product of 128 x 64 x 16 takes 62 cycles, one of 128 x 128 x 16
// 72, so that steps of 64 rows with two buffers of s and dp were bound by their products.  8192 tokens x 16 heads x 128 columns
// causal, us: steps of 64 with a row per thread 980, half a row 917, steps of 128 as they are 845; capped 1607, 1209, 1060.
// Up to 64 columns the blocks of short sequences spend their time on setting up, and two per SM hide that from each other: 1562
// sequences of 128, 4 heads x 64 causal, 635 us, with one block per SM and steps of 128 rows 846; documents of 60 to 8000, 944 and 1010.
#include <cuda_bf16.h>
#include "attention_tc.cuh"

namespace tn {

namespace {

using namespace attn;

constexpr int kX = 128, kPart = 32;      // rows, columns of a thread

// Above 64 columns a block per SM takes steps of 128 rows of Y; up to 64, two blocks per SM take steps of 64.
template <int kD>
struct BwdShape {
  static constexpr int chunks = kD / 64;
  static constexpr int y = kD == 128 ? 128 : 64, parts = y / kPart;
  static constexpr int slots = kD == 128 ? 2 : 3;
  static constexpr int x_bytes = kX * 128 * chunks, y_bytes = y * 128 * chunks;      // of one operand's tile
  static constexpr int soft_warps = 4 * parts;
  static constexpr int threads = 32 * (soft_warps + 2);
  static constexpr int smem = 2 * x_bytes + 2 * slots * y_bytes + 1024;
  static constexpr int dp_col = y, acc_col = 2 * y;
  static constexpr int tmem_cols = kD == 128 ? 512 : 256;
  static_assert(acc_col + 2 * kD <= tmem_cols, "s, dp and two results");
};

struct BwdMaps {
  CUtensorMap q, k, v, go;      // boxes of a step's rows
};

template <int kD>
struct BwdShared {
  uint64_t x, full[2][BwdShape<kD>::slots], empty[2][BwdShape<kD>::slots], score, read, weight, dp, ds[2], acc, vec_full[2];      // ds by turns: two warps wait for it
  uint32_t tmem;
  int abort;
  alignas(16) float vec[2][2][BwdShape<kD>::y];      // of a tile of queries less lse, less delta; two tiles take turns
};

// A thread's columns [c0, c0 + 16) of an accumulator, times w, to a row of the result; zeros where the row has no terms
__device__ __forceinline__ void store_acc(uint32_t tm, int from, int to, int D, bool mine, bool some, float w, __nv_bfloat16* row) {
  for (int c0 = from; c0 < to; c0 += 16) {
    float o[16];
    tmem_ld16_nowait(tm + c0, reinterpret_cast<uint32_t*>(o));
    tmem_ld_wait();
    if (mine) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = some ? o[e] : 0.f;
      *reinterpret_cast<uint4*>(row + c0) = pack8(o, w);
      if (c0 + 8 < D) *reinterpret_cast<uint4*>(row + c0 + 8) = pack8(o + 8, w);
    }
    __syncwarp();
  }
}

// kKeys: the block owns keys; kSplit: ds in two terms
template <int kD, bool kKeys, Cap kCap, bool kBias, bool kSplit>
__device__ __forceinline__ void bwd_block(const BwdMaps& maps, const AttnArgs& a, BwdShared<kD>& sh, uint8_t* smem_raw, int tile_at, int head) {
  using Shape = BwdShape<kD>;
  constexpr int kSlots = Shape::slots, kY = Shape::y, kParts = Shape::parts;
  volatile int* s_abort = &sh.abort;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const Tile tile = tile_of<true>(kKeys ? a.rk : a.rq, a.B, kX, tile_at);
  if (!tile.any) return;
  const int tile_rows = min(kX, tile.rows.n - tile.first);
  Span qs{tile.rows.b, tile.rows.first, 0}, ks = qs;
  if (tile.seq >= 0) {
    qs = span_of(a.rq, tile.seq);
    ks = span_of(a.rk, tile.seq);
  }
  const Span& xs = kKeys ? ks : qs;
  const Span& ys = kKeys ? qs : ks;
  const int last = min(tile.first + kX, xs.n) - 1;            // row of the sequence
  const int R = a.H / a.G;
  // rows of Y that rows of X meet: [lo, hi), and where all of them meet all: [all_lo, all_hi)
  int lo = 0, hi = 0, all_lo = 0, all_hi = 0;
  if (tile.first < xs.n) {
    if (kKeys) {
      lo = first_query(a, tile.seq, tile.first, qs.n, ks.n) & ~15;
      hi = qs.n;
      all_lo = first_query(a, tile.seq, last, qs.n, ks.n);
      all_hi = qs.n;
    } else {
      hi = keys_seen(a, tile.seq, last, qs.n, ks.n);
      all_hi = keys_seen(a, tile.seq, tile.first, qs.n, ks.n);
    }
  }
  const int steps_ = hi > lo ? (hi - lo + kY - 1) / kY * (kKeys ? R : 1) : 0;
  if (steps_ == 0) {
    const int per = a.D / 8;
    for (int i = threadIdx.x; i < tile_rows * per; i += Shape::threads) {
      const long long row = tile.rows.first + tile.first + i / per;
      *reinterpret_cast<uint4*>(at_out(kKeys ? a.gk : a.gq, tile.rows.b, row, head) + i % per * 8) = make_uint4(0, 0, 0, 0);
      if (kKeys) *reinterpret_cast<uint4*>(at_out(a.gv, tile.rows.b, row, head) + i % per * 8) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  // what one lane's loads and products are addressed with is known to be the same for the warp
  const int steps = one_of_warp(steps_);
  lo = one_of_warp(lo);
  hi = one_of_warp(hi);
  const int y_end = one_of_warp(ys.n), y_begin = one_of_warp(ys.first), y_b = one_of_warp(ys.b), x_begin = one_of_warp(xs.first + tile.first);
  head = one_of_warp(head);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* ring_gen = smem_raw + (base - smem_u32(smem_raw)) + 2 * Shape::x_bytes;
  const uint32_t ring = base + 2 * Shape::x_bytes;      // tiles of Y1, then of Y2
  if (threadIdx.x == 0) {
    *s_abort = 0;
    mbar_init(smem_u32(&sh.x), 1);
    for (int o = 0; o < 2; ++o)
      for (int s = 0; s < kSlots; ++s) { mbar_init(smem_u32(&sh.full[o][s]), 1); mbar_init(smem_u32(&sh.empty[o][s]), 1); }
    for (uint64_t* b : {&sh.score, &sh.dp, &sh.acc, &sh.vec_full[0], &sh.vec_full[1]}) mbar_init(smem_u32(b), 1);
    for (uint64_t* b : {&sh.read, &sh.weight, &sh.ds[0], &sh.ds[1]}) mbar_init(smem_u32(b), kX * kParts);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc<Shape::tmem_cols>(&sh.tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // The kernel behind this one may start now, and not before: it may want tensor memory ahead of its own wait, and a block of this kernel
  // that had none yet would then wait for a block that waits for this kernel.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = sh.tmem;
  const int d16 = round16(a.D);
  const long long q_rows = flat_rows(a.rq, a.B), q_flat = (a.rq.off ? 0 : (long long)qs.b * a.rq.T) + qs.first;

  if (warp == Shape::soft_warps) {
    // ---- loads: Y1 and Y2 of a step, each into a ring of its own, and where queries are columns their lse and delta
    const bool lead = elect_one();
    if (lead) {
      const uint32_t bar = smem_u32(&sh.x);
      mbar_expect_tx(bar, 2 * Shape::x_bytes);
      for (int o = 0; o < 2; ++o)
        for (int c = 0; c < Shape::chunks; ++c)
          for (int r = 0; r < kX; r += kY)
            tma_load_4d(base + o * Shape::x_bytes + c * (kX * 128) + r * 128, kKeys ? (o ? &maps.v : &maps.k) : (o ? &maps.go : &maps.q), 64 * c,
                        x_begin + r, head, xs.b, bar);
    }
    __syncwarp();
    int y0 = lo, h = kKeys ? head * R : head / R;
    bool ok = true;
    float l[kY / 32], d[kY / 32];
    auto fetch = [&]() {
#pragma unroll
      for (int e = 0; e < kY / 32; ++e) {
        const int i = y0 + e * 32 + lane;
        const long long from = h * q_rows + q_flat + i;
        l[e] = i < hi ? -a.lse[from] : 0.f;
        d[e] = i < hi ? -a.delta[from] : 0.f;
      }
    };
    if (kKeys) fetch();
    for (int it = 0; it < steps && ok; ++it) {
      const int s = it % kSlots;
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        ok = ok && (it < kSlots || mbar_wait_warp(smem_u32(&sh.empty[o][s]), ((it / kSlots) & 1) ^ 1, s_abort));
        if (!ok) { *s_abort = 1; break; }
        if (lead) {
          const uint32_t bar = smem_u32(&sh.full[o][s]);
          mbar_expect_tx(bar, Shape::y_bytes);
          for (int c = 0; c < Shape::chunks; ++c)
            tma_load_4d(ring + (o * kSlots + s) * Shape::y_bytes + c * (kY * 128), kKeys ? (o ? &maps.go : &maps.q) : (o ? &maps.v : &maps.k), 64 * c,
                        y_begin + y0, h, y_b, bar);
        }
        __syncwarp();
      }
      if (kKeys) {
        // step it - 2 has been through with these places
        ok = ok && (it < 2 || mbar_wait_warp(smem_u32(&sh.ds[it & 1]), ((it >> 1) & 1) ^ 1, s_abort));
        if (!ok) *s_abort = 1;
#pragma unroll
        for (int e = 0; e < kY / 32; ++e) {
          sh.vec[it & 1][0][e * 32 + lane] = l[e];
          sh.vec[it & 1][1][e * 32 + lane] = d[e];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.vec_full[it & 1]));
      }
      y0 += kY;
      if (kKeys && y0 >= hi) { y0 = lo; ++h; }
      if (kKeys && it + 1 < steps) fetch();
    }
  } else if (warp == Shape::soft_warps + 1) {
    // ---- products
    const bool lead = elect_one();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    bool ok = mbar_wait_warp(smem_u32(&sh.x), 0, s_abort);
    auto wait = [&](uint64_t& bar, int parity) {
      ok = ok && mbar_wait_warp(smem_u32(&bar), parity, s_abort);
      tc_fence_after();
      return ok;
    };
    // X(o) Y(o)^T of step it, whose columns start at row y0 of Y
    auto outer = [&](int o, int it, int y0, uint64_t& done) {
      const int s = it % kSlots;
      if (!wait(sh.full[o][s], (it / kSlots) & 1)) return;
      const int end = y_end - y0;
      if (end < kY && (end & 15))      // rows behind the sequence's end
        zero_rows<kY>(ring_gen + (o * kSlots + s) * Shape::y_bytes, Shape::chunks, end, round16(end), lane);
      const uint32_t id = idesc_of(round16(min(kY, hi - y0)), false);
      if (lead) {
        const uint64_t xd = make_smem_desc(base + o * Shape::x_bytes, 16u, 1024u), yd = make_smem_desc(ring + (o * kSlots + s) * Shape::y_bytes, 16u, 1024u);
#pragma unroll
        for (int k = 0; k < kD / 16; ++k)
          if (k * 16 < d16) umma_f16(tm + o * Shape::dp_col, xd + step_k<kX>(k), yd + step_k<kY>(k), id, k > 0);
        umma_commit(smem_u32(&done));
      }
      __syncwarp();
    };
    // acc += left Y(o): left operands lie where s (for p) or dp (for ds) of each thread's columns began
    auto inner = [&](int o, int it, int y0, uint32_t left, uint32_t acc, bool first) {
      const int n = round16(min(kY, hi - y0)) / 16;
      const uint32_t id = idesc_of(d16, true);
      if (lead) {
        const uint64_t yd = make_smem_desc(ring + (o * kSlots + it % kSlots) * Shape::y_bytes, kY * 128, 1024u);
#pragma unroll
        for (int k = 0; k < kY / 16; ++k)
          if (k < n) umma_f16_ts(tm + acc, tm + left + (k / 2) * kPart + (k & 1) * 8, yd + step_mn(k), id, !first || k > 0);
      }
      __syncwarp();
    };
    auto free_slot = [&](int o, int it) {
      if (lead && it + kSlots < steps) umma_commit(smem_u32(&sh.empty[o][it % kSlots]));
      __syncwarp();
    };
    int y0 = lo;
    outer(0, 0, y0, sh.score);
    outer(1, 0, y0, sh.dp);
    if (!kKeys) free_slot(1, 0);
    for (int it = 0; it < steps && ok; ++it) {
      const bool more = it + 1 < steps;
      const int next = kKeys && y0 + kY >= hi ? lo : y0 + kY;
      if (!wait(kKeys ? sh.weight : sh.read, it & 1)) break;
      if (kKeys) {
        inner(1, it, y0, 0, Shape::acc_col + kD, it == 0);
        free_slot(1, it);
      }
      if (more) outer(0, it + 1, next, sh.score);
      if (!wait(sh.ds[it & 1], (it >> 1) & 1)) break;
      inner(0, it, y0, Shape::dp_col, Shape::acc_col, it == 0);
      if (kSplit) inner(0, it, y0, Shape::dp_col + kPart / 2, Shape::acc_col, false);
      free_slot(0, it);
      if (more) {
        outer(1, it + 1, next, sh.dp);
        if (!kKeys) free_slot(1, it + 1);
      }
      y0 = next;
    }
    if (ok && lead) umma_commit(smem_u32(&sh.acc));
    __syncwarp();
    if (!ok) *s_abort = 1;
  } else {
    // ---- p and ds: 32 columns of a row of X per thread
    const int c0 = (warp >> 2) * kPart, r = (warp & 3) * 32 + lane;
    const int x = tile.first + r;
    const uint32_t tm_row = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tm = tm_row + c0;
    const float c = kCap ? a.scale / a.cap : a.scale * kLog2e;
    const float cap2 = a.cap * kLog2e;
    // keys: the queries [meet, qs.n) see this one; queries: keys [0, meet) are seen
    const int meet = x < xs.n ? (kKeys ? first_query(a, tile.seq, x, qs.n, ks.n) : keys_seen(a, tile.seq, x, qs.n, ks.n)) : (kKeys ? lo : hi);
    const int shift = ks.n - qs.n;
    const int place = place_of(a, x, qs.n, ks.n), place0 = place_of(a, tile.first, qs.n, ks.n), places = a.newest ? 1 : kX;      // of queries' owners
    float lse = 0.f, delta = 0.f;      // negative
    if (!kKeys && x < xs.n) {
      lse = -a.lse[head * q_rows + q_flat + x];
      delta = -a.delta[head * q_rows + q_flat + x];
    }
    int y0 = lo, h = kKeys ? head * R : head;
    bool ok = true;
    for (int it = 0; it < steps; ++it) {
      const float slope2 = kBias ? a.slopes[h] * kLog2e : 0.f;
      const float *lse_y = sh.vec[it & 1][0] + c0, *delta_y = sh.vec[it & 1][1] + c0;
      const bool any = y0 + c0 < hi;                       // columns of this thread's
      const bool masked = kKeys ? y0 + c0 < all_lo || y0 + c0 + kPart > all_hi : y0 + c0 + kPart > all_hi;
      const int meets = meet - y0 - c0, ends = (kKeys ? hi : meet) - y0 - c0;
      if (kKeys) ok = ok && mbar_wait_warp(smem_u32(&sh.vec_full[it & 1]), (it >> 1) & 1, s_abort);
      ok = ok && mbar_wait_warp(smem_u32(&sh.score), it & 1, s_abort);
      if (!ok) { *s_abort = 1; break; }
      tc_fence_after();
      float2 s[kPart / 2];
      uint32_t w[kPart / 2];
      float4 y4;
      if (any) {
        tmem_ld32_nowait(tm, reinterpret_cast<uint32_t*>(s));
        tmem_ld_wait();
      }
      if (!kKeys) {      // the next scores need not wait for what is made of these
        tc_fence_before();
        mbar_arrive(smem_u32(&sh.read));
      }
      if (any) {
        bool near = true;
        if (kCap) {
          // which tanh it is goes by scores that are seen, not by what else the columns hold
          float far[2] = {0.f, 0.f};
          if (masked) {
#pragma unroll
            for (int i = 0; i < kPart / 2; ++i) {
              if (kKeys ? 2 * i < meets || 2 * i >= ends : 2 * i >= ends) s[i].x = 0.f;
              if (kKeys ? 2 * i + 1 < meets || 2 * i + 1 >= ends : 2 * i + 1 >= ends) s[i].y = 0.f;
            }
          }
#pragma unroll
          for (int e = 0; e < kPart / 2; ++e) {
            s[e] = mul2(s[e], both(c));
            far[e & 1] = max3(far[e & 1], fabsf(s[e].x), fabsf(s[e].y));
          }
          near = __all_sync(0xffffffffu, x >= xs.n || fmaxf(far[0], far[1]) <= 1.f);
        }
        // the distance of columns from a row is linear where all lie on one side
        const float from = (float)(!kKeys ? place - y0 - c0 : a.newest ? ks.n - 1 - x : y0 + c0 + shift - x), per = !kKeys ? -1.f : a.newest ? 0.f : 1.f;
        const bool one_side = kBias && (kKeys ? a.newest || y0 + c0 + shift >= tile.first + kX || y0 + c0 + kPart + shift <= tile.first
                                              : place0 >= y0 + c0 + kPart || place0 + places <= y0 + c0);
        const float2 tilt = both(from + per > 0.f ? -slope2 : slope2);
#pragma unroll
        for (int i = 0; i < kPart / 2; ++i) {
          if (kKeys && i % 2 == 0) y4 = *reinterpret_cast<const float4*>(lse_y + 2 * i);
          const float2 ls = !kKeys ? both(lse) : i % 2 == 0 ? make_float2(y4.x, y4.y) : make_float2(y4.z, y4.w);
          float2 arg, slope;
          if (kCap) {
            const float2 th = near ? tanh_small(s[i]) : tanh_any<kCap>(s[i]);
            arg = fma2(th, both(cap2), ls);
            slope = fma2(mul2(th, both(-1.f)), th, both(1.f));
          } else {
            arg = fma2(s[i], both(c), ls);
          }
          if (kBias) {
            const float2 away = make_float2(from + per * (float)(2 * i), from + per * (float)(2 * i + 1));
            if (one_side) arg = fma2(away, tilt, arg);
            else arg = make_float2(fmaf(-slope2, fabsf(away.x), arg.x), fmaf(-slope2, fabsf(away.y), arg.y));
          }
          float2 p = make_float2(ex2(arg.x), ex2(arg.y));
          if (masked) {
            if (kKeys ? 2 * i < meets || 2 * i >= ends : 2 * i >= ends) p.x = 0.f;
            if (kKeys ? 2 * i + 1 < meets || 2 * i + 1 >= ends : 2 * i + 1 >= ends) p.y = 0.f;
          }
          if (kKeys) w[i] = pack_bf16(p.x, p.y);
          s[i] = kCap ? mul2(p, slope) : p;
        }
      }
      if (kKeys) {
        if (any) {
          tmem_st16(tm, w);
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(smem_u32(&sh.weight));
      }
      ok = ok && mbar_wait_warp(smem_u32(&sh.dp), it & 1, s_abort);
      if (!ok) { *s_abort = 1; break; }
      tc_fence_after();
      if (any) {
        float2 d[kPart / 2];
        tmem_ld32_nowait(tm + Shape::dp_col, reinterpret_cast<uint32_t*>(d));
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < kPart / 2; ++i) {
          if (kKeys && i % 2 == 0) y4 = *reinterpret_cast<const float4*>(delta_y + 2 * i);
          const float2 de = !kKeys ? both(delta) : i % 2 == 0 ? make_float2(y4.x, y4.y) : make_float2(y4.z, y4.w);
          float2 ds = mul2(s[i], add2(d[i], de));
          if (masked) {                         // (what dp is made of there may be anything)
            if (kKeys ? 2 * i < meets || 2 * i >= ends : 2 * i >= ends) ds.x = 0.f;
            if (kKeys ? 2 * i + 1 < meets || 2 * i + 1 >= ends : 2 * i + 1 >= ends) ds.y = 0.f;
          }
          w[i] = pack_bf16(ds.x, ds.y);
          if (kSplit) s[i] = ds;
        }
        tmem_st16(tm + Shape::dp_col, w);
        if (kSplit) {
#pragma unroll
          for (int i = 0; i < kPart / 2; ++i)
            w[i] = pack_bf16(s[i].x - __uint_as_float(w[i] << 16), s[i].y - __uint_as_float(w[i] & 0xffff0000u));
          tmem_st16(tm + Shape::dp_col + kPart / 2, w);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(smem_u32(&sh.ds[it & 1]));
      y0 += kY;
      if (kKeys && y0 >= hi) { y0 = lo; ++h; }
    }
    if (ok) {
      ok = mbar_wait_warp(smem_u32(&sh.acc), 0, s_abort);
      if (!ok) *s_abort = 1;
      tc_fence_after();
    }
    if (ok) {
      // each warpgroup stores some columns of a result
      const bool mine = r < tile_rows, some = x < xs.n;
      const long long row = tile.rows.first + x;
      const uint32_t acc = tm_row + Shape::acc_col;
      const int group = warp >> 2;
      auto store = [&](uint32_t tm_acc, float w, const AttnOperand& to, int of, int n) {
        const int per = (d16 / 16 + n - 1) / n * 16;
        store_acc(tm_acc, of * per, min(a.D, (of + 1) * per), a.D, mine, some, w, at_out(to, tile.rows.b, row, head));
      };
      if (!kKeys) store(acc, a.scale, a.gq, group, kParts);
      else if (group < kParts / 2) store(acc, a.scale, a.gk, group, kParts / 2);
      else store(acc + kD, 1.f, a.gv, group - kParts / 2, kParts / 2);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*s_abort) {
    if (threadIdx.x == 0) set_status(a.status, kMbarTimeout, kKeys ? 41 : 42, (int)blockIdx.x);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);        // copies in flight land
    __syncthreads();
  }
  if (warp == 0) tmem_dealloc<Shape::tmem_cols>(tmem);
}

// The first key_tiles * G blocks own keys, the others queries.  Early keys are seen by the most queries and late queries see the most
// keys: those go first.
template <int kD, Cap kCap, bool kBias, bool kSplit>
__global__ void __launch_bounds__(BwdShape<kD>::threads, kD == 128 ? 1 : 2)
attention_bwd_tc_kernel(const __grid_constant__ BwdMaps maps, const __grid_constant__ AttnArgs a, int key_tiles, int query_tiles) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ BwdShared<kD> sh;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int at = blockIdx.x;
  if (at < key_tiles * a.G)
    bwd_block<kD, true, kCap, kBias, kSplit>(maps, a, sh, smem_raw, at / a.G, at % a.G);
  else
    bwd_block<kD, false, kCap, kBias, kSplit>(maps, a, sh, smem_raw, query_tiles - 1 - (at - key_tiles * a.G) / a.H, (at - key_tiles * a.G) % a.H);
}

// delta[h][row] = sum over the columns of do (o + rest); `lanes` threads, a power of two, per row of a head
__global__ void __launch_bounds__(256) attention_delta_kernel(const AttnArgs a, long long rows, int lanes) {
  pdl_sync();
  const long long at_row = ((long long)blockIdx.x * 256 + threadIdx.x) / lanes;
  const int lane = threadIdx.x % lanes;
  float v = 0.f;
  const long long row = at_row / a.H;
  const int h = (int)(at_row % a.H);
  if (row < rows && lane * 8 < a.D) {
    const int b = a.rq.off ? 0 : (int)(row / a.rq.T);
    const long long t = a.rq.off ? row : row % a.rq.T;
    const uint4 x = *reinterpret_cast<const uint4*>(at(a.go, b, t, h) + lane * 8), y = *reinterpret_cast<const uint4*>(at(a.o, b, t, h) + lane * 8);
    const uint4 z = *reinterpret_cast<const uint4*>(at(a.rest, b, t, h) + lane * 8);
    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v += __uint_as_float(xw[i] << 16) * (__uint_as_float(yw[i] << 16) + __uint_as_float(zw[i] << 16)) +
           __uint_as_float(xw[i] & 0xffff0000u) * (__uint_as_float(yw[i] & 0xffff0000u) + __uint_as_float(zw[i] & 0xffff0000u));
  }
  for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (row < rows && lane == 0) a.delta[h * rows + row] = v;
}

template <int kD, Cap kCap, bool kBias, bool kSplit>
cudaError_t launch(const BwdMaps& maps, const AttnArgs& a, cudaStream_t st) {
  auto* k = attention_bwd_tc_kernel<kD, kCap, kBias, kSplit>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdShape<kD>::smem);      // of the current device
  if (e != cudaSuccess) return e;
  const long long kt = tile_count(a.rk, a.B, kX), qt = tile_count(a.rq, a.B, kX);
  if (kt * a.G + qt * a.H >= (1LL << 31)) return cudaErrorInvalidConfiguration;
  return launch_pdl(k, dim3((unsigned)(kt * a.G + qt * a.H)), dim3(BwdShape<kD>::threads), BwdShape<kD>::smem, st, maps, a, (int)kt, (int)qt);
}
template <int kD, bool kSplit>
cudaError_t launch(const BwdMaps& maps, const AttnArgs& a, cudaStream_t st) {
  return with_cap(a, [&](auto cap) {
    return a.slopes ? launch<kD, decltype(cap)::value, true, kSplit>(maps, a, st) : launch<kD, decltype(cap)::value, false, kSplit>(maps, a, st);
  });
}

}  // namespace

const char* launch_attention_bwd(const AttnArgs& a, cudaStream_t st) {
  const long long rows = a.rq.off ? a.rq.T : (long long)a.B * a.rq.T;
  int lanes = 1;
  while (lanes * 8 < a.D) lanes <<= 1;
  cudaError_t e = launch_pdl(attention_delta_kernel, dim3((unsigned)((rows * a.H * lanes + 255) / 256)), dim3(256), 0, st, a, rows, lanes);
  if (e == cudaSuccess && attention_short_takes(a, true)) return launch_attention_short_bwd(a, st);
  BwdMaps maps;
  const int box = a.D > 64 ? BwdShape<128>::y : BwdShape<64>::y;
  if (!operand_map(a.q, a.D, a.rq, a.B, a.H, box, &maps.q) || !operand_map(a.k, a.D, a.rk, a.B, a.G, box, &maps.k) ||
      !operand_map(a.v, a.D, a.rk, a.B, a.G, box, &maps.v) || !operand_map(a.go, a.D, a.rq, a.B, a.H, box, &maps.go))
    return "attention: cuTensorMapEncodeTiled failed";
  const bool split = a.D < 32 || (mean_length(a.rq, a.B) <= 128 && mean_length(a.rk, a.B) <= 128);
  if (e == cudaSuccess)
    e = a.D > 64 ? (split ? launch<128, true>(maps, a, st) : launch<128, false>(maps, a, st))
                 : (split ? launch<64, true>(maps, a, st) : launch<64, false>(maps, a, st));
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace tn
