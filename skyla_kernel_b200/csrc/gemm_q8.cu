// The matrix product of two sets of 8-bit rows (q8.cuh) on the tensor cores: tokens x [M, K] and a weight
// W [N, K] (rows are outputs), both K-major, each row with a scale of its own.
//   acc[t, f] = sum_k x[t, k] W[f, k]   tcgen05.mma kind::i8, 32-bit integers in TMEM: exact in every order, so
//                                       how a product is cut never shows in its result
//   v = acc * x_scale[t] * w_scale[f]   y = v, y += v, or y = silu(v of the gate) * v of the up
// Three kernels; a K block is 128 bytes, one swizzle row, here 128 elements, and an instruction takes 32 of them:
//   q8_rows_kernel   few tokens: the weight streams through every SM once; the weight's rows are the MMA's 128 rows
//                    and the tokens its columns;
//   q8_tile_kernel   tiles of 128 tokens: the tokens are the MMA's rows, so that a thread of the epilogue owns a
//                    token's row;
//   q8_pair_kernel   tiles of 256 tokens on two SMs, where there are many.
// plan() chooses by what they were measured to take.
// Every mbarrier wait is bounded: on a timeout the block records an error code (1 a stage to load into, 2 a stage loaded,
// 3 an accumulator finished, 5 one drained, 7 and 8 a cluster's exchange arrived and sent), lets the loads it issued
// land, frees its TMEM and returns.
#include <cuda.h>

#include <atomic>
#include <cstring>

#include "q8.cuh"
#include "tc_common.cuh"
using namespace skyla;
SKYLA_EXPORT_ERROR_MESSAGE()

namespace {
using namespace skyla::tc;
using skyla::q8::scaled;
using skyla::q8::silu_times;

enum Mode : int { kStoreBf16 = 0, kStoreF32 = 1, kAccumF32 = 2, kGluBf16 = 3 };

constexpr int BM = 128;      // rows of an MMA
constexpr int KB = 128;      // bytes, and elements, of a K block
constexpr int kThreads = 192;
constexpr int kMaxWidth = 131071;  // products of at most 2^14 whose sums stay within 32 bits

struct Args {
  void* y; int64_t ldy;
  int M, N, K;
  const float* x_scale; const float* w_scale;  // [M], [N] (2N gated)
  int* error_flag;
};

__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// D 32-bit integers, A and B signed 8-bit, both K-major, N columns, M = 128
__device__ __forceinline__ uint32_t idesc_i8(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
// The 128 threads of the epilogue meet and agree: whether all of them say so.  (A wait that gave up in one warp and
// not in another must not leave the others at a barrier.)
__device__ __forceinline__ bool all_agree(bool mine) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r) : "r"((uint32_t)mine) : "memory");
  return r != 0;
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&p);
}

// ---------------------------------------------------------------------------------- few tokens: weight streaming
// The structure of the bfloat16 kernel of the same kind (gemm_tc.cu, where its measurements stand): one box brings
// `kkb` K blocks of a tile of R weight rows; tiles are cut so that every SM streams; short tiles stack `kstack` K
// blocks into one MMA, whose diagonal blocks are the partial sums; from 17 tokens on K is cut into a thread-block
// cluster whose blocks exchange their tiles by bulk copies through distributed shared memory.
// Bound by the memory, and for small weights by a launch's start and end: 8 tokens x 4,096 to 2 x 12,288 in 18.3 us (5.5 TB/s
// of weight), 64 x 12,288 to 4,096, added, in 13.2 (3.8 TB/s), 1 x 4,096 to 6,144 in 8.0 (3.1 TB/s).
constexpr int kRowsMaxStages = 24;
constexpr int kRowsSmemBytes = 212 * 1024;

struct RowsArgs {
  int rows_per_block, n_stages, kkb, kstack, tmem_cols;
  int kb_per_split;
};

enum RowsKind : int { kPlain = 0, kCluster = 1, kStacked = 2 };
template <int BN, int MODE, int KIND>
__global__ void __launch_bounds__(kThreads, 1)
q8_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Args a,
               const RowsArgs ra) {
  constexpr int kATiles = MODE == kGluBf16 ? 2 : 1;
  constexpr int kBBytes = BN * KB;
  constexpr bool clustered = KIND == kCluster;
  constexpr bool stacked = KIND == kStacked;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t tmem_base_slot;
  __shared__ volatile int abort_flag;
  __shared__ float tok_scale[BN];

  const int n_stages = ra.n_stages, kkb = ra.kkb, R = ra.rows_per_block;
  const int a_tile = R * KB;  // R rows of 128 bytes: a multiple of 1024
  const uint32_t stage_bytes = (uint32_t)(kkb * (kATiles * a_tile + kBBytes));
  const uint32_t bars = (smem_u32(smem_raw) + 15u) & ~15u;
  const uint32_t base = (bars + 8u * (2 * kRowsMaxStages + 3) + 1023u) & ~1023u;
  const uint32_t landing = base + (uint32_t)n_stages * stage_bytes;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kRowsMaxStages + s); };
  const uint32_t tmem_full_bar = bars + 8u * (2 * kRowsMaxStages);
  const uint32_t land_bar = bars + 8u * (2 * kRowsMaxStages + 1);
  const uint32_t sent_bar = bars + 8u * (2 * kRowsMaxStages + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int f0 = blockIdx.x * R;
  const int total_kb = (a.K + KB - 1) / KB;
  const int kb0 = blockIdx.z * ra.kb_per_split;
  const int n_kb = max(0, min(ra.kb_per_split, total_kb - kb0));
  const int n_st = (n_kb + kkb - 1) / kkb;
  // every block walks its stages from a start of its own, so that the blocks read different lines of the tokens' rows
  const int st_start = n_st > 0 ? (int)(((unsigned)blockIdx.x * 5u) % (unsigned)n_st) : 0;
  auto st_of = [&](int i) { int t = i + st_start; return t >= n_st ? t - n_st : t; };
  const uint32_t tx_bytes = (uint32_t)(kkb * kATiles * a_tile) + (uint32_t)(kkb * kBBytes);

  auto load_weights = [&](int i, int s) {
    const uint32_t sa = base + s * stage_bytes;
    const int kb = kb0 + st_of(i) * kkb;
    mbar_expect_tx(full_bar(s), tx_bytes);
    if (kkb == 1) {
      tma_load_2d(sa, &map_w, full_bar(s), kb * KB, f0);
      if (MODE == kGluBf16) tma_load_2d(sa + a_tile, &map_w, full_bar(s), kb * KB, a.N + f0);
    } else {
      tma_load_3d(sa, &map_w, full_bar(s), 0, f0, kb);
      if (MODE == kGluBf16) tma_load_3d(sa + kkb * a_tile, &map_w, full_bar(s), 0, a.N + f0, kb);
    }
  };
  uint32_t my_rank = 0, n_ranks = 1;
  if (clustered) {
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(my_rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n_ranks));
  }
  // K splits as a cluster: rank r owns the tokens [r * per, r * per + per) of the tile
  const int per = (a.M + (int)n_ranks - 1) / (int)n_ranks;
  const int owners = (a.M + per - 1) / per;
  const int n_dst = owners - ((int)my_rank < owners ? 1 : 0);  // peers that this block sends tokens to
  const int n_pre = min(n_st, n_stages);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < n_stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(tmem_full_bar, 1);
    mbar_init(land_bar, 1);
    mbar_init(sent_bar, n_dst > 0 ? n_dst : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    // weights are finished before any launch that reads them (the caller's weight object waits for them), so the
    // ring's first filling is asked for at once
    for (int i = 0; i < n_pre; ++i) load_weights(i, i);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_slot)), "r"((uint32_t)ra.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_base_slot;
  allow_dependents();
  // nobody may send into a peer's landing zone before that peer's barrier exists: all arrive here, senders wait later
  if (clustered) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  bool met_cluster = false;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      auto load_tokens = [&](int i, int s) {
        const uint32_t sb = base + s * stage_bytes + kkb * kATiles * a_tile;
        const int kb = kb0 + st_of(i) * kkb;
        if (kkb == 1) tma_load_2d(sb, &map_x, full_bar(s), kb * KB, 0);
        else tma_load_3d(sb, &map_x, full_bar(s), 0, 0, kb);
      };
      grid_dependency_wait();
      for (int i = 0; i < n_pre; ++i) load_tokens(i, i);
      int i = n_pre, s = 0;
      uint32_t phase = 1;
      for (; i < n_st; ++i) {
        if (!mbar_wait(empty_bar(s), phase ^ 1, &abort_flag, a.error_flag, 1)) break;
        load_weights(i, s);
        load_tokens(i, s);
        if (++s == n_stages) { s = 0; phase ^= 1; }
      }
      if (i < n_st) {  // gave up: let the loads in flight land before the block's memory goes away
        for (int j = max(0, i - n_stages); j < i; ++j) {
          const long long t0 = clock64();
          while (!mbar_try_wait(full_bar(j % n_stages), (j / n_stages) & 1) && clock64() - t0 < kWaitCycles) {}
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const int kstack = stacked ? ra.kstack : 1;
      const uint32_t idesc = idesc_i8(kstack * BN);
      int s = 0;
      uint32_t phase = 0, started = 0;
      for (int i = 0; i < n_st; ++i) {
        if (!mbar_wait(full_bar(s), phase, &abort_flag, a.error_flag, 2)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t sa = base + s * stage_bytes, sb = sa + kkb * kATiles * a_tile;
        // K blocks past the end of K hold zeros (the loads fill them)
        for (int j = 0; j < kkb; j += kstack) {
          const uint64_t da = umma_desc(sa + j * a_tile), db = umma_desc(sb + j * kBBytes);
          const uint64_t du = umma_desc(sa + (kkb + j) * a_tile);
#pragma unroll
          for (int k = 0; k < KB / 32; ++k) {
            umma_i8(tmem_base, da + 2 * k, db + 2 * k, idesc, started);
            if (MODE == kGluBf16) umma_i8(tmem_base + BN, du + 2 * k, db + 2 * k, idesc, started);
            started = 1u;
          }
        }
        umma_commit(empty_bar(s));
        if (++s == n_stages) { s = 0; phase ^= 1; }
      }
      umma_commit(tmem_full_bar);
    }
  } else {
    // ------------------------------------------------------------ epilogue warps
    const int quad = warp & 3;
    const int r_local = quad * 32 + lane;  // row of the tile that this thread's TMEM lane holds
    const int f = f0 + r_local;
    const bool mine = r_local < R && f < a.N;
    const int et = threadIdx.x - 64;
    // what does not depend on the product is fetched while the main loop runs
    const float ws = mine ? a.w_scale[f] : 0.f;
    const float us = MODE == kGluBf16 && mine ? a.w_scale[a.N + f] : 0.f;
    grid_dependency_wait();
    for (int t = et; t < BN; t += 128) tok_scale[t] = t < a.M ? a.x_scale[t] : 0.f;
    const int kstack = stacked ? ra.kstack : 1;
    int* red = reinterpret_cast<int*>(smem_raw + (landing - smem_u32(smem_raw)));
    float old_pre[4] = {0.f, 0.f, 0.f, 0.f}, old16[16];
    if (MODE == kAccumF32 && stacked) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int idx = et + 128 * n;
        const int tok = idx / R, ff = f0 + idx - tok * R;
        if (idx < a.M * R && ff < a.N) old_pre[n] = ((const float*)a.y)[(int64_t)tok * a.ldy + ff];
      }
    }
    if (MODE == kAccumF32 && KIND == kPlain && mine) {
#pragma unroll
      for (int j = 0; j < 16; ++j) old16[j] = j < a.M ? ((const float*)a.y)[(int64_t)j * a.ldy + f] : 0.f;
    }
    const int my_n = max(0, min(per, a.M - (int)my_rank * per));
    constexpr uint32_t kRowBytes = BM * 4;  // a token's 128 outputs of the tile
    // in a cluster's owner a warp takes every fourth token and a lane four neighbouring outputs of the tile
    const int f4 = f0 + 4 * lane;
    const bool mine4 = 4 * lane < R && f4 < a.N;  // (R and N are multiples of 4 there)
    float4 old4[4], ws4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (clustered) {
      if (et == 0 && my_n > 0) mbar_expect_tx(land_bar, (n_ranks - 1) * (uint32_t)my_n * kRowBytes);
      if (mine4) ws4 = make_float4(a.w_scale[f4], a.w_scale[f4 + 1], a.w_scale[f4 + 2], a.w_scale[f4 + 3]);
      if (MODE == kAccumF32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = quad + 4 * j;
          old4[j] = (mine4 && i < my_n) ? *reinterpret_cast<const float4*>((const float*)a.y + (int64_t)((int)my_rank * per + i) * a.ldy + f4)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
    }
    asm volatile("barrier.sync 1, 128;" ::: "memory");  // the tokens' scales
    const bool ok = n_kb > 0 && mbar_wait(tmem_full_bar, 0, &abort_flag, a.error_flag, 3);
    if (ok) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16);
    if (clustered) {
      // Every split writes its accumulator, token by token, into shared memory of its own (the ring, idle by now),
      // one region per owner, and sends each region to its owner's landing zone with one bulk copy, which the
      // owner's barrier counts in.  Columns past the last token are written too: nobody reads them.
      const bool warp_reads = ok && quad * 32 < R;  // uniform for the warp
      const uint32_t travel = base + 4u * (uint32_t)r_local;
#pragma unroll 1
      for (int c0 = 0; c0 < BN && warp_reads; c0 += 16) {
        if (c0 >= a.M) break;
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tmem_wait_ld();
        const uint32_t at = travel + (uint32_t)c0 * kRowBytes;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + (uint32_t)j * kRowBytes), "r"(r[j]) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("barrier.sync 1, 128;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // every peer's barrier exists from here on
      met_cluster = true;
      if (et == 0) {
        for (uint32_t d = 1; ok && d < n_ranks; ++d) {
          const uint32_t dst = (my_rank + d) % n_ranks;
          const int dst_n = max(0, min(per, a.M - (int)dst * per));
          if (dst_n == 0) continue;
          uint32_t remote_zone, remote_bar;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote_zone) : "r"(landing + my_rank * (uint32_t)per * kRowBytes), "r"(dst));
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote_bar) : "r"(land_bar), "r"(dst));
          asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(remote_zone), "r"(base + dst * (uint32_t)per * kRowBytes), "r"((uint32_t)dst_n * kRowBytes), "r"(remote_bar)
                       : "memory");
        }
      }
      bool landed = ok;
      if (landed && my_n > 0) landed = mbar_wait(land_bar, 0, &abort_flag, a.error_flag, 7);
      if (et == 32 && landed && my_n > 0) {  // what the peers sent has arrived: they may leave
        for (uint32_t d = 1; d < n_ranks; ++d) {
          uint32_t remote_bar;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote_bar) : "r"(sent_bar), "r"((my_rank + d) % n_ranks));
          asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
        }
      }
      const uint32_t rank_stride = (uint32_t)per * kRowBytes;
      const uint32_t zone = landing + 16u * (uint32_t)lane;                      // [source rank][owned token][output]
      const uint32_t own = base + my_rank * rank_stride + 16u * (uint32_t)lane;  // this block's own share of its tokens
#pragma unroll 1
      for (int j = 0; quad + 4 * j < my_n; ++j) {
        const int i = quad + 4 * j, col = (int)my_rank * per + i;
        if (!landed || !mine4) continue;
        int4 sum = make_int4(0, 0, 0, 0);
        for (uint32_t src = 0; src < n_ranks; ++src) {
          int4 v;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"((src == my_rank ? own : zone + src * rank_stride) + (uint32_t)i * kRowBytes));
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        const float xs = tok_scale[col];
        const float4 v = make_float4(scaled(sum.x, xs, ws4.x), scaled(sum.y, xs, ws4.y), scaled(sum.z, xs, ws4.z), scaled(sum.w, xs, ws4.w));
        if (MODE == kStoreBf16) {
          *reinterpret_cast<uint2*>((__nv_bfloat16*)a.y + (int64_t)col * a.ldy + f4) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        } else if (MODE == kStoreF32) {
          *reinterpret_cast<float4*>((float*)a.y + (int64_t)col * a.ldy + f4) = v;
        } else {
          float* p = (float*)a.y + (int64_t)col * a.ldy + f4;
          const float4 o = j == 0 ? old4[0] : j == 1 ? old4[1] : j == 2 ? old4[2] : j == 3 ? old4[3] : *reinterpret_cast<const float4*>(p);
          *reinterpret_cast<float4*>(p) = make_float4(__fadd_rn(o.x, v.x), __fadd_rn(o.y, v.y), __fadd_rn(o.z, v.z), __fadd_rn(o.w, v.w));
        }
      }
    } else if (stacked) {
      // lane L of the accumulator is row L % R of K-block group L / R; its partial sums are the columns
      // [q * BN, q * BN + BN) of its own group q.  red[(q * BN + tok) * R + r], then a sum over q.
      if (ok) {
        const int L = quad * 32 + lane;
        const int q_mine = L / R, r_mine = L - q_mine * R;
        const int q_lo = (quad * 32) / R, q_hi = min(kstack - 1, (quad * 32 + 31) / R);  // uniform for the warp
        for (int q = q_lo; q <= q_hi; ++q) {
#pragma unroll 1
          for (int c0 = 0; c0 < BN; c0 += 16) {
            if (c0 >= a.M) break;
            uint32_t r[16];
            tmem_ld16(taddr + q * BN + c0, r);
            tmem_wait_ld();
            if (q == q_mine) {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (c0 + j < a.M) red[(q * BN + c0 + j) * R + r_mine] = (int)r[j];
            }
          }
        }
      }
      asm volatile("barrier.sync 1, 128;" ::: "memory");
      const float inv_R = 1.0f / (float)R;
      for (int idx = et; ok && idx < a.M * R; idx += 128) {
        // idx / R without the integer division: (idx + 0.5) / R is at least 1 / (2 R) away from an integer
        const int tok = (int)(((float)idx + 0.5f) * inv_R), rr = idx - tok * R;
        const int ff = f0 + rr;
        if (ff >= a.N) continue;
        int sum = 0;
        for (int q = 0; q < kstack; ++q) sum += red[(q * BN + tok) * R + rr];
        const float v = scaled(sum, tok_scale[tok], a.w_scale[ff]);
        if (MODE == kStoreBf16) ((__nv_bfloat16*)a.y)[(int64_t)tok * a.ldy + ff] = __float2bfloat16_rn(v);
        else if (MODE == kStoreF32) ((float*)a.y)[(int64_t)tok * a.ldy + ff] = v;
        else {
          float* p = (float*)a.y + (int64_t)tok * a.ldy + ff;
          const int n = (idx - et) >> 7;  // which of this thread's items
          *p = __fadd_rn(n == 0 ? old_pre[0] : n == 1 ? old_pre[1] : n == 2 ? old_pre[2] : n == 3 ? old_pre[3] : *p, v);
        }
      }
    } else {
      const bool warp_has_rows = ok && quad * 32 < R;  // uniform for the warp
#pragma unroll 1
      for (int c0 = 0; c0 < BN && warp_has_rows; c0 += 16) {
        if (c0 >= a.M) break;
        uint32_t r[16], u[16];
        __syncwarp();
        tmem_ld16(taddr + c0, r);
        if (MODE == kGluBf16) tmem_ld16(taddr + BN + c0, u);
        tmem_wait_ld();
        if (!mine) continue;
        float old[16];
        if (MODE == kAccumF32) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            old[j] = c0 == 0 ? old16[j] : (c0 + j < a.M ? ((const float*)a.y)[(int64_t)(c0 + j) * a.ldy + f] : 0.f);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int tok = c0 + j;
          if (tok >= a.M) break;
          const float v = scaled((int)r[j], tok_scale[tok], ws);
          if (MODE == kStoreBf16) ((__nv_bfloat16*)a.y)[(int64_t)tok * a.ldy + f] = __float2bfloat16_rn(v);
          else if (MODE == kStoreF32) ((float*)a.y)[(int64_t)tok * a.ldy + f] = v;
          else if (MODE == kAccumF32) ((float*)a.y)[(int64_t)tok * a.ldy + f] = __fadd_rn(old[j], v);
          else ((__nv_bfloat16*)a.y)[(int64_t)tok * a.ldy + f] = __float2bfloat16_rn(silu_times(v, scaled((int)u[j], tok_scale[tok], us)));
        }
      }
    }
  }
  if (clustered) {
    // A block's shared memory has to outlive the copies that read it: it leaves when every peer that it sent to has
    // told it so.  A peer that gave up never tells; the wait is bounded like every other.
    if (!met_cluster) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (threadIdx.x == 64 && n_dst > 0 && !abort_flag) mbar_wait(sent_bar, 0, &abort_flag, a.error_flag, 8);
  }
  // ------------------------------------------------------------------ teardown
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    if (lane == 0 && n_kb > 0) {  // the accumulator must be idle before its columns are freed
      const long long t0 = clock64();
      while (!mbar_try_wait(tmem_full_bar, 0) && clock64() - t0 < kWaitCycles) {}
    }
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)ra.tmem_cols) : "memory");
  }
}

// ---------------------------------------------------------------------------------- many tokens
// One block per SM walks tiles of 128 tokens x BF accumulator columns (a gated weight: BF / 2 gate rows and the BF / 2
// up rows of the same outputs), two accumulators in turn: the epilogue of one tile runs beside the products of the
// next.  warp 0 loads, warp 1 issues, warps 2 to 5 are the epilogue, a thread per token.  32 or 64 outputs of the tile's
// tokens at a time are laid out in one of two 16 KB buffers and leave by a TMA store (or reduce-add: y += v never reads
// y), or, where y's rows do not allow that, row by row in order.
// SPLIT: few tiles; the blocks of a cluster share one tile, each with a run of its K blocks.  They leave their
// accumulators in shared memory (the ring, idle by then), and each finishes an equal part of the outputs, or of the
// tokens, from all of them: whole numbers, so the result does not show the cut.
// 256 tokens x 4,096 to 4,096, added, on 128 blocks of 64 columns: 9.7 us, 6.5 of them 24 KB a K block into an SM (120 GB/s,
// what one takes in); 8,192 x 4,096 to 2 x 12,288 on 256 columns: 518 us (3,180 TOP/s).  Of 2,048 x 4,096 to 6,144 the imma
// pipe takes 72 % of an SM's active cycles, which are 75 % of the time: whole rounds of tiles.
constexpr int kOutBytes = BM * 128;  // 128 tokens x 128 bytes
constexpr int kMaxSplits = 4;

template <int MODE, int BF>
struct TileCfg {
  // K blocks of a stage.  (A TMA load takes its unit about 0.1 us whatever it brings: narrow tiles bring two a load.
  // A gated tile's gate and up rows come by loads of their own and have to lie together for one instruction of BF
  // columns: one K block a stage.  Two, with instructions of half the width: 416 against 344 us for 4,096 tokens.)
  static constexpr int kKkb = BF == 256 || MODE == kGluBf16 ? 1 : 2;
  static constexpr int kXBytes = BM * KB, kWBytes = BF * KB;  // of one K block
  static constexpr int kStageBytes = kKkb * (kXBytes + kWBytes);
  static constexpr int kStagesRaw = (196 * 1024) / kStageBytes;
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;  // 4 for 256 columns, 3 for 128 (gated 6), 4 for 64
  static constexpr int kSmemBytes = kStages * kStageBytes + 2 * kOutBytes + 1024 /*align*/ + 256 /*barriers*/;
  static constexpr int kTmemCols = 2 * BF;
  static_assert(kSmemBytes + BF * 4 + 64 <= 227 * 1024, "shared memory of a block");
  static_assert(kStages * kStageBytes >= BM * BF * 4, "a split's accumulator fits the ring");
};

// 16 bytes at column piece c of a row of 128 bytes, where a 128-byte swizzle puts them: the threads of a warp, a row
// each, then write to different banks
__device__ __forceinline__ void put16(uint32_t row_smem, int row, int c, uint32_t a, uint32_t b, uint32_t d, uint32_t e) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
               ::"r"(row_smem + (uint32_t)((c ^ (row & 7)) << 4)), "r"(a), "r"(b), "r"(d), "r"(e) : "memory");
}

// The epilogue of a tile: the chunks first, first + step, ... of its outputs (32 of 32-bit, 64 of bfloat16), from the
// accumulator's columns as `columns16(column, registers)` brings sixteen of them for this thread's token.
template <int MODE, int BF, typename Columns>
__device__ __forceinline__ void drain(const Args& a, const CUtensorMap* map_y, int by_tma, const float* ws, float xs, int f0, int tok0,
                                      int quad, int lane, bool sender, uint32_t out_smem, int& n_sent, int first, int step,
                                      volatile int& abort_flag, Columns columns16) {
  constexpr int kTileOutputs = MODE == kGluBf16 ? BF / 2 : BF;
  constexpr bool f32 = MODE == kStoreF32 || MODE == kAccumF32;
  constexpr int kCols = f32 ? 32 : (kTileOutputs < 64 ? kTileOutputs : 64);  // outputs of a buffer's rows
  constexpr int kChunks = kTileOutputs / kCols;
  const int row = quad * 32 + lane;
  // 32 columns at a time: values of this thread's token
  auto values = [&](int c0, float* v) {
    uint32_t r[32];
    __syncwarp();
    columns16(c0, r);
    columns16(c0 + 16, r + 16);
    if (MODE == kGluBf16) {
      uint32_t u[32];
      columns16(BF / 2 + c0, u);
      columns16(BF / 2 + c0 + 16, u + 16);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j)
        v[j] = silu_times(scaled((int)r[j], xs, ws[c0 + j]), scaled((int)u[j], xs, ws[BF / 2 + c0 + j]));
    } else {
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = scaled((int)r[j], xs, ws[c0 + j]);
    }
  };
#pragma unroll 1
  for (int chunk = first; chunk < kChunks; chunk += step) {
    const int c0 = chunk * kCols;
    if (f0 + c0 >= a.N) break;  // the same for all four warps
    const uint32_t out = out_smem + (uint32_t)(n_sent & 1) * kOutBytes;
    // who read this buffer last (two chunks ago) must be done with it: the send, or, row by row, the warps, which have
    // met since
    if (by_tma && sender) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    asm volatile("barrier.sync 1, 128;" ::: "memory");
    const uint32_t row_smem = out + (uint32_t)row * 128u;
#pragma unroll
    for (int h = 0; h < kCols / 32; ++h) {
      float v[32];
      values(c0 + 32 * h, v);
      if (f32) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          put16(row_smem, row, c, __float_as_uint(v[4 * c]), __float_as_uint(v[4 * c + 1]), __float_as_uint(v[4 * c + 2]),
                __float_as_uint(v[4 * c + 3]));
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          put16(row_smem, row, 4 * h + c, pack_bf16(v[8 * c], v[8 * c + 1]), pack_bf16(v[8 * c + 2], v[8 * c + 3]),
                pack_bf16(v[8 * c + 4], v[8 * c + 5]), pack_bf16(v[8 * c + 6], v[8 * c + 7]));
      }
    }
    if (by_tma) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the TMA unit reads what the threads wrote
    asm volatile("barrier.sync 1, 128;" ::: "memory");
    if (by_tma) {
      if (sender && !abort_flag) {
        if (MODE == kAccumF32)
          asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
                       ::"l"(map_y), "r"(out), "r"(f0 + c0), "r"(tok0) : "memory");
        else
          asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                       ::"l"(map_y), "r"(out), "r"(f0 + c0), "r"(tok0) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    } else {
      // a warp takes 32 rows, one after the other, its lanes neighbouring outputs.  (Compact code: a launch starts with
      // cold instruction caches.  Eight rows at a time, pairs of bfloat16 in one store: 333 tokens x 2,561 to 1,111 took
      // 10.4 instead of 8.7 us.)
      auto at_row = [&](int r, int c) {
        return out + (uint32_t)r * 128u + (uint32_t)((((c * (f32 ? 4 : 2)) >> 4) ^ (r & 7)) << 4) + (uint32_t)((c * (f32 ? 4 : 2)) & 15);
      };
      if (MODE == kAccumF32) {  // eight old values are on their way together
        const bool live = f0 + c0 + lane < a.N;
        float* y = (float*)a.y + (int64_t)(tok0 + quad * 32) * a.ldy + f0 + c0 + lane;
        const int rows = min(32, a.M - tok0 - quad * 32);
#pragma unroll 1
        for (int i0 = 0; i0 < rows; i0 += 8) {
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = live && i0 + i < rows ? y[(i0 + i) * a.ldy] : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float v;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at_row(quad * 32 + i0 + i, lane)) : "memory");
            if (live && i0 + i < rows) y[(i0 + i) * a.ldy] = __fadd_rn(o[i], v);
          }
        }
      } else {
#pragma unroll 4
        for (int i = 0; i < 32; ++i) {
          const int r = quad * 32 + i;
          if (tok0 + r >= a.M) break;
          const int64_t at = (int64_t)(tok0 + r) * a.ldy + f0 + c0;
#pragma unroll
          for (int h = 0; h < kCols / 32; ++h) {
            const int c = lane + 32 * h;
            if (f0 + c0 + c >= a.N) continue;
            if (f32) {
              float v;
              asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at_row(r, c)) : "memory");
              ((float*)a.y)[at + c] = v;
            } else {
              uint16_t v;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at_row(r, c)) : "memory");
              ((uint16_t*)a.y)[at + c] = v;
            }
          }
        }
      }
    }
    ++n_sent;
  }
}

// The scales of a tile's columns, by the 128 threads of the epilogue.
template <int MODE, int BF>
__device__ __forceinline__ void tile_scales(const Args& a, float* ws, int f0, int et) {
  for (int c = et; c < BF; c += 128) {
    const int f = MODE == kGluBf16 ? f0 + c % (BF / 2) : f0 + c;
    ws[c] = f < a.N ? a.w_scale[MODE == kGluBf16 && c >= BF / 2 ? a.N + f : f] : 0.f;
  }
}

struct TileArgs {
  int by_tma;         // map_y is y's: outputs leave by TMA
  int boxes;          // the maps of x and w bring a stage's K blocks at once (K in whole blocks); else one by one
  int x_rows;         // rows of a box of x: 128, or the tokens of a single tile to the next eight (the MMA then reads what
                      // lies behind them as rows that nobody reads).  Boxes that reach far beyond the tokens are slow.
  int n_t_tiles, n_tiles;
  int splits;         // blocks of a cluster (SPLIT), each with an equal run of the K blocks; else 1
};

// Sixteen columns of a token, summed over the accumulators of a cluster's blocks through distributed shared memory (`mine`:
// where the token's lie in each); the loads of all blocks are in flight together.
__device__ __forceinline__ void split_sum16(uint32_t mine, int splits, int c0, uint32_t* r) {
  uint32_t v[kMaxSplits][16];
#pragma unroll
  for (int q = 0; q < kMaxSplits; ++q) {
    if (q >= splits) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[q][j] = 0;
      continue;
    }
    uint32_t from;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(mine + (uint32_t)(c0 / 4) * (BM * 16u)), "r"((uint32_t)q));
#pragma unroll
    for (int c = 0; c < 4; ++c)
      asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[q][4 * c]), "=r"(v[q][4 * c + 1]),
                   "=r"(v[q][4 * c + 2]), "=r"(v[q][4 * c + 3]) : "r"(from + (uint32_t)c * (BM * 16u)) : "memory");
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) r[j] = v[0][j] + v[1][j] + v[2][j] + v[3][j];
}

// The end of a tile of 64 outputs that four blocks share: each finishes 32 of the tokens, a thread sixteen outputs of one,
// written straight away.  (The blocks taking turns at the columns through drain(), two of the four have nothing to do: 500
// tokens x 16,384 to 512 took 13.0 instead of 11.6 us.  With more outputs a thread, drain()'s order of writing wins: two
// splits of 4,096 to 4,096 at 128 tokens 8.7 against 9.8.)
template <int MODE, int BF>
__device__ __forceinline__ void finish_tokens(const Args& a, const TileArgs& ta, const float* ws, uint32_t ring, int f0, int tok0, int rank,
                                              int et) {
  constexpr bool f32 = MODE == kStoreF32 || MODE == kAccumF32;
  const int row = rank * 32 + et % 32, c0 = et / 32 * 16, tok = tok0 + row;
  const int f = f0 + c0, n = min(16, a.N - f);
  if (tok >= a.M || n <= 0) return;
  const float xs = a.x_scale[tok];
  const uint32_t mine = ring + 16u * (uint32_t)row;
  const bool whole = ta.by_tma && n == 16;  // as vectors: y's rows begin and end on 16 bytes
  float* y32 = (float*)a.y + (int64_t)tok * a.ldy + f;
  __nv_bfloat16* y16 = (__nv_bfloat16*)a.y + (int64_t)tok * a.ldy + f;
  float old[16];
  if (MODE == kAccumF32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 o = whole ? reinterpret_cast<const float4*>(y32)[j]
                             : make_float4(4 * j < n ? y32[4 * j] : 0.f, 4 * j + 1 < n ? y32[4 * j + 1] : 0.f,
                                           4 * j + 2 < n ? y32[4 * j + 2] : 0.f, 4 * j + 3 < n ? y32[4 * j + 3] : 0.f);
      old[4 * j] = o.x; old[4 * j + 1] = o.y; old[4 * j + 2] = o.z; old[4 * j + 3] = o.w;
    }
  }
  uint32_t r[16];
  float v[16];
  split_sum16(mine, 4, c0, r);
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = scaled((int)r[j], xs, ws[c0 + j]);
  if (MODE == kGluBf16) {
    split_sum16(mine, 4, BF / 2 + c0, r);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = silu_times(v[j], scaled((int)r[j], xs, ws[BF / 2 + c0 + j]));
  }
  if (MODE == kAccumF32) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __fadd_rn(old[j], v[j]);
  }
  if (!whole) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < n) {
        if (f32) y32[j] = v[j];
        else y16[j] = __float2bfloat16_rn(v[j]);
      }
  } else if (f32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<float4*>(y32)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      reinterpret_cast<uint4*>(y16)[j] = make_uint4(pack_bf16(v[8 * j], v[8 * j + 1]), pack_bf16(v[8 * j + 2], v[8 * j + 3]),
                                                    pack_bf16(v[8 * j + 4], v[8 * j + 5]), pack_bf16(v[8 * j + 6], v[8 * j + 7]));
  }
}

template <int MODE, int BF, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
q8_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
               const __grid_constant__ CUtensorMap map_y, const Args a, const TileArgs ta) {
  using C = TileCfg<MODE, BF>;
  constexpr int kStages = C::kStages;
  constexpr int kTileOutputs = MODE == kGluBf16 ? BF / 2 : BF;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t tmem_base_slot;
  __shared__ volatile int abort_flag;
  __shared__ __align__(16) float ws[BF];  // the scales of the tile's columns
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t out_smem = base + kStages * C::kStageBytes;
  const uint32_t bars = out_smem + 2 * kOutBytes;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kStages + s); };
  auto acc_full_bar = [&](int b) { return bars + 8u * (2 * kStages + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * kStages + 2 + b); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total_kb = (a.K + KB - 1) / KB;
  // the tiles of this block: first, first + step, ... ; a split's block has one
  const int rank = SPLIT ? (int)blockIdx.x % ta.splits : 0;
  const int first = SPLIT ? (int)blockIdx.x / ta.splits : (int)blockIdx.x;
  const int step = SPLIT ? ta.n_tiles : (int)gridDim.x;
  const int kb_lo = SPLIT ? rank * total_kb / ta.splits : 0;  // (at most 3 x 1,024)
  const int kb_hi = SPLIT ? (rank + 1) * total_kb / ta.splits : total_kb;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);
      mbar_init(acc_empty_bar(b), 4);  // one arrival per epilogue warp
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_slot)), "r"((uint32_t)C::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_base_slot;
  allow_dependents();

  constexpr int kKkb = C::kKkb;
  const int n_st = (kb_hi - kb_lo + kKkb - 1) / kKkb;  // stages of a tile
  const int x_bytes = ta.x_rows * KB;                  // of a K block: a multiple of 1024

  if (warp == 0) {
    if (lane == 0) {
      uint32_t armed = 0, armed_parity = 0;
      int stg = 0;
      bool ok = true, waited = false;
      for (int tile = first; ok && tile < ta.n_tiles; tile += step) {
        const int f_tile = tile / ta.n_t_tiles, t_tile = tile % ta.n_t_tiles;
        const int row0 = f_tile * kTileOutputs;
        // (blocks past the end of K, or of this split, are loaded as what lies there, zeros past the end, and not used)
        auto load_weights = [&](int i, int s) {
          const int kb = kb_lo + i * kKkb;
          const uint32_t sw = base + s * C::kStageBytes + kKkb * C::kXBytes;
          mbar_expect_tx(full_bar(s), (uint32_t)(kKkb * (x_bytes + C::kWBytes)));
          if (MODE == kGluBf16) {
            tma_load_2d(sw, &map_w, full_bar(s), kb * KB, row0);
            tma_load_2d(sw + C::kWBytes / 2, &map_w, full_bar(s), kb * KB, a.N + row0);
          } else if (kKkb > 1 && ta.boxes) {
            tma_load_3d(sw, &map_w, full_bar(s), 0, row0, kb);
          } else {
#pragma unroll
            for (int j = 0; j < kKkb; ++j) tma_load_2d(sw + j * C::kWBytes, &map_w, full_bar(s), (kb + j) * KB, row0);
          }
        };
        // weights are finished before any launch that reads them: the ring's first filling of them is asked for
        // before this grid waits for the one ahead of it
        const int n_pre = waited ? 0 : min(kStages, n_st);
        for (int i = 0; i < n_pre; ++i) load_weights(i, i);
        if (!waited) grid_dependency_wait();
        waited = true;
        for (int i = 0; i < n_st; ++i, ++stg) {
          const int s = stg % kStages;
          const uint32_t phase = (stg / kStages) & 1;
          if (stg >= n_pre) {
            if (!mbar_wait(empty_bar(s), phase ^ 1, &abort_flag, a.error_flag, 1)) { ok = false; break; }
            load_weights(i, s);
          }
          const uint32_t sx = base + s * C::kStageBytes;
          const int kb = kb_lo + i * kKkb;
          if (kKkb > 1 && ta.boxes) {
            tma_load_3d(sx, &map_x, full_bar(s), 0, t_tile * BM, kb);
          } else {
#pragma unroll
            for (int j = 0; j < kKkb; ++j) tma_load_2d(sx + j * x_bytes, &map_x, full_bar(s), (kb + j) * KB, t_tile * BM);
          }
          armed |= 1u << s;
          armed_parity = (armed_parity & ~(1u << s)) | (phase << s);
        }
      }
      if (!ok)  // gave up: let the loads already issued land before the block's memory goes away
        for (int s = 0; s < kStages; ++s)
          if (armed & (1u << s)) {
            const long long t0 = clock64();
            while (!mbar_try_wait(full_bar(s), (armed_parity >> s) & 1) && clock64() - t0 < kWaitCycles) {}
          }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_i8(BF);
      int stg = 0, it = 0;
      bool ok = true;
      for (int tile = first; ok && tile < ta.n_tiles; tile += step, ++it) {
        const int buf = it & 1;
        // the epilogue must have drained this accumulator (two tiles ago)
        if (!mbar_wait(acc_empty_bar(buf), ((it >> 1) & 1) ^ 1, &abort_flag, a.error_flag, 5)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem_base + buf * BF;
        uint32_t started = 0;
        for (int i = 0; i < n_st; ++i, ++stg) {
          const int s = stg % kStages;
          const uint32_t phase = (stg / kStages) & 1;
          if (!mbar_wait(full_bar(s), phase, &abort_flag, a.error_flag, 2)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sx = base + s * C::kStageBytes, sw = sx + kKkb * C::kXBytes;
#pragma unroll
          for (int j = 0; j < kKkb; ++j) {
            if (kb_lo + i * kKkb + j >= kb_hi) break;
            const uint64_t dx = umma_desc(sx + j * x_bytes), dw = umma_desc(sw + j * C::kWBytes);
#pragma unroll
            for (int k = 0; k < KB / 32; ++k) {
              umma_i8(d, dx + 2 * k, dw + 2 * k, idesc, started);
              started = 1u;
            }
          }
          umma_commit(empty_bar(s));
        }
        umma_commit(acc_full_bar(buf));
      }
    }
  } else {
    const int quad = warp & 3, row = quad * 32 + lane, et = threadIdx.x - 64;
    const bool sender = warp == 2 && lane == 0;
    int n_sent = 0, it = 0;
    bool waited = false;
    for (int tile = first; tile < ta.n_tiles; tile += step, ++it) {
      const int buf = it & 1;
      const int f_tile = tile / ta.n_t_tiles, t_tile = tile % ta.n_t_tiles;
      const int tok0 = t_tile * BM, tok = tok0 + row, f0 = f_tile * kTileOutputs;
      asm volatile("barrier.sync 1, 128;" ::: "memory");  // the last tile's scales have been read
      tile_scales<MODE, BF>(a, ws, f0, et);
      if (!waited) grid_dependency_wait();
      waited = true;
      const float xs = tok < a.M ? a.x_scale[tok] : 0.f;
      const bool ok = all_agree(mbar_wait(acc_full_bar(buf), (it >> 1) & 1, &abort_flag, a.error_flag, 3));
      if (!SPLIT && !ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t taddr = tmem_base + buf * BF + ((uint32_t)(quad * 32) << 16);
      if constexpr (SPLIT) {
        // the ring as a split leaves its accumulator there: [piece of four columns][row], a warp's rows 512 bytes in a row
        if (ok) {
          const uint32_t left = base + 16u * (uint32_t)row;
#pragma unroll 1
          for (int c0 = 0; c0 < BF; c0 += 32) {
            uint32_t r[32];
            __syncwarp();
            tmem_ld16(taddr + c0, r);
            tmem_ld16(taddr + c0 + 16, r + 16);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 8; ++c)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                           ::"r"(left + (uint32_t)(c0 / 4 + c) * (BM * 16u)), "r"(r[4 * c]), "r"(r[4 * c + 1]), "r"(r[4 * c + 2]),
                             "r"(r[4 * c + 3]) : "memory");
          }
        }
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (kTileOutputs == 64 && ta.splits == 4)
          finish_tokens<MODE, BF>(a, ta, ws, base, f0, tok0, rank, et);
        else
          drain<MODE, BF>(a, &map_y, ta.by_tma, ws, xs, f0, tok0, quad, lane, sender, out_smem, n_sent, rank, ta.splits, abort_flag,
                          [&](int c0, uint32_t* r) { split_sum16(base + 16u * (uint32_t)row, ta.splits, c0, r); });
      } else {
        drain<MODE, BF>(a, &map_y, ta.by_tma, ws, xs, f0, tok0, quad, lane, sender, out_smem, n_sent, 0, 1, abort_flag,
                        [&](int c0, uint32_t* r) { tmem_ld16(taddr + c0, r); });
      }
      // this warp has read its lanes of the accumulator: hand it back to the MMA warp
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty_bar(buf));
    }
    if (ta.by_tma && sender) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the buffers go away with the block
  }
  if (SPLIT) {
    // two meetings of all threads of the cluster: every accumulator lies in its ring; all have read them.  (The
    // epilogue's warps took the first one above.)
    if (warp < 2) {
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    if (lane == 0) {  // every accumulator must be idle before its columns are freed
      const int my_tiles = first < ta.n_tiles ? (ta.n_tiles - first + step - 1) / step : 0;
      for (int b = 0; b < 2; ++b) {
        const int uses = (my_tiles + 1 - b) / 2;  // tiles that used accumulator b
        if (uses > 0) {
          const long long t0 = clock64();
          while (!mbar_try_wait(acc_full_bar(b), (uses - 1) & 1) && clock64() - t0 < kWaitCycles) {}
        }
      }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)C::kTmemCols) : "memory");
  }
}

// ---------------------------------------------------------------------------------- many tokens, two SMs a tile
// The same work for products of many tiles: a cluster of two blocks takes tiles of 256 tokens x 256 columns with
// tcgen05's cta_group::2.  Each block holds its 128 tokens and HALF of the columns' weight rows (a gated weight: the
// first block the gate rows, the second the up rows); the instruction, issued by the first block, reads both blocks'
// shared memory and leaves each block its own tokens' accumulator.  So a K block brings 32 KB into an SM where
// q8_tile_kernel brings 48: 8,192 tokens x 4,096 to 2 x 12,288 in 468 us (3,530 TOP/s), 554 at the power limit (tiles of one
// SM: 518 and 628); 2,048 x 4,096 to 6,144 in 35.4 (38.5), which are 2.6 rounds of 74 pairs.  Both blocks' loads count into the first block's barrier; its commits free the stage, and
// hand over the accumulator, in both.
constexpr int kPairStageBytes = 2 * BM * KB;  // 128 tokens and 128 weight rows
constexpr int kPairStages = 6;
constexpr int kPairSmemBytes = kPairStages * kPairStageBytes + 2 * kOutBytes + 1024 + 256;
static_assert(kPairSmemBytes + 256 * 4 + 64 <= 227 * 1024, "shared memory of a block");

__device__ __forceinline__ uint32_t on_first(uint32_t addr) {  // the same place in the cluster's first block
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {  // to the barrier at this place in both blocks
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((uint16_t)3) : "memory");
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
q8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
               const __grid_constant__ CUtensorMap map_y, const Args a, const TileArgs ta) {
  constexpr int BF = 256, kStages = kPairStages;
  constexpr int kTileOutputs = MODE == kGluBf16 ? BF / 2 : BF;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t tmem_base_slot;
  __shared__ volatile int abort_flag;
  __shared__ __align__(16) float ws[BF];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t out_smem = base + kStages * kPairStageBytes;
  const uint32_t bars = out_smem + 2 * kOutBytes;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kStages + s); };
  auto acc_full_bar = [&](int b) { return bars + 8u * (2 * kStages + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * kStages + 2 + b); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total_kb = (a.K + KB - 1) / KB;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int first = (int)blockIdx.x / 2, step = (int)gridDim.x / 2;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);   // (in the first block) its loader, which expects both blocks' bytes
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);
      mbar_init(acc_empty_bar(b), 8);  // (in the first block) one arrival per epilogue warp of both
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // both blocks' barriers and accumulators exist from here on
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_base_slot;
  allow_dependents();

  if (warp == 0) {
    if (lane == 0) {
      int kbg = 0;
      bool ok = true, waited = false;
      for (int tile = first; ok && tile < ta.n_tiles; tile += step) {
        const int f_tile = tile / ta.n_t_tiles, t_tile = tile % ta.n_t_tiles;
        const int w_row = f_tile * kTileOutputs + (rank == 0 ? 0 : MODE == kGluBf16 ? a.N : BM);
        const int x_row = (2 * t_tile + (int)rank) * BM;
        auto load_weights = [&](int kb, int s) {
          if (rank == 0) mbar_expect_tx(full_bar(s), 2 * kPairStageBytes);
          tma_load_2d_pair(base + s * kPairStageBytes + BM * KB, &map_w, on_first(full_bar(s)), kb * KB, w_row);
        };
        // weights are finished before any launch that reads them
        const int n_pre = waited ? 0 : min(kStages, total_kb);
        for (int i = 0; i < n_pre; ++i) load_weights(i, i);
        if (!waited) grid_dependency_wait();
        waited = true;
        for (int kb = 0; kb < total_kb; ++kb, ++kbg) {
          const int s = kbg % kStages;
          if (kbg >= n_pre) {
            if (!mbar_wait(empty_bar(s), ((kbg / kStages) & 1) ^ 1, &abort_flag, a.error_flag, 1)) { ok = false; break; }
            load_weights(kb, s);
          }
          tma_load_2d_pair(base + s * kPairStageBytes, &map_x, on_first(full_bar(s)), kb * KB, x_row);
        }
      }
      if (!ok) {  // gave up: give the loads in flight, which count into the first block's barriers, time to land
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) {}
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = (idesc_i8(BF) & ~(0x1fu << 24)) | ((256u >> 4) << 24);  // M = 256
      int kbg = 0, it = 0;
      bool ok = true;
      for (int tile = first; ok && tile < ta.n_tiles; tile += step, ++it) {
        const int buf = it & 1;
        if (!mbar_wait(acc_empty_bar(buf), ((it >> 1) & 1) ^ 1, &abort_flag, a.error_flag, 5)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem_base + buf * BF;
        for (int kb = 0; kb < total_kb; ++kb, ++kbg) {
          const int s = kbg % kStages;
          if (!mbar_wait(full_bar(s), (kbg / kStages) & 1, &abort_flag, a.error_flag, 2)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sx = base + s * kPairStageBytes;
          const uint64_t dx = umma_desc(sx), dw = umma_desc(sx + BM * KB);
#pragma unroll
          for (int k = 0; k < KB / 32; ++k) {
            const uint32_t accumulate = (kb > 0 || k > 0) ? 1u : 0u;
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                ::"r"(d), "l"(dx + 2 * k), "l"(dw + 2 * k), "r"(idesc), "r"(accumulate) : "memory");
          }
          umma_commit_pair(empty_bar(s));
        }
        umma_commit_pair(acc_full_bar(buf));
      }
    }
  } else {
    const int quad = warp & 3, row = quad * 32 + lane, et = threadIdx.x - 64;
    const bool sender = warp == 2 && lane == 0;
    int n_sent = 0, it = 0;
    bool waited = false;
    for (int tile = first; tile < ta.n_tiles; tile += step, ++it) {
      const int buf = it & 1;
      const int f_tile = tile / ta.n_t_tiles, t_tile = tile % ta.n_t_tiles;
      const int tok0 = (2 * t_tile + (int)rank) * BM, tok = tok0 + row, f0 = f_tile * kTileOutputs;
      asm volatile("barrier.sync 1, 128;" ::: "memory");  // the last tile's scales have been read
      tile_scales<MODE, BF>(a, ws, f0, et);
      if (!waited) grid_dependency_wait();
      waited = true;
      const float xs = tok < a.M ? a.x_scale[tok] : 0.f;
      if (!all_agree(mbar_wait(acc_full_bar(buf), (it >> 1) & 1, &abort_flag, a.error_flag, 3))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t taddr = tmem_base + buf * BF + ((uint32_t)(quad * 32) << 16);
      if (tok0 < a.M)  // the same for the block
        drain<MODE, BF>(a, &map_y, ta.by_tma, ws, xs, f0, tok0, quad, lane, sender, out_smem, n_sent, 0, 1, abort_flag,
                        [&](int c0, uint32_t* r) { tmem_ld16(taddr + c0, r); });
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(on_first(acc_empty_bar(buf))) : "memory");
    }
    if (ta.by_tma && sender) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  if (warp == 1 && lane == 0) {  // every accumulator must be idle before its columns are freed
    const int my_tiles = first < ta.n_tiles ? (ta.n_tiles - first + step - 1) / step : 0;
    for (int b = 0; b < 2; ++b) {
      const int uses = (my_tiles + 1 - b) / 2;
      if (uses > 0) {
        const long long t0 = clock64();
        while (!mbar_try_wait(acc_full_bar(b), (uses - 1) & 1) && clock64() - t0 < kWaitCycles) {}
      }
    }
  }
  // neither block leaves while the other may read its shared memory, or count into its barriers
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
}

// ---------------------------------------------------------------------------------- host
struct Operands {
  const void* x; int64_t ldx;
  const void* w; int64_t ldw; int w_rows;
};

int encode(CUtensorMap* m, CUtensorMapDataType type, int dims, const void* ptr, const cuuint64_t* size, const cuuint64_t* stride,
           const cuuint32_t* box) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return fail(kLaunchFailed, "linear_q8: the driver does not offer cuTensorMapEncodeTiled");
  const cuuint32_t ones[3] = {1, 1, 1};
  CUresult r = fn(m, type, dims, const_cast<void*>(ptr), size, stride, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? kOk : fail(kLaunchFailed, "linear_q8: cuTensorMapEncodeTiled failed with %d", (int)r);
}
// 8-bit rows [rows, K]: boxes of box_rows rows x one K block, or, K in whole blocks, x kkb K blocks one after the other
int rows_map(CUtensorMap* m, const void* ptr, int64_t ld, int rows, int K, int box_rows, int kkb) {
  if (kkb > 1) {
    const cuuint64_t size[3] = {KB, (cuuint64_t)rows, (cuuint64_t)(K / KB)};
    const cuuint64_t stride[2] = {(cuuint64_t)ld, KB};
    const cuuint32_t box[3] = {KB, (cuuint32_t)box_rows, (cuuint32_t)kkb};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, ptr, size, stride, box);
  }
  const cuuint64_t size[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t stride[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {KB, (cuuint32_t)box_rows};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, ptr, size, stride, box);
}

constexpr int kMaxDevices = 64;
int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev >= 0 && dev < kMaxDevices ? dev : 0;
}
// What a device answers to a question, asked once.  Threads that come first together ask each for themselves; the answer
// that is stored first is everybody's, so that a plan and its launch go by the same one.
struct Asked {
  std::atomic<int> known[kMaxDevices];  // the answer + 1
  template <typename Ask>
  int operator()(Ask ask) {
    std::atomic<int>& k = known[current_device()];
    int v = k.load();
    if (v == 0) {
      const int mine = 1 + ask();
      if (k.compare_exchange_strong(v, mine)) v = mine;
    }
    return v - 1;
  }
};
int sm_count() {
  static Asked asked;
  return asked([] {
    int v = 0;
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, current_device());
    return v > 0 ? v : 148;
  });
}
// Shared memory of a kernel, reserved once per device.
typedef std::atomic<bool> Done[kMaxDevices];
template <typename K>
int reserve(K kernel, int bytes, Done& done) {
  const int dev = current_device();
  if (done[dev].load()) return kOk;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(kLaunchFailed, "linear_q8: cannot reserve %d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
  done[dev].store(true);
  return kOk;
}

struct RowsPlan { int rows, splits, kkb, kstack; };

// How many clusters of `size` blocks run at a time (one block per SM, clusters inside a GPC).  Asked for the streaming
// kernel; a block of the tile kernel has an SM to itself as well, so that as many of its clusters fit.
int cluster_room(int size) {
  static Asked asked[2];
  return asked[size == 4]([size] {
    auto kernel = q8_rows_kernel<64, kAccumF32, kCluster>;
    static Done done;
    if (reserve(kernel, kRowsSmemBytes, done) != kOk) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1024, 1, size);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kRowsSmemBytes - 4096;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = size;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int v = 0;
    if (cudaOccupancyMaxActiveClusters(&v, kernel, &cfg) == cudaSuccess) return v > 0 ? v : 0;
    cudaGetLastError();
    return 0;
  });
}

// The tile height is the smallest multiple of 8 whose tiles fill the SMs in whole waves.  Up to 16 tokens, tiles of at
// most 64 rows stack 128 / rows K blocks into one MMA; a box brings about 32 KB of weights.  From 17 tokens on a product
// that is not gated is cut along K into a cluster of 2 or 4, tiles as tall as lets all clusters run at once, whichever
// moves fewer bytes per block (its share of the weight and of the tokens' rows).
RowsPlan plan_rows(int N, int K, bool gated, int bn, bool fours) {
  const int sms = sm_count();
  const int n_kb = (K + KB - 1) / KB;
  const bool whole = K % KB == 0;  // boxes of several K blocks
  const int waves = (N + sms * 128 - 1) / (sms * 128);
  int rows = (N + sms * waves - 1) / (sms * waves);
  rows = (rows + 7) / 8 * 8;
  rows = rows < 8 ? 8 : rows > 128 ? 128 : rows;
  RowsPlan best{rows, 1, 1, 1};
  if (!gated && bn > 16 && fours) {
    long long best_cost = 0;
    for (int splits = 2; splits <= 4; splits += 2) {
      const int room = cluster_room(splits);
      if (n_kb < 4 * splits || room < 1) continue;
      int r = (N + room - 1) / room;
      r = (r + 7) / 8 * 8;
      if (r > 128) continue;
      const int share = (n_kb + splits - 1) / splits;
      const long long cost = (long long)(r + bn) * share;
      if (best.splits == 1 || cost < best_cost) {
        // boxes of two K blocks, unless whole boxes would leave the last split without one; the widest token tile's
        // landing zone leaves the ring room for one
        const bool pairs = whole && bn <= 64 && (splits - 1) * ((share + 1) / 2 * 2) < n_kb;
        best = RowsPlan{r, splits, pairs ? 2 : 1, 1};
        best_cost = cost;
      }
    }
    if (best.splits > 1) return best;
  }
  if (!whole) return best;
  if (gated || bn > 16) {
    best.kkb = bn <= 64 && n_kb > 1 ? 2 : 1;
    return best;
  }
  int kstack = 128 / rows;
  if (kstack > 256 / bn) kstack = 256 / bn;
  if (kstack > n_kb) kstack = n_kb;
  const int group = kstack * rows * KB;  // bytes of weights that one MMA takes
  int per_box = (28 * 1024 + group - 1) / group;
  if (per_box > 16 / kstack) per_box = 16 / kstack;
  if (per_box > (n_kb + kstack - 1) / kstack) per_box = (n_kb + kstack - 1) / kstack;
  if (per_box < 1) per_box = 1;
  while (per_box > 1 && per_box * kstack * (rows + bn) * KB > 48 * 1024) --per_box;
  best.kkb = per_box * kstack;
  best.kstack = kstack;
  return best;
}

template <int BN, int MODE>
int launch_rows(const Operands& o, const Args& a, const RowsPlan& p, cudaStream_t stream) {
  constexpr bool gated = MODE == kGluBf16;
  constexpr int kATiles = gated ? 2 : 1;
  CUtensorMap mw, mx;
  if (int rc = rows_map(&mw, o.w, o.ldw, o.w_rows, a.K, p.rows, p.kkb)) return rc;
  if (int rc = rows_map(&mx, o.x, o.ldx, a.M, a.K, BN, p.kkb)) return rc;
  RowsArgs ra;
  ra.rows_per_block = p.rows;
  ra.kkb = p.kkb;
  ra.kstack = p.kstack;
  const int total_kb = (a.K + KB - 1) / KB;
  ra.kb_per_split = ((total_kb + p.splits - 1) / p.splits + p.kkb - 1) / p.kkb * p.kkb;  // whole boxes
  ra.tmem_cols = 32;
  while (ra.tmem_cols < kATiles * p.kstack * BN) ra.tmem_cols *= 2;
  const int stage = p.kkb * (kATiles * p.rows + BN) * KB;
  // behind the ring: the cluster's landing zone or the stacked sums, at least what the MMA, reading 128 rows whatever
  // the tile's height is, may run into
  int landing = 0;
  if (p.splits > 1) landing = ((BN + p.splits - 1) / p.splits * p.splits + 4) * BM * 4;
  if (p.kstack > 1) landing = p.kstack * BN * p.rows * 4;
  const int over_read = (BM - p.kstack * p.rows) * KB;
  if (landing < over_read) landing = over_read;
  const int fixed = 16 + 8 * (2 * kRowsMaxStages + 3) + 1024 + landing;
  ra.n_stages = (kRowsSmemBytes - fixed) / stage;
  if (ra.n_stages > kRowsMaxStages) ra.n_stages = kRowsMaxStages;
  if (ra.n_stages < 2) return fail(kBadArgument, "linear_q8: stages of %d bytes do not fit twice", stage);
  if (p.splits > 1 && ra.n_stages * stage < landing)  // the splits' tiles wait in the idle ring for their bulk copies
    return fail(kBadArgument, "linear_q8: a ring of %d bytes is too small for the K splits' tiles", ra.n_stages * stage);
  if (p.splits > 1 && (p.splits - 1) * ra.kb_per_split >= total_kb)
    return fail(kBadArgument, "linear_q8: %d splits leave one without K blocks", p.splits);
  const int smem = fixed + ra.n_stages * stage;
  const dim3 grid((unsigned)((a.N + p.rows - 1) / p.rows), 1, (unsigned)p.splits);
  // (plan_rows stacks K blocks up to 16 tokens only and cuts K beyond only, neither for a gated weight)
  if (p.splits > 1) {
    if constexpr (!gated && BN > 16) {
      static Done done;
      auto kernel = q8_rows_kernel<BN, MODE, kCluster>;
      if (int rc = reserve(kernel, kRowsSmemBytes, done)) return rc;
      launch_overlapped_cluster(kernel, grid, dim3(kThreads), (size_t)smem, stream, (unsigned)p.splits, mw, mx, a, ra);
    } else {
      return fail(kBadArgument, "linear_q8: %d splits of K for tiles of %d tokens", p.splits, BN);
    }
  } else if (p.kstack > 1) {
    if constexpr (!gated && BN == 16) {
      static Done done;
      auto kernel = q8_rows_kernel<BN, MODE, kStacked>;
      if (int rc = reserve(kernel, kRowsSmemBytes, done)) return rc;
      launch_overlapped(kernel, grid, dim3(kThreads), (size_t)smem, stream, mw, mx, a, ra);
    } else {
      return fail(kBadArgument, "linear_q8: %d K blocks stacked for tiles of %d tokens", p.kstack, BN);
    }
  } else {
    static Done done;
    auto kernel = q8_rows_kernel<BN, MODE, kPlain>;
    if (int rc = reserve(kernel, kRowsSmemBytes, done)) return rc;
    launch_overlapped(kernel, grid, dim3(kThreads), (size_t)smem, stream, mw, mx, a, ra);
  }
  return check_launch("linear_q8");
}

// How many pairs of blocks run at a time.
int pair_room() {
  static Asked asked;
  return asked([] {
    auto kernel = q8_pair_kernel<kStoreBf16>;
    static Done done;
    if (reserve(kernel, kPairSmemBytes, done) != kOk) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2048);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kPairSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int v = 0;
    if (cudaOccupancyMaxActiveClusters(&v, kernel, &cfg) == cudaSuccess) return v > 0 ? v : 0;
    cudaGetLastError();
    return 0;
  });
}

// What the three kernels were measured to take, in nanoseconds, for products of 17 to 2,048 tokens and the layer sizes
// 4,096 / 6,144 / 12,288 / 25,600 and smaller odd ones (right to about a tenth).
// Weight streaming: a cluster's block takes 15 a KB of weight and tokens, and 70 for each token that it finishes; a block
// with all of K 21 a KB (at least 300 a K block), and 60 a token for its short runs of outputs.
double rows_ns(const RowsPlan& p, int M, int N, int K, bool gated, int bn, int sms) {
  const int n_kb = (K + KB - 1) / KB;
  if (p.splits > 1) {
    const double kb = (n_kb + p.splits - 1) / p.splits;
    return 3600 + 15.0 * kb * (p.rows + bn) * KB / 1024 + 70.0 * ((M + p.splits - 1) / p.splits);
  }
  const int waves = ((N + p.rows - 1) / p.rows + sms - 1) / sms;
  const double stream = 21.0 * (p.rows * (gated ? 2 : 1) + bn) * KB / 1024;
  return 3000 + (double)waves * n_kb * (stream > 300 ? stream : 300) + 60.0 * M;
}
// Tiles: a K block takes 370 / 245 / 205 at 256 / 128 / 64 columns, 540 / 300 / 205 where one tile of tokens reads each
// weight once, from memory; a tile costs 5,200 / 3,450 / 2,800 beside its K blocks; a cluster's meetings and exchange
// 2,900 (two blocks) or 4,200 (1,700 where a tile has 64 outputs).  Tiles of two SMs (columns = 512): 335 a K block and
// 5,000 beside.  (A gated product of 200 tokens by weight streaming, two instructions of 256 columns for 32 bytes of K:
// 39 against 30 us.)
struct TilePlan { int columns, splits; double ns; };
TilePlan plan_tiles(int M, int N, int K, bool gated, int sms) {
  const long long n_kb = (K + KB - 1) / KB, n_t = (M + BM - 1) / BM;
  TilePlan best{256, 1, 0};
  for (int columns = 64; columns <= 256; columns *= 2) {
    if (gated && columns == 64) continue;
    const double per_kb = columns == 256 ? (n_t == 1 ? 540 : 370) : columns == 128 ? (n_t == 1 ? 300 : 245) : 205;
    const double beside = columns == 256 ? 5200 : columns == 128 ? 3450 : 2800;
    const int outputs = gated ? columns / 2 : columns;
    const long long tiles = n_t * ((N + outputs - 1) / outputs);
    for (int splits = 1; splits <= kMaxSplits; splits *= 2) {
      if (splits > 1 && (tiles > cluster_room(splits) || n_kb < 2 * splits)) break;
      const long long waves = (tiles * splits + sms - 1) / sms;
      double main = (double)((n_kb + splits - 1) / splits) * per_kb;
      if (waves > 1 && main < beside / 2) main = beside / 2;  // (the epilogue of all but the last tile runs beside the next)
      const double ns = (double)waves * main + beside + (splits == 2 ? 2900 : splits == 4 ? (outputs == 64 ? 1700 : 4200) : 0);
      if (best.ns == 0 || ns < best.ns) best = TilePlan{columns, splits, ns};
    }
  }
  const int room = n_t > 1 ? pair_room() : 0;
  if (room > 0) {
    const int outputs = gated ? 128 : 256;
    const long long tiles = (n_t + 1) / 2 * ((N + outputs - 1) / outputs), waves = (tiles + room - 1) / room;
    const double main = n_kb * 335.0 > 2500 || waves == 1 ? n_kb * 335.0 : 2500;
    const double ns = (double)waves * main + 5000;
    if (ns < best.ns) best = TilePlan{512, 1, ns};
  }
  return best;
}

// A map of y for the epilogue's TMA stores, where its rows allow them (else a valid map that is not used).  (A TMA store
// clips at whole 16-byte pieces: a row that ends inside one would write beyond it.)
int output_map(CUtensorMap* my, const CUtensorMap& any, const Args& a, bool f32, int* by_tma) {
  const int size = f32 ? 4 : 2;
  *by_tma = (uintptr_t)a.y % 16 == 0 && a.ldy * size % 16 == 0 && (int64_t)a.N * size % 16 == 0;
  *my = any;
  if (!*by_tma) return kOk;
  const cuuint64_t dims[2] = {(cuuint64_t)a.N, (cuuint64_t)a.M};
  const cuuint64_t stride[1] = {(cuuint64_t)a.ldy * size};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), BM};
  return encode(my, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.y, dims, stride, box);
}
// A launch of `blocks` blocks in clusters of `cluster` along x (1: none).
template <typename... KArgs, typename... Given>
void launch_cluster_x(void (*kernel)(KArgs...), unsigned blocks, int cluster, int smem, cudaStream_t stream, Given&&... given) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (overlap_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, kernel, std::forward<Given>(given)...);  // errors are read by check_launch()
}

template <int MODE, int BF, bool SPLIT>
int launch_tiles(const Operands& o, const Args& a, int splits, cudaStream_t stream) {
  using C = TileCfg<MODE, BF>;
  constexpr int kTileOutputs = MODE == kGluBf16 ? BF / 2 : BF;
  constexpr bool f32 = MODE == kStoreF32 || MODE == kAccumF32;
  TileArgs ta;
  ta.n_t_tiles = (a.M + BM - 1) / BM;
  const long long tiles = (long long)ta.n_t_tiles * ((a.N + kTileOutputs - 1) / kTileOutputs);
  if (tiles > 0x3fffffffLL) return fail(kBadArgument, "linear_q8: too many tiles");
  ta.n_tiles = (int)tiles;
  CUtensorMap mx, mw, my;
  ta.boxes = C::kKkb > 1 && a.K % KB == 0;
  const int kkb = ta.boxes ? C::kKkb : 1;
  ta.x_rows = a.M < BM ? (a.M + 7) / 8 * 8 : BM;
  if (int rc = rows_map(&mx, o.x, o.ldx, a.M, a.K, ta.x_rows, kkb)) return rc;
  if (int rc = rows_map(&mw, o.w, o.ldw, o.w_rows, a.K, MODE == kGluBf16 ? BF / 2 : BF, kkb)) return rc;
  if (int rc = output_map(&my, mx, a, f32, &ta.by_tma)) return rc;
  static Done done;
  auto kernel = q8_tile_kernel<MODE, BF, SPLIT>;
  if (int rc = reserve(kernel, C::kSmemBytes, done)) return rc;
  const int sms = sm_count();
  ta.splits = SPLIT ? splits : 1;
  launch_cluster_x(kernel, SPLIT ? (unsigned)(tiles * splits) : (unsigned)(tiles < sms ? tiles : sms), SPLIT ? splits : 1, C::kSmemBytes, stream,
                   mx, mw, my, a, ta);
  return check_launch("linear_q8");
}
template <int MODE, int BF>
int launch_tiles(const Operands& o, const Args& a, int splits, cudaStream_t stream) {
  return splits > 1 ? launch_tiles<MODE, BF, true>(o, a, splits, stream) : launch_tiles<MODE, BF, false>(o, a, 1, stream);
}

template <int MODE>
int launch_pairs(const Operands& o, const Args& a, cudaStream_t stream) {
  constexpr int kTileOutputs = MODE == kGluBf16 ? 128 : 256;
  TileArgs ta = {};
  ta.n_t_tiles = (a.M + 2 * BM - 1) / (2 * BM);
  const long long tiles = (long long)ta.n_t_tiles * ((a.N + kTileOutputs - 1) / kTileOutputs);
  if (tiles > 0x3fffffffLL) return fail(kBadArgument, "linear_q8: too many tiles");
  ta.n_tiles = (int)tiles;
  ta.splits = 1;
  CUtensorMap mx, mw, my;
  if (int rc = rows_map(&mx, o.x, o.ldx, a.M, a.K, BM, 1)) return rc;
  if (int rc = rows_map(&mw, o.w, o.ldw, o.w_rows, a.K, BM, 1)) return rc;
  if (int rc = output_map(&my, mx, a, MODE == kStoreF32 || MODE == kAccumF32, &ta.by_tma)) return rc;
  static Done done;
  auto kernel = q8_pair_kernel<MODE>;
  if (int rc = reserve(kernel, kPairSmemBytes, done)) return rc;
  const long long room = pair_room();
  launch_cluster_x(kernel, (unsigned)(2 * (tiles < room ? tiles : room)), 2, kPairSmemBytes, stream, mx, mw, my, a, ta);
  return check_launch("linear_q8");
}

// The kernel of a product: tiles of p.columns (512: of two SMs; 0: weight streaming by r).  Up to 16 tokens stream always.
// (Not the best for narrow outputs of a long K that does not stack, gated or not in whole blocks: few SMs walk all of K. 16 x
// 11,142 to 171 take 24.8 us where 17 tokens, in tiles with K over four blocks, take 8.0; 8 x 16,384 to 2 x 512 38.6, 17
// tokens 11.3.)
struct Plan { RowsPlan r; int bn; TilePlan p; };
Plan plan(int M, int N, int K, bool gated, bool fours) {
  Plan c;
  c.bn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  c.r = plan_rows(N, K, gated, c.bn, fours);
  c.p = TilePlan{0, 1, 0};
  if (M <= 16) return c;
  const int sms = sm_count();
  const TilePlan tiles = plan_tiles(M, N, K, gated, sms);
  if (M > 128 || rows_ns(c.r, M, N, K, gated, c.bn, sms) >= tiles.ns) c.p = tiles;
  return c;
}
// the owners of a cluster write four neighbouring outputs of a token at once
bool in_fours(const void* y, int64_t ldy, int N, int mode) {
  return N % 4 == 0 && ldy % 4 == 0 && (uintptr_t)y % (mode == kStoreBf16 ? 8 : 16) == 0;
}

template <int MODE>
int launch(const Operands& o, const Args& a, cudaStream_t stream) {
  constexpr bool gated = MODE == kGluBf16;
  const Plan c = plan(a.M, a.N, a.K, gated, in_fours(a.y, a.ldy, a.N, MODE));
  switch (c.p.columns) {
    case 512: return launch_pairs<MODE>(o, a, stream);
    case 256: return launch_tiles<MODE, 256>(o, a, c.p.splits, stream);
    case 128: return launch_tiles<MODE, 128>(o, a, c.p.splits, stream);
    case 64: return launch_tiles<gated ? kStoreBf16 : MODE, 64>(o, a, c.p.splits, stream);  // (no gated tile is this narrow)
  }
  switch (c.bn) {
    case 16: return launch_rows<16, MODE>(o, a, c.r, stream);
    case 32: return launch_rows<32, MODE>(o, a, c.r, stream);
    case 64: return launch_rows<64, MODE>(o, a, c.r, stream);
    default: return launch_rows<128, MODE>(o, a, c.r, stream);
  }
}
}  // namespace

// x [M, K] and w [N (2N gated: the gate rows, then the up rows), K], rows that begin on multiples of 16 bytes.
// mode 0: y = v (bfloat16), 1: y = v (float32), 2: y += v (float32), 3: y = silu(gate) * up (bfloat16).
// The weight and its scales are read before the launch ahead in the stream has ended.
extern "C" int skyla_linear_q8(const void* x, int64_t ldx, const float* x_scale, const void* w, int64_t ldw, const float* w_scale,
                               int M, int N, int K, void* y, int64_t ldy, int mode, int* error_flag, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return kOk;
  if (K <= 0 || K > kMaxWidth) return fail(kBadArgument, "linear_q8: K=%d is outside 1..%d", K, kMaxWidth);
  if (mode < kStoreBf16 || mode > kGluBf16) return fail(kBadArgument, "linear_q8: unknown mode %d", mode);
  if (N > (1 << 29) || M > (1 << 29)) return fail(kBadArgument, "linear_q8: %d tokens, %d outputs: at most 2^29", M, N);
  if ((uintptr_t)x % 16 || (uintptr_t)w % 16 || ldx % 16 || ldw % 16)
    return fail(kBadArgument, "linear_q8: rows that do not begin on multiples of 16 bytes");
  const Operands o{x, ldx, w, ldw, mode == kGluBf16 ? 2 * N : N};
  const Args a{y, ldy, M, N, K, x_scale, w_scale, error_flag};
  switch (mode) {
    case kStoreBf16: return launch<kStoreBf16>(o, a, stream);
    case kStoreF32: return launch<kStoreF32>(o, a, stream);
    case kAccumF32: return launch<kAccumF32>(o, a, stream);
    default: return launch<kGluBf16>(o, a, stream);
  }
}

// Which kernel takes a product of these sizes whose y is aligned, for tests and measurements: tiles, columns * 16 + splits
// (512 columns: two SMs a tile); weight streaming, minus the splits (1, 2, 4), or minus 16 times the K blocks of an MMA.
extern "C" int skyla_linear_q8_plan(int M, int N, int K, int gated) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan c = plan(M, N, K, gated != 0, N % 4 == 0);
  if (c.p.columns > 0) return c.p.columns * 16 + c.p.splits;
  return c.r.kstack > 1 ? -16 * c.r.kstack : -c.r.splits;
}
