// Product of block-scaled 4-bit operands on tcgen05, with the epilogues of a transformer's linear layers:
//   y[m, n] = (sum_k A[m, k] SA[m, k / B] W[n, k] SW[n, k / B]) * row_scale[m] * col_scale[n] + bias[n]
// B = 16 (FF_FP4_NV) or 32 (FF_FP4_MX) columns per block scale. The tensor cores apply the block scales while
// they multiply (kind::mxf4nvf4 / kind::mxf4, f32 accumulators in TMEM); the row scales, which are powers of
// two, and the bias are applied in f32 in the epilogue, which rounds once, to the output's type.
//
// One CTA per SM, 640 threads, persistent over tiles:
//   warp 0     TMA producer: per stage 256 columns (128 bytes of codes, 128-byte swizzle) of A and W rows and
//              their scale chunks
//   warp 1     TMEM allocator; copies each stage's scale chunks to TMEM (tcgen05.cp, in order with the MMAs of
//              the same thread) and issues the MMAs, 64 columns each
//   warp 2     column scales and biases, four tiles ahead
//   warps 4-19 epilogue: two groups, one per accumulator, one output row per lane
// Tiles: 128 x 128 per CTA, or (PAIR) 256 x 256 over a cluster of two CTAs, where each CTA loads its 128 rows
// of A, half of W's 256 rows and all of the tile's W scales (each SM's tensor core reads them from its own
// TMEM), and shared memory moves half as many bytes per multiply-add.
//
// Measured, FF_FP4_NV unless said, from rest: 8192^3 195 us (5.6 PFLOP/s, 3.4 times the bf16 rate of the same GPU; FF_FP4_MX
// 185), under the power cap, the tensor pipe active 69% of the cycles at 4096 x 4096 x 8192. 65600 x 5504 x 1024 with SwiGLU
// 205 us (3.6 PFLOP/s), where reading the accumulators, activating and storing takes about as long as the products do (when it
// took 209: 190 without the column parameters, 183 without the stores, 159 with the MMAs alone); launched without a pause the
// power cap lowers the SM clock to 1.52 GHz and it takes 247. 65600 x 1024 x 2730 with a residual 100 us (118 at 1.35 GHz);
// 65600 x 1024 x 1024 44 us. 8200 x 2304 x 768 with norm and rotation 27 us, bound by its epilogue (21 without the reads of the
// angles). One row of 1024 against 30877: 8 us, the latency of a launch and of two tiles.
#include "common.h"
#include "fp4.cuh"
#include "gemm_fp4.h"
#include "gemm_tc.cuh"

namespace ff {

namespace {

template <bool PAIR, bool QKV>
struct Fp4Cfg {
  static constexpr int BN = PAIR ? 256 : 128;
  static constexpr int TILE_M = PAIR ? 256 : 128;
  static constexpr int HALF = BN / 2;  // tile columns per epilogue warp
  static constexpr int CODE_BYTES = 128 * 128;  // 128 rows of A, or of W, per CTA and stage
  static constexpr int SFA_BYTES = 4 * kSfChunk;
  static constexpr int SFB_BYTES = (BN / 128) * 4 * kSfChunk;
  static constexpr int STAGE_BYTES = 2 * CODE_BYTES + SFA_BYTES + SFB_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int GROUP_WARPS = 8;  // epilogue warps that work on one accumulator
  static constexpr int GROUPS = 2;       // take turns with the tiles
  static constexpr int THREADS = 128 + GROUPS * 32 * GROUP_WARPS;
  static constexpr int STAGING = 4096;      // per epilogue warp: 32 rows x 128 B
  static constexpr int COLP = 2 * BN * 4;   // column scales and biases of a tile
  static constexpr int COLP_BUFS = 4;       // tiles that they are read ahead
  static constexpr int NORM_BYTES = 4 * 64 * 4;  // q and k norm weights and biases
  static constexpr int BAR_BYTES = 512;
  static constexpr int SMEM =
      1024 + STAGES * STAGE_BYTES + GROUPS * GROUP_WARPS * STAGING + COLP_BUFS * COLP + (QKV ? NORM_BYTES : 0) + BAR_BYTES;
  // TMEM: two accumulators and two buffers of scales, each for one chunk of A's and W's columns. Two 256-column
  // accumulators and the scales do not fit 512 columns: the pair's accumulators share 32 columns, the last of
  // the first and the first of the second, which the epilogue empties first.
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr uint32_t ACC_STRIDE = PAIR ? 224 : 128;
  static constexpr uint32_t SFA_BASE = 480, SFB_BASE = 488;  // + 4 and + BN / 32 columns per buffer
  static_assert(STAGE_BYTES % 1024 == 0, "stages keep the swizzle's alignment");
  static_assert(ACC_STRIDE + BN <= SFA_BASE && SFB_BASE + 2 * (BN / 32) <= TMEM_COLS, "TMEM");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// silu(g) * u = g / (1 + 2^(-g log2 e)) * u, each gate with its own reciprocal: right over the whole range of f32 (far below
// zero the power is infinite and silu zero) as long as the product with u comes last. One reciprocal for two gates needs
// bounds on the powers and was no faster (65600 x 5504 x 1024 204.0 us, 204.9 with it; 8200 x 4096 x 768 19.0 and 18.9).
__device__ __forceinline__ float2 silu_up2(float2 g, float2 u) {
  const float2 t = mul2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  const float2 d = add2(make_float2(1.f, 1.f), make_float2(ex2_approx(t.x), ex2_approx(t.y)));
  return mul2(mul2(g, make_float2(rcp_approx(d.x), rcp_approx(d.y))), u);
}
// tanh GELU: x * sigmoid(2 sqrt(2 / pi) (x + 0.044715 x^3)), on two lanes with three MUFU operations instead of four: one
// reciprocal of the product of both denominators (5184 x 4736 x 1024 21.7 us, 21.9 with two). An x below -7.6, where the
// power passes 2^62, counts as -7.6, so that the product stays finite: the result is off by at most 2^-59. A NaN stays
// in its lane: its power counts as 2^62.
__device__ __forceinline__ float2 gelu2(float2 x) {
  constexpr float c1 = -2.302208198f, c3 = -2.302208198f * 0.044715f;  // times -2 sqrt(2 / pi) log2 e
  float2 c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c.x) : "f"(x.x), "f"(-7.6f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c.y) : "f"(x.y), "f"(-7.6f));
  const float2 t = mul2(c, fma2(mul2(c, c), make_float2(c3, c3), make_float2(c1, c1)));
  const float2 d = add2(make_float2(1.f, 1.f), make_float2(ex2_approx(fminf(t.x, 62.f)), ex2_approx(fminf(t.y, 62.f))));
  const float r = rcp_approx(d.x * d.y);
  return mul2(c, mul2(make_float2(r, r), make_float2(d.y, d.x)));
}

// r[j] = r[j] * (rs * cs[j]) + bias[j] for N accumulators in place (as f32 bits); FF_FP4_MX has no row and column
// scales. cs and bias in shared memory, read by every lane at once.
template <int N, bool MX>
__device__ __forceinline__ void scale_cols(uint32_t* r, float rs, const float* cs, const float* bias) {
  const float2 rs2 = make_float2(rs, rs);
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const float4 b = *reinterpret_cast<const float4*>(bias + j);
    float2 lo = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
    float2 hi = make_float2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
    if constexpr (MX) {
      lo = add2(lo, make_float2(b.x, b.y));
      hi = add2(hi, make_float2(b.z, b.w));
    } else {
      const float4 c = *reinterpret_cast<const float4*>(cs + j);
      lo = fma2(lo, mul2(rs2, make_float2(c.x, c.y)), make_float2(b.x, b.y));
      hi = fma2(hi, mul2(rs2, make_float2(c.z, c.w)), make_float2(b.z, b.w));
    }
    r[j] = __float_as_uint(lo.x);
    r[j + 1] = __float_as_uint(lo.y);
    r[j + 2] = __float_as_uint(hi.x);
    r[j + 3] = __float_as_uint(hi.y);
  }
}
// Waits, within the limit, for copies or MMAs in flight, whether or not the kernel is being given up.
__device__ __forceinline__ bool drain_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  const unsigned long long t0 = globaltimer();
  while (!mbar_try_wait(addr, parity))
    if (globaltimer() - t0 > kWaitLimitNs) return false;
  return true;
}
// Keeps the compiler from starting a later group's loads early: the epilogue has registers for one group.
__device__ __forceinline__ void group_end() { asm volatile("" ::: "memory"); }

// The scale copies and MMAs of one stage: chunk g of the scales goes to buffer g % 2, in order with the MMAs that
// read it.
template <bool PAIR, bool MX, class C>
__device__ __forceinline__ void fp4_stage_mmas(uint32_t d, uint32_t tmem, uint32_t sa, int steps, bool first) {
  constexpr int CH = sf_chunks_per_step(MX);
  constexpr int BT = C::BN / 128;
  const uint32_t ssa = sa + 2 * C::CODE_BYTES, ssb = ssa + C::SFA_BYTES;
  const uint64_t adesc = sdesc_k_sw128(sa), bdesc = sdesc_k_sw128(sa + C::CODE_BYTES);
  constexpr uint32_t idesc = idesc_fp4(C::TILE_M, C::BN, MX);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k < steps) {
      const int g = MX ? k / 2 : k;
      const uint32_t sfa = tmem + C::SFA_BASE + (g & 1) * 4, sfb = tmem + C::SFB_BASE + (g & 1) * (C::BN / 32);
      if (!MX || (k & 1) == 0) {
        tc_cp_sf<PAIR>(sfa, sdesc_sf(ssa + g * kSfChunk));
#pragma unroll
        for (int t = 0; t < BT; ++t) tc_cp_sf<PAIR>(sfb + 4 * t, sdesc_sf(ssb + (t * CH + g) * kSfChunk));
      }
      mma_fp4<PAIR, MX>(d, adesc + 2 * k, bdesc + 2 * k, idesc | (MX ? idesc_sf_id((k & 1) * 2) : 0u), sfa, sfb,
                        !(first && k == 0));
    }
  }
}

template <bool PAIR, bool MX, int EPI, class OutT>
__global__ void __launch_bounds__(Fp4Cfg<PAIR, EPI == EPI_QKV_NORM_ROPE>::THREADS, 1)
    gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSW,
                    const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmR,
                    const Fp4GemmArgs args) {
  constexpr bool RES = EPI == EPI_RESIDUAL;
  constexpr bool F32OUT = sizeof(OutT) == 4;
  constexpr bool QKV = EPI == EPI_QKV_NORM_ROPE;
  using C = Fp4Cfg<PAIR, QKV>;
  constexpr int STAGES = C::STAGES, BN = C::BN, HALF = C::HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + STAGES * C::STAGE_BYTES;
  float* colp = reinterpret_cast<float*>(staging + C::GROUPS * C::GROUP_WARPS * C::STAGING);
  float* normp = colp + C::COLP_BUFS * (C::COLP / 4);  // EPI_QKV_NORM_ROPE: q weight, q bias, k weight, k bias
  uint64_t* full = reinterpret_cast<uint64_t*>(normp + (QKV ? C::NORM_BYTES / 4 : 0));
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;  // an accumulator has been read
  uint64_t* tearly = tempty + 2;  // PAIR: the columns that it shares with the other one have been read
  uint64_t* pfull = tearly + 2;  // a tile's column scales and biases are in shared memory
  uint64_t* pempty = pfull + C::COLP_BUFS;
  uint64_t* drain = pempty + C::COLP_BUFS;
  uint64_t* resbar = drain + 1;  // one per epilogue warp (EPI_RESIDUAL)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(resbar + 2 * C::GROUP_WARPS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_n = args.tiles_n;
  const int tiles = args.tiles_m * tiles_n;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int unit = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int units = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  // Tile i of this CTA (pair): strided over the units, so that the tiles in work at one time share A and W in L2;
  // for EPI_QKV_NORM_ROPE runs along N, whose tiles share the rows' angles.
  const int t_first = QKV ? static_cast<int>(static_cast<int64_t>(unit) * tiles / units) : unit;
  const int t_step = QKV ? 1 : units;
  const int my_tiles = QKV ? static_cast<int>(static_cast<int64_t>(unit + 1) * tiles / units) - t_first
                           : (tiles - unit + units - 1) / units;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if constexpr (PAIR)
      return mbar_wait_cluster<true>(bar, parity, abort_flag, args.err, code);
    else
      return mbar_wait<true>(bar, parity, abort_flag, args.err, code);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], (PAIR ? 2 : 1) * C::GROUP_WARPS);
      mbar_init(&tearly[a], 2 * C::GROUP_WARPS / 2);
    }
    for (int p = 0; p < C::COLP_BUFS; ++p) {
      mbar_init(&pfull[p], 1);
      mbar_init(&pempty[p], C::GROUP_WARPS);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < 2 * C::GROUP_WARPS; ++i) mbar_init(&resbar[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tmA);
    tma_prefetch_map(&tmW);
    tma_prefetch_map(&tmSA);
    tma_prefetch_map(&tmSW);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc2(tmem_slot, C::TMEM_COLS);
      tmem_relinquish2();
    } else {
      tmem_alloc(tmem_slot, C::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int last_phase[STAGES];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) last_phase[s] = -1;
      constexpr int ch = sf_chunks_per_step(MX);  // scale chunks per stage and 128-row tile
      constexpr uint32_t stage_bytes = 2 * C::CODE_BYTES + (1 + BN / 128) * ch * kSfChunk;
      const int row_chunks = args.num_kb * ch;  // scale chunks of one 128-row tile
      auto load_w = [&](uint8_t* sa, uint64_t* bar, int kb, int tn) {
        uint8_t* ssb = sa + 2 * C::CODE_BYTES + C::SFA_BYTES;
        if constexpr (PAIR) {
          const uint32_t fb = mapa_shared(smem_u32(bar), 0u);
          tma_load_2d_pair(sa + C::CODE_BYTES, &tmW, fb, kb * 128, tn * BN + static_cast<int>(rank) * 128);
          tma_load_2d_pair(ssb, &tmSW, fb, 0, 2 * tn * row_chunks + kb * ch);
          tma_load_2d_pair(ssb + ch * kSfChunk, &tmSW, fb, 0, (2 * tn + 1) * row_chunks + kb * ch);
        } else {
          tma_load_2d(sa + C::CODE_BYTES, &tmW, bar, kb * 128, tn * BN);
          tma_load_2d(ssb, &tmSW, bar, 0, tn * row_chunks + kb * ch);
        }
      };
      auto load_a = [&](uint8_t* sa, uint64_t* bar, int kb, int tm) {
        uint8_t* ssa = sa + 2 * C::CODE_BYTES;
        if constexpr (PAIR) {
          const uint32_t fb = mapa_shared(smem_u32(bar), 0u);
          const int rt = 2 * tm + static_cast<int>(rank);
          tma_load_2d_pair(sa, &tmA, fb, kb * 128, rt * 128);
          tma_load_2d_pair(ssa, &tmSA, fb, 0, rt * row_chunks + kb * ch);
        } else {
          tma_load_2d(sa, &tmA, bar, kb * 128, tm * 128);
          tma_load_2d(ssa, &tmSA, bar, 0, tm * row_chunks + kb * ch);
        }
      };
      auto expect = [&](uint64_t* bar) {
        if (!PAIR) mbar_arrive_expect_tx(bar, stage_bytes);
        if (PAIR && leader) mbar_arrive_expect_tx(bar, 2 * stage_bytes);
      };
      // With w_const the weights of the first stages come in before the wait for the previous kernel.
      const int pre = args.w_const ? (args.num_kb < STAGES ? args.num_kb : STAGES) : 0;
      for (int kb = 0; kb < pre; ++kb) {
        expect(&full[kb]);
        load_w(smem + kb * C::STAGE_BYTES, &full[kb], kb, t_first % tiles_n);
      }
      pdl_wait();
      bool ok = true, first = true;
      for (int i = 0; i < my_tiles && ok; ++i) {
        const int t = t_first + i * t_step;
        const int tm = t / tiles_n, tn = t % tiles_n;
        for (int kb = 0; kb < args.num_kb; ++kb) {
          uint8_t* sa = smem + stage * C::STAGE_BYTES;
          if (!(first && kb < pre)) {
            if (!wait(&empty[stage], phase ^ 1u, kDevTimeoutSmemEmpty)) {
              ok = false;
              break;
            }
            expect(&full[stage]);
            load_w(sa, &full[stage], kb, tn);
          }
          load_a(sa, &full[stage], kb, tm);
          last_phase[stage] = static_cast<int>(phase);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        first = false;
      }
      if (!ok && leader) {
        // Let every issued copy land before the CTA exits (bounded).
        for (int s = 0; s < STAGES; ++s)
          if (last_phase[s] >= 0) drain_wait(&full[s], static_cast<uint32_t>(last_phase[s]));
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ scale copies and MMAs (the even CTA of a pair)
    // One elected lane (elect.sync): the compiler then knows that the operands of the tcgen05 instructions are
    // uniform. With a lane == 0 branch each instruction cost 50-60 cycles to issue and the issue rate bound the
    // kernel (8192^3 FF_FP4_NV: pair tiles 367 -> 215 us, 128 x 128 tiles 510 -> 273 us).
    pdl_wait();
    if (leader && elect_one()) {
      auto commit_both = [&](uint64_t* bar) {
        if constexpr (PAIR)
          tc_commit2_both(bar);
        else
          tc_commit(bar);
      };
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < my_tiles && ok; ++i) {
        const uint32_t acc = i & 1, use = (i >> 1) & 1;
        if (!wait(&tempty[acc], use ^ 1u, kDevTimeoutTmemEmpty)) break;
        if (PAIR && i > 0 && !wait(&tearly[acc ^ 1u], ((i - 1) >> 1) & 1, kDevTimeoutTmemEmpty)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * C::ACC_STRIDE;
        for (int kb = 0; kb < args.num_kb; ++kb) {
          if (!wait(&full[stage], phase, kDevTimeoutTmaFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * C::STAGE_BYTES);
          const int left = (args.K - kb * kFp4Step + 63) >> 6;  // 64-column steps to the end of the row
          fp4_stage_mmas<PAIR, MX, C>(d, tmem, sa, left, kb == 0);
          commit_both(&empty[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        commit_both(&tfull[acc]);
      }
      // Drain: every MMA this thread issued must finish before TMEM is released.
      if constexpr (PAIR)
        tc_commit2(drain);
      else
        tc_commit(drain);
      if (!drain_wait(drain, 0)) atomicCAS(args.err, 0, kDevTimeoutDrain);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ column scales and biases, up to four tiles ahead
    pdl_wait();
    for (int i = 0; i < my_tiles; ++i) {
      const int buf = i % C::COLP_BUFS;
      if (!wait(&pempty[buf], ((i / C::COLP_BUFS) & 1) ^ 1u, kDevTimeoutTmemEmpty)) break;
      float* const cs = colp + buf * (C::COLP / 4);
      const int n0 = (t_first + i * t_step) % tiles_n * BN;
      float c[BN / 32], b[BN / 32];  // all loads before the first store: one latency per tile
#pragma unroll
      for (int j = 0; j < BN / 32; ++j) {
        const int n = n0 + 32 * j + lane;
        c[j] = !MX && n < args.N ? __ldg(args.col_scale + n) : 0.f;  // zero past N
        b[j] = args.bias != nullptr && n < args.N ? __ldg(args.bias + n) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < BN / 32; ++j) {
        if constexpr (!MX) cs[32 * j + lane] = c[j];
        cs[BN + 32 * j + lane] = b[j];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[buf]);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    // Two groups of eight warps, one per accumulator, take turns with the tiles: a group has the time of two
    // mainloops for a tile. A warp reads one lane quarter (32 rows) and half of the tile's columns, 32 at a time.
    pdl_wait();
    const int ew = warp - 4;
    const int group = ew >> 3;       // also the accumulator that it works on
    const int q = warp & 3;          // TMEM lane quarter
    const int half = (ew >> 2) & 1;  // of the tile's columns
    uint8_t* const stg = staging + ew * C::STAGING;
    if constexpr (EPI == EPI_QKV_NORM_ROPE) {
      for (int i = threadIdx.x - 128; i < 64; i += C::GROUPS * 32 * C::GROUP_WARPS) {
        normp[i] = args.q_w[i];
        normp[64 + i] = args.q_b != nullptr ? args.q_b[i] : 0.f;
        normp[128 + i] = args.k_w[i];
        normp[192 + i] = args.k_b != nullptr ? args.k_b[i] : 0.f;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(C::GROUPS * 32 * C::GROUP_WARPS) : "memory");  // the epilogue warps
    }
    constexpr bool SWIGLU = EPI == EPI_SWIGLU;
    constexpr int STEPS = HALF / 64;           // 64 tile columns per step
    constexpr int WIDTH = SWIGLU ? 32 : 64;    // output columns per step
    uint32_t res_phase = 0;
    // The lane's row scale, read a tile ahead: with the epilogue at work all the time its latency would be exposed.
    auto row_scale_of = [&](int i) {
      if (MX || i >= my_tiles) return 1.f;
      const int row = (t_first + i * t_step) / tiles_n * C::TILE_M + static_cast<int>(rank) * 128 + q * 32 + lane;
      return row < args.M ? __ldg(args.row_scale + row) : 0.f;
    };
    float rs_next = row_scale_of(group);
    for (int i = group; i < my_tiles; i += C::GROUPS) {
      const int acc = group;
      const uint32_t use = (i >> 1) & 1;
      const int t = t_first + i * t_step;
      const int tm = t / tiles_n, tn = t - tm * tiles_n;
      const int buf = i % C::COLP_BUFS;
      const float* const cs_t = colp + buf * (C::COLP / 4);  // the tile's column scales, then its biases
      const int m_block = tm * C::TILE_M + static_cast<int>(rank) * 128 + q * 32;
      const int m = m_block + lane;
      const bool row_ok = m < args.M;
      const int n_tile = tn * BN;
      const float rs = rs_next;
      const uint32_t pos = QKV && row_ok ? static_cast<uint32_t>(m % args.tokens) : 0u;
      const uint32_t tbase = tmem + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc) * C::ACC_STRIDE;
      bool ok = true;
#pragma unroll 1
      for (int step = 0; step < STEPS; ++step) {
        // The first group goes from the last columns down, the second from the first columns up, so that each
        // begins with the columns that the accumulators share. ca: the step's first tile column.
        const int ca = half * HALF + (acc == 0 ? STEPS - 1 - step : step) * 64;
        const int out0 = SWIGLU ? (n_tile + ca) >> 1 : n_tile + ca;
        const bool any = m_block < args.M && out0 < args.out_cols;  // the warp has something to write
        const float *csa = cs_t + ca, *ba = csa + BN;
        __syncwarp();
        if (lane == 0) {
          if constexpr (!F32OUT) bulk_wait_read_all();  // the staging buffer is free
          if constexpr (RES) {
            if (any) {  // the residual comes in while the mainloop runs
              mbar_arrive_expect_tx(&resbar[ew], C::STAGING);
              tma_load_2d(stg, &tmR, &resbar[ew], out0, m_block);
            }
          }
        }
        __syncwarp();
        if (step == 0) {
          ok = wait(&pfull[buf], (i / C::COLP_BUFS) & 1, kDevTimeoutTmemFull) && wait(&tfull[acc], use, kDevTimeoutTmemFull);
          if (!ok) {
            if constexpr (RES) {  // let the residual copy land before the CTA exits
              if (any) drain_wait(&resbar[ew], res_phase);
            }
            break;
          }
          tc_fence_after();
        }
        // Hand back the shared columns (step 0), or the whole accumulator: every read of them has completed.
        auto arrive = [&](uint64_t* bar) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR && !leader)
              mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(bar), 0u));
            else
              mbar_arrive(bar);
          }
        };
        auto arrive_early = [&]() {
          if (PAIR && step == 0 && half != acc) arrive(&tearly[acc]);
        };
        auto arrive_empty = [&]() {
          if (step == STEPS - 1) {
            arrive(&tempty[acc]);
            rs_next = row_scale_of(i + C::GROUPS);
          }
        };
        auto read32 = [&](int col, uint32_t(&r)[32]) {
          __syncwarp();
          if (any) {
            tmem_ld32(tbase + col, r);
            tmem_ld_wait();
          }
        };
        auto wait_residual = [&]() {
          if constexpr (RES) {
            if (any) {
              ok = mbar_wait(&resbar[ew], res_phase, abort_flag, args.err, kDevTimeoutTmaFull);
              if (!ok) drain_wait(&resbar[ew], res_phase);
              res_phase ^= 1u;
              __syncwarp();
            }
          }
        };
        // Eight 16-bit output columns, at 16-byte slot g of the lane's staged row.
        auto stage8 = [&](int g, const float(&y)[8]) {
          if constexpr (!F32OUT) {
            uint4* const slot = reinterpret_cast<uint4*>(
                SWIGLU ? stg + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4) : stg + lane * 128 + ((g ^ (lane & 7)) << 4));
            float z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = y[j];
            if constexpr (RES) {
              const uint4 u = *slot;
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 f = Pair16<OutT>::unpack(w[j]);
                z[2 * j] += f.x;
                z[2 * j + 1] += f.y;
              }
            }
            *slot = make_uint4(Pair16<OutT>::pack(z[0], z[1]), Pair16<OutT>::pack(z[2], z[3]),
                               Pair16<OutT>::pack(z[4], z[5]), Pair16<OutT>::pack(z[6], z[7]));
            group_end();
          }
        };
        if constexpr (QKV) {
          // The step's 64 columns are one head. Its halves are read one after the other: statistics of the first, of
          // the second, then the second's result and, read again, the first's. A lane that holds the whole head needs
          // 168 registers, which leaves room for one group of warps only (8200 x 2304 x 768 29 us, 65600 x 3 * 1024 x 1024
          // 235; this way 26.5 and 199; two warps per head that exchange their sums 27.1 and 220).
          const int head = out0 >> 6;
          uint32_t r[32];
          auto scaled_half = [&](int h) {
            read32(ca + 32 * h, r);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              scale_cols<8, MX>(r + 8 * g, rs, csa + 32 * h + 8 * g, ba + 32 * h + 8 * g);
              group_end();
            }
          };
          auto pair_of = [&](int j) { return make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])); };
          if (!any) {
            arrive_empty();
            continue;
          }
          if (head >= args.q_heads + args.k_heads) {  // v
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              scaled_half(h);
              if (h == 1) arrive_empty();
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                float z[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = __uint_as_float(r[8 * g + j]);
                stage8(4 * h + g, z);
              }
            }
          } else {
            // Angles of four pairs, read one group ahead of their use; volatile, with the pointers stepped in place,
            // so that the compiler neither reads all of them at once nor keeps an address for each.
            const float *cp = args.rope_cos + pos, *sp = args.rope_sin + pos;
            cp += 16 * static_cast<int64_t>(args.tokens);
            sp += 16 * static_cast<int64_t>(args.tokens);
            float rope[2][8];
            auto load_angles = [&](float(&a)[8]) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                asm volatile(
                    "ld.global.nc.f32 %0, [%2];\n\tld.global.nc.f32 %1, [%3];\n\t"
                    "add.s64 %2, %2, %4;\n\tadd.s64 %3, %3, %4;"
                    : "=&f"(a[2 * j]), "=&f"(a[2 * j + 1]), "+l"(cp), "+l"(sp)
                    : "l"(static_cast<int64_t>(args.tokens) * 4));
            };
            load_angles(rope[0]);
            // Mean and sum of squared differences of each half, then of both: with 32 values each,
            // M2 = M2a + M2b + 16 (mean_a - mean_b)^2.
            float mean[2] = {0.f, 0.f}, square[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              scaled_half(h);
              if (args.norm == FF_NORM_LAYER) {
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int j = 0; j < 16; ++j) sum = add2(sum, pair_of(j));
                mean[h] = (sum.x + sum.y) * (1.f / 32.f);
              }
              float2 sq = make_float2(0.f, 0.f);
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 d = add2(pair_of(j), make_float2(-mean[h], -mean[h]));
                sq = fma2(d, d, sq);
              }
              square[h] = sq.x + sq.y;
            }
            const float diff = mean[0] - mean[1], neg = -0.5f * (mean[0] + mean[1]);
            const float rstd = rsqrtf((square[0] + square[1] + 16.f * diff * diff) * (1.f / 64.f) + args.qk_eps);
            const float2 m2 = make_float2(neg, neg), r2 = make_float2(rstd, rstd);
            const float* const w = normp + (head < args.q_heads ? 0 : 128);  // weights, then biases (zero for RMS)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int h = 1 - k;
              if (k == 1) {
                scaled_half(0);
                arrive_empty();
              }
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                if (k == 0 && g == 3) {
                  cp = args.rope_cos + pos;
                  sp = args.rope_sin + pos;
                }
                if (k == 0 || g < 3) load_angles(rope[(g + 1) & 1]);
                const float* const wg = w + 32 * h + 8 * g;
                float z[8];
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                  const float4 w4 = *reinterpret_cast<const float4*>(wg + 2 * j);
                  const float4 b4 = *reinterpret_cast<const float4*>(wg + 64 + 2 * j);
                  const float2 x[2] = {
                      fma2(add2(pair_of(4 * g + j), m2), mul2(r2, make_float2(w4.x, w4.y)), make_float2(b4.x, b4.y)),
                      fma2(add2(pair_of(4 * g + j + 1), m2), mul2(r2, make_float2(w4.z, w4.w)), make_float2(b4.z, b4.w))};
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    const float c = rope[g & 1][2 * (j + i)], sn = rope[g & 1][2 * (j + i) + 1];
                    z[2 * (j + i)] = x[i].x * c - x[i].y * sn;
                    z[2 * (j + i) + 1] = x[i].x * sn + x[i].y * c;
                  }
                }
                stage8(4 * h + g, z);
              }
            }
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {
            const int sub = acc == 0 ? 1 - k : k;  // the shared columns first
            uint32_t r[32];
            read32(ca + 32 * sub, r);
            if (k == 0) {
              arrive_early();
              wait_residual();
            } else {
              arrive_empty();
            }
            if (!any) continue;
            const float *cs = csa + 32 * sub, *bs = ba + 32 * sub;
            if constexpr (F32OUT) {
              float* const out = static_cast<float*>(args.out);
              const int rows = args.M - m_block < 32 ? args.M - m_block : 32;
              scale_cols<32, MX>(r, rs, cs, bs);
              stage_row128(stg, lane, r);
              __syncwarp();
              const int n = out0 + 32 * sub + lane;
              for (int k = 0; k < rows; ++k)  // one row of 32 columns per store: any row stride and column count
                if (n < args.N)
                  out[static_cast<int64_t>(m_block + k) * args.ldo + n] =
                      *reinterpret_cast<const float*>(stg + k * 128 + (((lane >> 2) ^ (k & 7)) << 4) + (lane & 3) * 4);
              __syncwarp();
            } else {
              // Eight output columns at a time: scale, activate, round, stage.
              if constexpr (SWIGLU) {  // 16 gates, then their 16 ups
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                  scale_cols<8, MX>(r + 8 * g, rs, cs + 8 * g, bs + 8 * g);
                  scale_cols<8, MX>(r + 16 + 8 * g, rs, cs + 16 + 8 * g, bs + 16 + 8 * g);
                  float y[8];
#pragma unroll
                  for (int j = 0; j < 8; j += 2) {
                    const uint32_t *gt = r + 8 * g + j, *up = gt + 16;
                    const float2 h = silu_up2(make_float2(__uint_as_float(gt[0]), __uint_as_float(gt[1])),
                                              make_float2(__uint_as_float(up[0]), __uint_as_float(up[1])));
                    y[j] = h.x;
                    y[j + 1] = h.y;
                  }
                  stage8(2 * sub + g, y);
                }
              } else {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  scale_cols<8, MX>(r + 8 * g, rs, cs + 8 * g, bs + 8 * g);
                  float y[8];
#pragma unroll
                  for (int j = 0; j < 8; j += 2) {
                    float2 v = make_float2(__uint_as_float(r[8 * g + j]), __uint_as_float(r[8 * g + j + 1]));
                    if constexpr (EPI == EPI_GELU_F16) v = gelu2(v);
                    y[j] = v.x;
                    y[j + 1] = v.y;
                  }
                  stage8(4 * sub + g, y);
                }
              }
            }
          }
          if (!ok) break;
          if (!any) continue;
        }
        if constexpr (!F32OUT) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0 && out0 < args.tma_cols) {
            tma_store_2d(&tmC, stg, out0, m_block);
            bulk_commit_group();
          }
          // A TMA store clips its box to whole 16-byte granules of a row: the last out_cols % 8 columns are written
          // one by one by the lane that has staged them.
          const int c = args.tma_cols, left = args.out_cols - c;
          if (left != 0 && c >= out0 && c < out0 + WIDTH && row_ok) {
            const uint4 u = SWIGLU ? staged_chunk64(stg, lane, (c - out0) >> 3) : staged_chunk128(stg, lane, (c - out0) >> 3);
            uint16_t* dst = static_cast<uint16_t*>(args.out) + static_cast<int64_t>(m) * args.ldo + c;
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 7; ++e)
              if (e < left) dst[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
          }
        }
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&pempty[buf]);
    }
    if (!F32OUT && lane == 0) bulk_wait_all();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR)
      tmem_dealloc2(tmem, C::TMEM_COLS);
    else
      tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

struct Fp4Maps {
  CUtensorMap a, w, sa, sw, c, r;
};

template <bool PAIR, bool MX, int EPI, class OutT>
int launch_fp4(const Fp4Maps& t, const Fp4GemmArgs& a, cudaStream_t stream) {
  using C = Fp4Cfg<PAIR, EPI == EPI_QKV_NORM_ROPE>;
  auto kernel = gemm_fp4_kernel<PAIR, MX, EPI, OutT>;
  static int most[64] = {};  // CTAs (pairs) resident at once per device, 0 = not configured yet
  int dev = 0;
  cudaGetDevice(&dev);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  int units = dev >= 0 && dev < 64 ? most[dev] : 0;
  if (units == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
      return check_launch("gemm_fp4: cudaFuncSetAttribute");
    units = sm_count();
    if (PAIR) {
      cfg.gridDim = dim3(2 * (sm_count() / 2));
      if (cudaOccupancyMaxActiveClusters(&units, kernel, &cfg) != cudaSuccess || units < 1)
        return check_launch("gemm_fp4: cudaOccupancyMaxActiveClusters");
    }
    if (dev >= 0 && dev < 64) most[dev] = units;
  }
  const int64_t tiles = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
  cfg.gridDim = dim3((PAIR ? 2 : 1) * static_cast<unsigned>(tiles < units ? tiles : units));
  if (cudaLaunchKernelEx(&cfg, kernel, t.a, t.w, t.sa, t.sw, t.c, t.r, a) != cudaSuccess)
    return check_launch("gemm_fp4_kernel");
  return check_launch("gemm_fp4_kernel");
}

template <bool PAIR, bool MX>
int dispatch_fp4(int epi, int dtype, const Fp4Maps& t, const Fp4GemmArgs& a, cudaStream_t s) {
  const bool bf = dtype == FF_BF16;
  using H = __half;
  using B = __nv_bfloat16;
  switch (epi) {
    case EPI_BIAS:
      if (dtype == FF_F32) return launch_fp4<PAIR, MX, EPI_BIAS, float>(t, a, s);
      return bf ? launch_fp4<PAIR, MX, EPI_BIAS, B>(t, a, s) : launch_fp4<PAIR, MX, EPI_BIAS, H>(t, a, s);
    case EPI_GELU_F16: return bf ? launch_fp4<PAIR, MX, EPI_GELU_F16, B>(t, a, s) : launch_fp4<PAIR, MX, EPI_GELU_F16, H>(t, a, s);
    case EPI_SWIGLU: return bf ? launch_fp4<PAIR, MX, EPI_SWIGLU, B>(t, a, s) : launch_fp4<PAIR, MX, EPI_SWIGLU, H>(t, a, s);
    case EPI_RESIDUAL: return bf ? launch_fp4<PAIR, MX, EPI_RESIDUAL, B>(t, a, s) : launch_fp4<PAIR, MX, EPI_RESIDUAL, H>(t, a, s);
    default:
      if constexpr (PAIR) {
        set_error("ff_gemm_fp4: no pair tiles for the QKV epilogue");
        return FF_ERR_INVALID_ARGUMENT;
      } else {
        return bf ? launch_fp4<false, MX, EPI_QKV_NORM_ROPE, B>(t, a, s) : launch_fp4<false, MX, EPI_QKV_NORM_ROPE, H>(t, a, s);
      }
  }
}

int sf_map(CUtensorMap* map, const uint8_t* scales, int rows, int cols, bool mx) {
  const int ch = sf_chunks_per_step(mx);
  const uint64_t chunks = static_cast<uint64_t>((rows + 127) / 128) * ((cols + kFp4Step - 1) / kFp4Step) * ch;
  return make_tmap_2d_pitched(map, scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, kSfChunk / 4, chunks, kSfChunk,
                              kSfChunk / 4, static_cast<uint32_t>(ch), CU_TENSOR_MAP_SWIZZLE_NONE);
}

int code_map(CUtensorMap* map, const uint8_t* codes, int rows, int cols) {
  const uint64_t pitch = static_cast<uint64_t>(fp4_row_bytes(cols));
  return make_tmap_2d_pitched(map, codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, pitch, static_cast<uint64_t>(rows), pitch, 128,
                              128, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Whether 256 x 256 tiles over CTA pairs are the faster choice: rounds of tiles times the time of one, measured at
// K = 1024 and 8192: 128 x 128 tiles 1.45 us (their epilogue) or 0.30 us per 256 columns of K, pair tiles 2.75 us or
// 0.415 us. (65600 x 5504 x 1024 SwiGLU 206 us in pairs, 230 us without; 65600 x 1024 x 2730 101 and 139 us;
// 8200 x 4096 x 768 20.7 and 19.9 us.)
bool choose_pair_fp4(int M, int N, int K) {
  const int64_t steps = (K + kFp4Step - 1) / kFp4Step, sms = sm_count(), pairs = sms / 2;
  const int64_t single = static_cast<int64_t>((M + 127) / 128) * ((N + 127) / 128);
  const int64_t pair = static_cast<int64_t>((M + 255) / 256) * ((N + 255) / 256);
  const double t_single = static_cast<double>((single + sms - 1) / sms) * (steps > 4 ? 0.30 * steps : 1.45);
  const double t_pair = static_cast<double>((pair + pairs - 1) / pairs) * (steps > 6 ? 0.415 * steps : 2.75);
  return t_pair < t_single;
}

}  // namespace

int gemm_fp4(const Fp4Operand& A, const Fp4Operand& W, int fmt, int M, int N, int K, const ff_fp4_epilogue* e, int tile,
             bool w_const, cudaStream_t stream) {
  FF_REQUIRE(fmt == FF_FP4_NV || fmt == FF_FP4_MX, "ff_gemm_fp4: unknown format %d", fmt);
  FF_REQUIRE(e != nullptr, "ff_gemm_fp4: NULL epilogue");
  FF_REQUIRE(M >= 0 && N >= 1 && K >= 1 && M <= (1 << 30) && N <= (1 << 30) && K <= (1 << 24), "ff_gemm_fp4: bad shape M=%d N=%d K=%d",
             M, N, K);
  const int epi = e->kind;
  FF_REQUIRE(epi == EPI_BIAS || epi == EPI_GELU_F16 || epi == EPI_SWIGLU || epi == EPI_RESIDUAL || epi == EPI_QKV_NORM_ROPE,
             "ff_gemm_fp4: unknown epilogue %d", epi);
  FF_REQUIRE(e->out_dtype == FF_F16 || e->out_dtype == FF_BF16 || (e->out_dtype == FF_F32 && epi == EPI_BIAS),
             "ff_gemm_fp4: output type %d is not available for epilogue %d", e->out_dtype, epi);
  FF_REQUIRE(tile == 0 || tile == 128 || tile == FF_TILE_PAIR256, "ff_gemm_fp4: tile must be 0, 128 or FF_TILE_PAIR256 (got %d)",
             tile);
  FF_REQUIRE(epi != EPI_QKV_NORM_ROPE || tile != FF_TILE_PAIR256, "ff_gemm_fp4: no pair tiles for the QKV epilogue");
  FF_REQUIRE(epi != EPI_SWIGLU || N % 32 == 0, "ff_gemm_fp4: SwiGLU needs N %% 32 == 0 (N=%d)", N);
  const int out_cols = epi == EPI_SWIGLU ? (e->out_cols > 0 ? e->out_cols : N / 2) : N;
  FF_REQUIRE(epi != EPI_SWIGLU || out_cols <= N / 2, "ff_gemm_fp4: SwiGLU writes at most N / 2 columns (out_cols=%d, N=%d)",
             out_cols, N);
  FF_REQUIRE(e->ldo >= out_cols, "ff_gemm_fp4: output row stride %lld for %d columns", static_cast<long long>(e->ldo), out_cols);
  // A single row is never stepped over: any stride will do, rounded up to what the tensor maps take.
  const int64_t ldo = M == 1 ? (e->ldo + 7) / 8 * 8 : e->ldo, ldr = M == 1 ? (e->ldr + 7) / 8 * 8 : e->ldr;
  if (epi == EPI_QKV_NORM_ROPE) {
    FF_REQUIRE(e->norm == FF_NORM_RMS || e->norm == FF_NORM_LAYER, "ff_gemm_fp4: unknown head norm %d", e->norm);
    FF_REQUIRE(e->q_heads >= 0 && e->k_heads >= 0 && N % 64 == 0 && static_cast<int64_t>(e->q_heads) + e->k_heads <= N / 64,
               "ff_gemm_fp4: %d + %d heads of 64 columns do not fit N=%d", e->q_heads, e->k_heads, N);
    FF_REQUIRE(e->q_w && e->k_w && e->rope_cos && e->rope_sin && e->tokens >= 1 && e->tokens <= (1 << 25),
               "ff_gemm_fp4: the QKV epilogue needs q and k norm weights, rotation tables and tokens");
  }
  if (M == 0) return FF_OK;
  FF_REQUIRE(A.codes && A.scales && W.codes && W.scales && e->out, "ff_gemm_fp4: NULL pointer");
  FF_REQUIRE(fmt == FF_FP4_MX || (A.row_scale && W.row_scale), "ff_gemm_fp4: FF_FP4_NV needs row and column scales");
  FF_REQUIRE(epi != EPI_RESIDUAL || (e->residual && e->ldr >= N), "ff_gemm_fp4: the residual epilogue needs the residual and its row stride");
  FF_REQUIRE(aligned16(A.codes) && aligned16(A.scales) && aligned16(W.codes) && aligned16(W.scales),
             "ff_gemm_fp4: codes and scales must be 16-byte aligned");
  const bool f32 = e->out_dtype == FF_F32;
  FF_REQUIRE(f32 || (aligned16(e->out) && ldo % 8 == 0), "ff_gemm_fp4: 16-bit outputs need 16-byte aligned rows (ldo %% 8 == 0)");
  FF_REQUIRE(!f32 || reinterpret_cast<uintptr_t>(e->out) % 4 == 0, "ff_gemm_fp4: out is not aligned to its type");
  FF_REQUIRE(epi != EPI_RESIDUAL || (aligned16(e->residual) && ldr % 8 == 0), "ff_gemm_fp4: residual rows must be 16-byte aligned");

  const bool pair = tile == FF_TILE_PAIR256 || (tile == 0 && epi != EPI_QKV_NORM_ROPE && choose_pair_fp4(M, N, K));
  Fp4Maps t;
  const bool mx = fmt == FF_FP4_MX;
  int rc;
  if ((rc = code_map(&t.a, A.codes, M, K)) != FF_OK || (rc = code_map(&t.w, W.codes, N, K)) != FF_OK ||
      (rc = sf_map(&t.sa, A.scales, M, K, mx)) != FF_OK || (rc = sf_map(&t.sw, W.scales, N, K, mx)) != FF_OK)
    return rc;
  t.c = t.a;
  t.r = t.a;
  const CUtensorMapDataType dt = e->out_dtype == FF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (!f32) {
    const bool narrow = epi == EPI_SWIGLU;  // 32 output columns per warp
    // whole 16-byte granules only (none: a map that no store uses); the kernel writes the rest of a row itself
    rc = make_tmap_2d_pitched(&t.c, e->out, dt, 2, static_cast<uint64_t>(out_cols < 8 ? 8 : out_cols & ~7), static_cast<uint64_t>(M),
                              static_cast<uint64_t>(ldo) * 2, narrow ? 32 : 64, 32,
                              narrow ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != FF_OK) return rc;
  }
  if (epi == EPI_RESIDUAL) {
    rc = make_tmap_2d_pitched(&t.r, e->residual, dt, 2, static_cast<uint64_t>(N), static_cast<uint64_t>(M),
                              static_cast<uint64_t>(ldr) * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != FF_OK) return rc;
  }
  Fp4GemmArgs a{};
  a.M = M;
  a.N = N;
  a.K = K;
  a.num_kb = (K + kFp4Step - 1) / kFp4Step;
  a.tiles_m = pair ? (M + 255) / 256 : (M + 127) / 128;
  a.tiles_n = pair ? (N + 255) / 256 : (N + 127) / 128;
  FF_REQUIRE(static_cast<int64_t>(a.tiles_m) * a.tiles_n < (1ll << 31), "ff_gemm_fp4: too many tiles");
  a.row_scale = A.row_scale;
  a.col_scale = W.row_scale;
  a.bias = e->bias;
  a.out = e->out;
  a.ldo = ldo;
  a.out_cols = out_cols;
  a.tma_cols = out_cols & ~7;
  a.norm = e->norm;
  a.q_heads = e->q_heads;
  a.k_heads = e->k_heads;
  a.qk_eps = e->qk_eps;
  a.q_w = e->q_w;
  a.k_w = e->k_w;
  if (e->norm == FF_NORM_LAYER) {  // an RMS norm has no bias, whatever the caller set
    a.q_b = e->q_b;
    a.k_b = e->k_b;
  }
  a.rope_cos = e->rope_cos;
  a.rope_sin = e->rope_sin;
  a.tokens = e->tokens > 0 ? e->tokens : 1;
  a.w_const = w_const;
  a.err = device_error_word();
  FF_REQUIRE(a.err != nullptr, "ff_gemm_fp4: no device error word");
  if (mx) return pair ? dispatch_fp4<true, true>(epi, e->out_dtype, t, a, stream) : dispatch_fp4<false, true>(epi, e->out_dtype, t, a, stream);
  return pair ? dispatch_fp4<true, false>(epi, e->out_dtype, t, a, stream) : dispatch_fp4<false, false>(epi, e->out_dtype, t, a, stream);
}

}  // namespace ff

using namespace ff;

extern "C" int ff_gemm_fp4(const uint8_t* A, const uint8_t* A_scales, const float* row_scale, const uint8_t* W,
                           const uint8_t* W_scales, const float* col_scale, int fmt, int M, int N, int K,
                           const ff_fp4_epilogue* epilogue, int tile, void* stream) {
  return gemm_fp4({A, A_scales, row_scale}, {W, W_scales, col_scale}, fmt, M, N, K, epilogue, tile, false,
                  static_cast<cudaStream_t>(stream));
}

namespace {
constexpr int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
}  // namespace

extern "C" int64_t ff_linear_fp4_workspace_bytes(int M, int K, int fmt) {
  if (M < 0 || K < 1 || (fmt != FF_FP4_NV && fmt != FF_FP4_MX)) return 0;
  return up256(ff_fp4_code_bytes(M, K)) + up256(ff_fp4_scale_bytes(M, K, fmt)) + up256(4ll * M);
}

extern "C" int ff_linear_fp4(const void* x, int dtype, int64_t ldx, const float* gamma, const float* beta, float eps,
                             const uint8_t* W, const uint8_t* W_scales, const float* col_scale, int fmt, int M, int N,
                             int K, const ff_fp4_epilogue* epilogue, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  FF_REQUIRE(M >= 0 && K >= 1, "ff_linear_fp4: bad shape M=%d N=%d K=%d", M, N, K);
  FF_REQUIRE(fmt == FF_FP4_NV || fmt == FF_FP4_MX, "ff_linear_fp4: unknown format %d", fmt);
  FF_REQUIRE(M == 0 || (workspace != nullptr && aligned16(workspace) &&
                        workspace_bytes >= ff_linear_fp4_workspace_bytes(M, K, fmt)),
             "ff_linear_fp4: workspace must be 16-byte aligned and hold %lld bytes (got %lld)",
             static_cast<long long>(ff_linear_fp4_workspace_bytes(M, K, fmt)), static_cast<long long>(workspace_bytes));
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + up256(ff_fp4_code_bytes(M, K));
  float* row_scale = reinterpret_cast<float*>(scales + up256(ff_fp4_scale_bytes(M, K, fmt)));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = quantize_fp4(x, dtype, ldx, gamma, beta, eps, M, K, fmt, codes, scales, row_scale, s);
  if (rc != FF_OK) return rc;
  // The product may start on the weights while the quantisation runs: the quantisation kernel itself began
  // after everything before it in the stream was done, so nothing that is still running writes them.
  return gemm_fp4({codes, scales, row_scale}, {W, W_scales, col_scale}, fmt, M, N, K, epilogue, 0, true, s);
}
