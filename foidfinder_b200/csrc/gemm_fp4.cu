// Product of block-scaled 4-bit operands on tcgen05, with the epilogues of a transformer's linear layers:
//   y[m, n] = (sum_k A[m, k] SA[m, k / B] W[n, k] SW[n, k / B]) * row_scale[m] * col_scale[n] + bias[n]
// B = 16 (FF_FP4_NV) or 32 (FF_FP4_MX) columns per block scale. The tensor cores apply the block scales while
// they multiply (kind::mxf4nvf4 / kind::mxf4, f32 accumulators in TMEM); the row scales, which are powers of
// two, and the bias are applied in f32 in the epilogue, which rounds once, to the output's type.
//
// One CTA per SM, 320 threads, persistent over tiles:
//   warp 0     TMA producer: per stage 256 columns (128 bytes of codes, 128-byte swizzle) of A and W rows and
//              their scale chunks
//   warp 1     TMEM allocator; copies each stage's scale chunks to TMEM (tcgen05.cp, in order with the MMAs of
//              the same thread) and issues the MMAs, 64 columns each
//   warps 2-9  epilogue: two warps per TMEM lane quarter, one output row per lane
// Tiles: 128 x 128 per CTA, or (PAIR) 256 x 256 over a cluster of two CTAs, where each CTA loads its 128 rows
// of A, half of W's 256 rows and all of the tile's W scales (each SM's tensor core reads them from its own
// TMEM), and shared memory moves half as many bytes per multiply-add.
#include "common.h"
#include "fp4.cuh"
#include "gemm_fp4.h"
#include "gemm_tc.cuh"

namespace ff {

namespace {

template <bool PAIR, bool RES>
struct Fp4Cfg {
  static constexpr int BN = PAIR ? 256 : 128;
  static constexpr int TILE_M = PAIR ? 256 : 128;
  static constexpr int HALF = BN / 2;  // columns per epilogue warp
  static constexpr int CODE_BYTES = 128 * 128;  // 128 rows of A, or of W, per CTA and stage
  static constexpr int SFA_BYTES = 4 * kSfChunk;
  static constexpr int SFB_BYTES = (BN / 128) * 4 * kSfChunk;
  static constexpr int STAGE_BYTES = 2 * CODE_BYTES + SFA_BYTES + SFB_BYTES;
  static constexpr int STAGES = PAIR || RES ? 4 : 5;
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int STAGING = RES ? 8192 : 4096;  // per epilogue warp: 32 rows x 128 B, twice with a residual
  static constexpr int COLP = 2 * HALF * 4;          // per epilogue warp: column scales and biases of its columns
  static constexpr int NORM_BYTES = 4 * 64 * 4;      // q and k norm weights and biases
  static constexpr int BAR_BYTES = 512;
  static constexpr int SMEM =
      1024 + STAGES * STAGE_BYTES + EPI_WARPS * (STAGING + COLP) + NORM_BYTES + BAR_BYTES;
  static constexpr int ACCS = PAIR ? 1 : 2;
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr uint32_t SF_BASE = 256;               // TMEM column of the scales
  static constexpr uint32_t SF_COLS = 16 + 4 * (BN / 32);  // per stage: A's, then W's
  static_assert(STAGE_BYTES % 1024 == 0, "stages keep the swizzle's alignment");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// tanh GELU: x * sigmoid(2 sqrt(2 / pi) (x + 0.044715 x^3)), MUFU ex2 and rcp (a few ulp).
__device__ __forceinline__ float gelu_sigmoid(float x) {
  const float t = -2.302208198f * (x + 0.044715f * x * x * x);  // -2 sqrt(2 / pi) log2 e
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2_approx(fminf(t, 126.f))));
  return x * r;
}

// y[j] = acc[j] * (rs * cs[j]) + bias[j]; cs and bias in shared memory (read by every lane at once).
__device__ __forceinline__ void scale32(const uint32_t (&r)[32], float rs, const float* cs, const float* bias,
                                        float (&y)[32]) {
  const float2 rs2 = make_float2(rs, rs);
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 c = *reinterpret_cast<const float4*>(cs + j);
    const float4 b = *reinterpret_cast<const float4*>(bias + j);
    const float2 lo = fma2(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])),
                           mul2(rs2, make_float2(c.x, c.y)), make_float2(b.x, b.y));
    const float2 hi = fma2(make_float2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])),
                           mul2(rs2, make_float2(c.z, c.w)), make_float2(b.z, b.w));
    y[j] = lo.x;
    y[j + 1] = lo.y;
    y[j + 2] = hi.x;
    y[j + 3] = hi.y;
  }
}

// The scale copies and MMAs of one stage.
template <bool PAIR, bool MX, class C>
__device__ __forceinline__ void fp4_stage_mmas(uint32_t d, uint32_t sa, uint32_t sf, int steps, bool first) {
  constexpr int CH = sf_chunks_per_step(MX);
  const uint32_t sfa = sf, sfb = sf + 16;
  const uint32_t ssa = sa + 2 * C::CODE_BYTES, ssb = ssa + C::SFA_BYTES;
  constexpr int BT = C::BN / 128;
#pragma unroll
  for (int g = 0; g < CH; ++g) {
    tc_cp_sf<PAIR>(sfa + 4 * g, sdesc_sf(ssa + g * kSfChunk));
#pragma unroll
    for (int t = 0; t < BT; ++t) tc_cp_sf<PAIR>(sfb + 4 * BT * g + 4 * t, sdesc_sf(ssb + (t * CH + g) * kSfChunk));
  }
  const uint64_t adesc = sdesc_k_sw128(sa), bdesc = sdesc_k_sw128(sa + C::CODE_BYTES);
  constexpr uint32_t idesc = idesc_fp4(C::TILE_M, C::BN, MX);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k < steps) {
      const int g = MX ? k / 2 : k;
      mma_fp4<PAIR, MX>(d, adesc + 2 * k, bdesc + 2 * k, idesc | (MX ? idesc_sf_id((k & 1) * 2) : 0u), sfa + 4 * g,
                        sfb + 4 * BT * g, !(first && k == 0));
    }
  }
}

template <bool PAIR, int EPI, class OutT>
__global__ void __launch_bounds__(Fp4Cfg<PAIR, EPI == EPI_RESIDUAL>::THREADS, 1)
    gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSW,
                    const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmR,
                    const Fp4GemmArgs args) {
  constexpr bool RES = EPI == EPI_RESIDUAL;
  constexpr bool F32OUT = sizeof(OutT) == 4;
  using C = Fp4Cfg<PAIR, RES>;
  constexpr int STAGES = C::STAGES, BN = C::BN, HALF = C::HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + STAGES * C::STAGE_BYTES;
  float* colp = reinterpret_cast<float*>(staging + C::EPI_WARPS * C::STAGING);
  float* normp = colp + C::EPI_WARPS * 2 * HALF;  // q weight, q bias, k weight, k bias
  uint64_t* full = reinterpret_cast<uint64_t*>(normp + 4 * 64);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + C::ACCS;
  uint64_t* drain = tempty + C::ACCS;
  uint64_t* resbar = drain + 1;  // two per epilogue warp (EPI_RESIDUAL)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(resbar + 2 * C::EPI_WARPS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_n = args.tiles_n;
  const int tiles = args.tiles_m * tiles_n;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int unit = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int units = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
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
    for (int a = 0; a < C::ACCS; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], (PAIR ? 2 : 1) * C::EPI_WARPS);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < 2 * C::EPI_WARPS; ++i) mbar_init(&resbar[i], 1);
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
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int last_phase[STAGES];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) last_phase[s] = -1;
      const int ch = args.mx ? 2 : 4;  // scale chunks per stage and 128-row tile
      const uint32_t stage_bytes = 2 * C::CODE_BYTES + (1 + BN / 128) * ch * kSfChunk;
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
      const int pre = (args.w_const && unit < tiles) ? (args.num_kb < STAGES ? args.num_kb : STAGES) : 0;
      for (int kb = 0; kb < pre; ++kb) {
        expect(&full[kb]);
        load_w(smem + kb * C::STAGE_BYTES, &full[kb], kb, unit % tiles_n);
      }
      pdl_wait();
      bool ok = true, first = true;
      for (int t = unit; t < tiles && ok; t += units) {
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
          if (last_phase[s] >= 0) {
            const uint32_t addr = smem_u32(&full[s]);
            const unsigned long long t0 = globaltimer();
            while (!mbar_try_wait(addr, static_cast<uint32_t>(last_phase[s])) && globaltimer() - t0 < kWaitLimitNs) {
            }
          }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ scale copies and MMAs (the even CTA of a pair)
    pdl_wait();
    if (lane == 0 && leader) {
      auto commit_both = [&](uint64_t* bar) {
        if constexpr (PAIR)
          tc_commit2_both(bar);
        else
          tc_commit(bar);
      };
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0, sf_buf = 0;
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units) {
        if (!wait(&tempty[acc], acc_phase ^ 1u, kDevTimeoutTmemEmpty)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(acc * BN);
        for (int kb = 0; kb < args.num_kb; ++kb) {
          if (!wait(&full[stage], phase, kDevTimeoutTmaFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * C::STAGE_BYTES);
          const uint32_t sf = tmem + C::SF_BASE + sf_buf * C::SF_COLS;
          const int left = (args.K - kb * kFp4Step + 63) >> 6;  // 64-column steps to the end of the row
          if (args.mx)
            fp4_stage_mmas<PAIR, true, C>(d, sa, sf, left, kb == 0);
          else
            fp4_stage_mmas<PAIR, false, C>(d, sa, sf, left, kb == 0);
          commit_both(&empty[stage]);
          sf_buf ^= 1u;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        commit_both(&tfull[acc]);
        if (++acc == C::ACCS) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      // Drain: every MMA this thread issued must finish before TMEM is released.
      if constexpr (PAIR)
        tc_commit2(drain);
      else
        tc_commit(drain);
      const uint32_t addr = smem_u32(drain);
      const unsigned long long t0 = globaltimer();
      while (!mbar_try_wait(addr, 0)) {
        if (globaltimer() - t0 > kWaitLimitNs) {
          atomicCAS(args.err, 0, kDevTimeoutDrain);
          break;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    pdl_wait();
    const int ew = warp - 2;
    const int q = warp & 3;    // TMEM lane quarter
    const int half = ew >> 2;  // which half of the tile's columns
    uint8_t* const stg = staging + ew * C::STAGING;
    float* const cs_s = colp + ew * 2 * HALF;
    float* const b_s = cs_s + HALF;
    constexpr bool SPLIT = EPI == EPI_SWIGLU && BN == 128;  // the warp's columns: 32 gates and their 32 ups
    if constexpr (EPI == EPI_QKV_NORM_ROPE) {
      for (int i = threadIdx.x - 64; i < 64; i += 256) {
        normp[i] = args.q_w[i];
        normp[64 + i] = args.q_b != nullptr ? args.q_b[i] : 0.f;
        normp[128 + i] = args.k_w[i];
        normp[192 + i] = args.k_b != nullptr ? args.k_b[i] : 0.f;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the eight epilogue warps
    }
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t res_phase[2] = {0, 0};
    bool ok = true;
    for (int t = unit; t < tiles; t += units) {
      const int tm = t / tiles_n, tn = t % tiles_n;
      const int m_block = tm * C::TILE_M + static_cast<int>(rank) * 128 + q * 32;
      const int m = m_block + lane;
      const bool row_ok = m < args.M;
      const bool any = m_block < args.M;  // some row of this warp is real
      const int n_tile = tn * BN;
      // Column scales and biases of this warp's columns (zero past N), row scale and rotation angles: read
      // before the wait for the accumulator.
      __syncwarp();
      for (int i = lane; i < HALF; i += 32) {
        const int n = n_tile + (SPLIT ? (i < 32 ? half * 32 + i : 32 + half * 32 + i) : half * HALF + i);
        const bool in = n < args.N;
        cs_s[i] = in ? (args.col_scale != nullptr ? __ldg(args.col_scale + n) : 1.f) : 0.f;
        b_s[i] = in && args.bias != nullptr ? __ldg(args.bias + n) : 0.f;
      }
      __syncwarp();
      const float rs = row_ok ? (args.row_scale != nullptr ? __ldg(args.row_scale + m) : 1.f) : 0.f;
      float rope_c[EPI == EPI_QKV_NORM_ROPE ? 32 : 1], rope_s[EPI == EPI_QKV_NORM_ROPE ? 32 : 1];
      if constexpr (EPI == EPI_QKV_NORM_ROPE) {
        if (n_tile + half * HALF < 64 * (args.q_heads + args.k_heads)) {
          const int pos = (row_ok ? m : 0) % args.tokens;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            rope_c[j] = __ldg(args.rope_cos + static_cast<int64_t>(j) * args.tokens + pos);
            rope_s[j] = __ldg(args.rope_sin + static_cast<int64_t>(j) * args.tokens + pos);
          }
        }
      }
      if constexpr (RES) {
        // The first chunk of the residual comes in while the mainloop runs.
        if (any && lane == 0) {
          bulk_wait_read_all();
          mbar_arrive_expect_tx(&resbar[2 * ew], 4096);
          tma_load_2d(stg, &tmR, &resbar[2 * ew], n_tile + half * HALF, m_block);
        }
      }
      if (!wait(&tfull[acc], acc_phase, kDevTimeoutTmemFull)) {
        ok = false;
        if constexpr (RES) {  // let the residual copy land before the CTA exits
          if (any && lane == 0) mbar_wait(&resbar[2 * ew], res_phase[0], abort_flag, args.err, kDevTimeoutDrain);
        }
        break;
      }
      tc_fence_after();
      const uint32_t tbase = tmem + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BN);
      // A TMA store clips its box to whole 16-byte granules of a row: the last out_cols % 8 columns, when they lie
      // in the 16-bit columns [n0, n0 + width) that this lane has staged, are written one by one.
      auto store_ragged = [&](int n0, int width, uint4 u) {
        const int c = args.tma_cols, left = args.out_cols - c;
        if (left == 0 || c < n0 || c >= n0 + width || !row_ok) return;
        uint16_t* dst = static_cast<uint16_t*>(args.out) + static_cast<int64_t>(m) * args.ldo + c;
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < left) dst[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
      };
      if (any) {
        if constexpr (F32OUT) {
          float* const out = static_cast<float*>(args.out);
          const int rows = args.M - m_block < 32 ? args.M - m_block : 32;
#pragma unroll 1
          for (int c = 0; c < HALF; c += 32) {
            const int n0 = n_tile + half * HALF + c;
            if (n0 >= args.N) break;
            uint32_t r[32];
            __syncwarp();
            tmem_ld32(tbase + half * HALF + c, r);
            tmem_ld_wait();
            float y[32];
            scale32(r, rs, cs_s + c, b_s + c, y);
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(y[j]);
            stage_row128(stg, lane, r);
            __syncwarp();
            for (int i = 0; i < rows; ++i)  // one row of 32 columns per store: any row stride and column count
              if (n0 + lane < args.N)
                out[static_cast<int64_t>(m_block + i) * args.ldo + n0 + lane] =
                    *reinterpret_cast<const float*>(stg + i * 128 + (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4);
          }
        } else if constexpr (EPI == EPI_SWIGLU) {
          constexpr int OUTS = BN == 256 ? 64 : 32;  // output columns per warp
          const int col0 = (n_tile >> 1) + half * OUTS;
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
#pragma unroll
          for (int sub = 0; sub < OUTS / 32; ++sub) {
            uint32_t rg[32], ru[32];
            const int ig = SPLIT ? 0 : sub * 32, iu = SPLIT ? 32 : 64 + sub * 32;  // among the warp's columns
            const int cg = SPLIT ? half * 32 : half * 128 + sub * 32;
            __syncwarp();
            tmem_ld32(tbase + cg, rg);
            tmem_ld32(tbase + cg + 64, ru);
            tmem_ld_wait();
            float g[32], u[32];
            scale32(rg, rs, cs_s + ig, b_s + ig, g);
            scale32(ru, rs, cs_s + iu, b_s + iu, u);
            uint32_t packed[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 h = silu_mul2(make_float2(g[2 * j], g[2 * j + 1]), make_float2(u[2 * j], u[2 * j + 1]));
              packed[j] = Pair16<OutT>::pack(h.x, h.y);
            }
            if constexpr (OUTS == 64)
              stage_half_row128(stg, lane, sub, packed);
            else
              stage_row64(stg, lane, packed);
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0 && col0 < args.tma_cols) {
            tma_store_2d(&tmC, stg, col0, m_block);
            bulk_commit_group();
          }
          const int rc = (args.tma_cols - col0) >> 3;
          store_ragged(col0, OUTS, OUTS == 64 ? staged_chunk128(stg, lane, rc & 7) : staged_chunk64(stg, lane, rc & 3));
        } else {
#pragma unroll
          for (int ch = 0; ch < HALF / 64; ++ch) {
            const int c0 = half * HALF + ch * 64;
            const int n0 = n_tile + c0;
            uint8_t* const buf = stg + (RES ? (ch & 1) * 4096 : 0);
            if constexpr (RES) {
              // The next chunk's residual into the other buffer, then this chunk's.
              if (lane == 0 && ch + 1 < HALF / 64) {
                bulk_wait_read_all();
                mbar_arrive_expect_tx(&resbar[2 * ew + ((ch + 1) & 1)], 4096);
                tma_load_2d(stg + ((ch + 1) & 1) * 4096, &tmR, &resbar[2 * ew + ((ch + 1) & 1)], n0 + 64, m_block);
              }
              if (!mbar_wait(&resbar[2 * ew + (ch & 1)], res_phase[ch & 1], abort_flag, args.err, kDevTimeoutTmaFull))
                ok = false;
              res_phase[ch & 1] ^= 1u;
            } else {
              if (lane == 0) bulk_wait_read_all();
            }
            __syncwarp();
            if constexpr (EPI == EPI_QKV_NORM_ROPE) {
              // A chunk is one head of 64 columns.
              float y[64];
#pragma unroll
              for (int sub = 0; sub < 2; ++sub) {
                uint32_t r[32];
                __syncwarp();
                tmem_ld32(tbase + c0 + sub * 32, r);
                tmem_ld_wait();
                float h[32];
                scale32(r, rs, cs_s + ch * 64 + sub * 32, b_s + ch * 64 + sub * 32, h);
#pragma unroll
                for (int j = 0; j < 32; ++j) y[sub * 32 + j] = h[j];
              }
              const int head = n0 >> 6;
              if (head < args.q_heads + args.k_heads) {
                const float* w = normp + (head < args.q_heads ? 0 : 128);
                float mean = 0.f;
                if (args.norm == FF_NORM_LAYER) {
#pragma unroll
                  for (int j = 0; j < 64; ++j) mean += y[j];
                  mean *= 1.f / 64.f;
                }
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                  y[j] -= mean;
                  ss = fmaf(y[j], y[j], ss);
                }
                const float rstd = rsqrtf(ss * (1.f / 64.f) + args.qk_eps);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  const float x0 = fmaf(y[2 * j] * rstd, w[2 * j], w[64 + 2 * j]);
                  const float x1 = fmaf(y[2 * j + 1] * rstd, w[2 * j + 1], w[64 + 2 * j + 1]);
                  y[2 * j] = x0 * rope_c[j] - x1 * rope_s[j];
                  y[2 * j + 1] = x0 * rope_s[j] + x1 * rope_c[j];
                }
              }
#pragma unroll
              for (int sub = 0; sub < 2; ++sub) {
                uint32_t packed[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) packed[j] = Pair16<OutT>::pack(y[sub * 32 + 2 * j], y[sub * 32 + 2 * j + 1]);
                stage_half_row128(buf, lane, sub, packed);
              }
            } else {
#pragma unroll
              for (int sub = 0; sub < 2; ++sub) {
                uint32_t r[32];
                __syncwarp();
                tmem_ld32(tbase + c0 + sub * 32, r);
                tmem_ld_wait();
                float y[32];
                scale32(r, rs, cs_s + ch * 64 + sub * 32, b_s + ch * 64 + sub * 32, y);
                if constexpr (EPI == EPI_GELU_F16) {
#pragma unroll
                  for (int j = 0; j < 32; ++j) y[j] = gelu_sigmoid(y[j]);
                }
                if constexpr (RES) {
#pragma unroll
                  for (int c = 0; c < 4; ++c) {
                    const uint4 u = staged_chunk128(buf, lane, 4 * sub + c);
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                      const float2 f = Pair16<OutT>::unpack(w[j]);
                      y[8 * c + 2 * j] += f.x;
                      y[8 * c + 2 * j + 1] += f.y;
                    }
                  }
                }
                uint32_t packed[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) packed[j] = Pair16<OutT>::pack(y[2 * j], y[2 * j + 1]);
                stage_half_row128(buf, lane, sub, packed);
              }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && n0 < args.tma_cols) {
              tma_store_2d(&tmC, buf, n0, m_block);
              bulk_commit_group();
            }
            store_ragged(n0, 64, staged_chunk128(buf, lane, (args.tma_cols - n0) >> 3 & 7));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR && !leader)
          mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0u));
        else
          mbar_arrive(&tempty[acc]);
      }
      if (!ok) break;
      if (++acc == C::ACCS) {
        acc = 0;
        acc_phase ^= 1u;
      }
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

template <bool PAIR, int EPI, class OutT>
int launch_fp4(const Fp4Maps& t, const Fp4GemmArgs& a, cudaStream_t stream) {
  using C = Fp4Cfg<PAIR, EPI == EPI_RESIDUAL>;
  auto kernel = gemm_fp4_kernel<PAIR, EPI, OutT>;
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

template <bool PAIR>
int dispatch_fp4(int epi, int dtype, const Fp4Maps& t, const Fp4GemmArgs& a, cudaStream_t s) {
  const bool bf = dtype == FF_BF16;
  using H = __half;
  using B = __nv_bfloat16;
  switch (epi) {
    case EPI_BIAS:
      if (dtype == FF_F32) return launch_fp4<PAIR, EPI_BIAS, float>(t, a, s);
      return bf ? launch_fp4<PAIR, EPI_BIAS, B>(t, a, s) : launch_fp4<PAIR, EPI_BIAS, H>(t, a, s);
    case EPI_GELU_F16: return bf ? launch_fp4<PAIR, EPI_GELU_F16, B>(t, a, s) : launch_fp4<PAIR, EPI_GELU_F16, H>(t, a, s);
    case EPI_SWIGLU: return bf ? launch_fp4<PAIR, EPI_SWIGLU, B>(t, a, s) : launch_fp4<PAIR, EPI_SWIGLU, H>(t, a, s);
    case EPI_RESIDUAL: return bf ? launch_fp4<PAIR, EPI_RESIDUAL, B>(t, a, s) : launch_fp4<PAIR, EPI_RESIDUAL, H>(t, a, s);
    default:
      return bf ? launch_fp4<PAIR, EPI_QKV_NORM_ROPE, B>(t, a, s) : launch_fp4<PAIR, EPI_QKV_NORM_ROPE, H>(t, a, s);
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
  FF_REQUIRE(epi != EPI_SWIGLU || N % 128 == 0, "ff_gemm_fp4: SwiGLU needs N %% 128 == 0 (N=%d)", N);
  const int out_cols = epi == EPI_SWIGLU ? (e->out_cols > 0 ? e->out_cols : N / 2) : N;
  FF_REQUIRE(epi != EPI_SWIGLU || out_cols <= N / 2, "ff_gemm_fp4: SwiGLU writes at most N / 2 columns (out_cols=%d, N=%d)",
             out_cols, N);
  FF_REQUIRE(e->ldo >= out_cols, "ff_gemm_fp4: output row stride %lld for %d columns", static_cast<long long>(e->ldo), out_cols);
  if (epi == EPI_QKV_NORM_ROPE) {
    FF_REQUIRE(e->norm == FF_NORM_RMS || e->norm == FF_NORM_LAYER, "ff_gemm_fp4: unknown head norm %d", e->norm);
    FF_REQUIRE(e->q_heads >= 0 && e->k_heads >= 0 && N % 64 == 0 && static_cast<int64_t>(e->q_heads) + e->k_heads <= N / 64,
               "ff_gemm_fp4: %d + %d heads of 64 columns do not fit N=%d", e->q_heads, e->k_heads, N);
    FF_REQUIRE(e->q_w && e->k_w && e->rope_cos && e->rope_sin && e->tokens >= 1,
               "ff_gemm_fp4: the QKV epilogue needs q and k norm weights, rotation tables and tokens");
  }
  if (M == 0) return FF_OK;
  FF_REQUIRE(A.codes && A.scales && W.codes && W.scales && e->out, "ff_gemm_fp4: NULL pointer");
  FF_REQUIRE(fmt == FF_FP4_MX || (A.row_scale && W.row_scale), "ff_gemm_fp4: FF_FP4_NV needs row and column scales");
  FF_REQUIRE(epi != EPI_RESIDUAL || (e->residual && e->ldr >= N), "ff_gemm_fp4: the residual epilogue needs the residual and its row stride");
  FF_REQUIRE(aligned16(A.codes) && aligned16(A.scales) && aligned16(W.codes) && aligned16(W.scales),
             "ff_gemm_fp4: codes and scales must be 16-byte aligned");
  const bool f32 = e->out_dtype == FF_F32;
  FF_REQUIRE(f32 || (aligned16(e->out) && e->ldo % 8 == 0), "ff_gemm_fp4: 16-bit outputs need 16-byte aligned rows (ldo %% 8 == 0)");
  FF_REQUIRE(!f32 || reinterpret_cast<uintptr_t>(e->out) % 4 == 0, "ff_gemm_fp4: out is not aligned to its type");
  FF_REQUIRE(epi != EPI_RESIDUAL || (aligned16(e->residual) && e->ldr % 8 == 0), "ff_gemm_fp4: residual rows must be 16-byte aligned");

  const int64_t pair_tiles = static_cast<int64_t>((M + 255) / 256) * ((N + 255) / 256);
  const bool pair = tile == FF_TILE_PAIR256 || (tile == 0 && pair_tiles >= sm_count());
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
    const bool narrow = epi == EPI_SWIGLU && !pair;  // 32 output columns per warp
    // whole 16-byte granules only (none: a map that no store uses); the kernel writes the rest of a row itself
    rc = make_tmap_2d_pitched(&t.c, e->out, dt, 2, static_cast<uint64_t>(out_cols < 8 ? 8 : out_cols & ~7), static_cast<uint64_t>(M),
                              static_cast<uint64_t>(e->ldo) * 2, narrow ? 32 : 64, 32,
                              narrow ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != FF_OK) return rc;
  }
  if (epi == EPI_RESIDUAL) {
    rc = make_tmap_2d_pitched(&t.r, e->residual, dt, 2, static_cast<uint64_t>(N), static_cast<uint64_t>(M),
                              static_cast<uint64_t>(e->ldr) * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
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
  a.mx = mx;
  a.row_scale = mx ? nullptr : A.row_scale;
  a.col_scale = mx ? nullptr : W.row_scale;
  a.bias = e->bias;
  a.out = e->out;
  a.ldo = e->ldo;
  a.out_cols = out_cols;
  a.tma_cols = out_cols & ~7;
  a.norm = e->norm;
  a.q_heads = e->q_heads;
  a.k_heads = e->k_heads;
  a.qk_eps = e->qk_eps;
  a.q_w = e->q_w;
  a.q_b = e->q_b;
  a.k_w = e->k_w;
  a.k_b = e->k_b;
  a.rope_cos = e->rope_cos;
  a.rope_sin = e->rope_sin;
  a.tokens = e->tokens > 0 ? e->tokens : 1;
  a.w_const = w_const;
  a.err = device_error_word();
  FF_REQUIRE(a.err != nullptr, "ff_gemm_fp4: no device error word");
  return pair ? dispatch_fp4<true>(epi, e->out_dtype, t, a, stream) : dispatch_fp4<false>(epi, e->out_dtype, t, a, stream);
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
