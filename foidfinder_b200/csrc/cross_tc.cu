// Attention of many queries per sequence to its keys and values on the 5th-generation tensor cores (tcgen05), heads of 65 to
// 128 columns (cross_tc64.cu has the narrower ones).
//   out = softmax(scale q k^T) v, head by head, keys that do not take part left out
//
// Bound by the exponentials (one per query, key and head) and the hand-overs between tensor core and softmax. Persistent
// CTAs (one per SM, 320 threads, all 512 TMEM columns) walk items: up to 256 queries (two tiles of 128) of one sequence
// and head, against that sequence's keys in tiles of 128; consecutive items overlap in the pipeline. Two streams, each with
// scores S, weights P and output O in TMEM, take a query tile each, or, of an item with one tile, every second key tile
// each, and are joined at its end.
//   warp 0     loads, by TMA: an item's queries, and key and value tiles in turn through one ring. A tile's rows are rows of
//              the whole matrix, whatever sequence they belong to.
//   warp 1     MMAs, by one elected thread: S_i = Q K^T of stream i to TMEM columns [128 i, +128), and O_i += P_i V, P_i read
//              from where S_i was, to columns [256 + 128 i, +dim). Order per key tile j of a pair: PV_0(j), S_0(j + 1), PV_1(j),
//              S_1(j + 1); MMAs of one thread execute in order, so S_i(j + 1) finds P_i(j) consumed. (A thread for each
//              stream let both fall in step and then wait together: 619 us where this took 463.)
//   warps 2-5  softmax of stream 0, warps 6-9 of stream 1, a query per thread: 32 scores at a time, the next 32 on their
//              way meanwhile, P = 2^(s - m + 7) (bf16: s - m - 28) in 16 bits, the sum of P in f32 before that rounding. m is the
//              maximum at some earlier time: the exponentials start at once, and the new maximum is found beside them.
//              Only where it has grown by more than 2^8 (P could pass 2^15, fp16's range) do m, O, the sum and the P so
//              far get rescaled, by a whole power of two, and the 32 exponentials repeated.
// Keys that take no part (past the sequence's end, or masked) get P = 0, and their rows of the value tile are overwritten
// with zeros in shared memory before the product, so that nothing they hold (NaN, infinities) counts. Both groups of
// softmax warps write the same zeros, each before it lets its own product start.
//
// Measured (at 1965 MHz): 2592 queries over 5184 keys of 4 images, 16 heads, fp16: 468 us, 940 TFLOP/s (512 us at the 1725 MHz that
// the power limit leaves in the long run; tensor pipe and exponentials each busy half of the time; a quarter of the
// exponentials as polynomials no gain); 1845 queries of 6 sequences, 32 heads over 8: over 512 keys 127 us, over 16 keys
// 55, 3.3 TB/s; ragged captions over ragged images (24 sequences, masked) 99 us.
#include <algorithm>

#include "common.h"
#include "cross_tc.cuh"

namespace ff {

namespace {

constexpr int kBK = 128;
constexpr int kTcThreads = 320;
constexpr int kSlots = 5;          // of the ring
constexpr int kTile = 2 * kAtom;   // 128 rows of 128 columns
constexpr int kOffRing = 2 * kTile;
constexpr int kOffJoin = kOffRing + kSlots * kTile;  // [3][128 rows]: ref, shift and sum of stream 1
constexpr int kOffTable = kOffJoin + 3 * 128 * 4;
constexpr int kOffBars = kOffTable + kTable * static_cast<int>(sizeof(Item));
constexpr int kTcSmem = 1024 + kOffBars + 256;
static_assert(kTcSmem <= 232448, "shared memory of a CTA");

// Whether the streams divide the keys of an item's only query tile, or (neither) the first has all of a single key tile.
__device__ __forceinline__ bool pair_of(const Item& i) { return i.nq > kBQ; }
__device__ __forceinline__ bool split_of(const Item& i) { return i.nq <= kBQ && i.nk > kBK; }
__device__ __forceinline__ int tiles_of(const Item& i) { return (i.nk + kBK - 1) / kBK; }

// TMEM columns of stream i.
__host__ __device__ constexpr uint32_t t_s(int i) { return 128u * i; }
__host__ __device__ constexpr uint32_t t_o(int i) { return 256u + 128u * i; }

// The first `chunks` times 32 weights of P scaled by corr.
template <class T>
__device__ __noinline__ void rescale_p(uint32_t ts, int chunks, float corr) {
  for (int c = 0; c < chunks; ++c) {
    uint32_t w[16];
    tmem_ld16(ts + 16 * c, w);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float2 v = Pair16<T>::unpack(w[e]);
      w[e] = Pair16<T>::pack(v.x * corr, v.y * corr);
    }
    tmem_st16(ts + 16 * c, w);
  }
}

// Zeros for the values of those of 32 keys that `out_of` says; out of line, it is rare.
__device__ __noinline__ void zero_values(uint8_t* v, uint32_t out_of, int lane) {
  for (int i = 0; i < 8; ++i) {
    const int key = 4 * i + (lane >> 3);  // 8 lanes, 128 bytes: no two on a bank
    if (out_of >> key & 1u) {
      uint8_t* const at = v + key * 128 + (lane & 7) * 16;
      *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(at + kAtom) = make_uint4(0, 0, 0, 0);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kTcThreads, 1)
    cross_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ TcArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Item* const table = reinterpret_cast<Item*>(smem + kOffTable);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint64_t* q_full = bar;
  uint64_t* q_empty = q_full + 1;
  uint64_t* full = q_empty + 1;       // [kSlots]
  uint64_t* empty = full + kSlots;    // [kSlots]
  uint64_t* s_full = empty + kSlots;  // [2], per query tile
  uint64_t* p_full = s_full + 2;      // [2]
  uint64_t* o_full = p_full + 2;      // [2]: a stream's last product of an item
  uint64_t* joined = o_full + 2;     // stream 1's maxima and sums are there: its 4 warps
  uint64_t* o_free = joined + 1;      // and its O has been read: stream 0's
  uint64_t* drain = o_free + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const CrossArgs& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int dim = p.dim, group = p.heads / p.kv_heads;
  int* const err = a.err;
  if (a.items == gridDim.x) {  // one item per CTA, perhaps none
    pdl_wait();
    const Item only = a.by_cost ? item_by_cost(a, reinterpret_cast<int2*>(smem + kOffRing), table) : item_at(a, blockIdx.x);
    if (only.nq == 0) return;
  }
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(joined, 4);
    mbar_init(o_free, 4);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tm_q);
    tma_prefetch_map(&tm_k);
    tma_prefetch_map(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  for (int n = a.by_cost ? kTable : threadIdx.x; n < kTable; n += kTcThreads) {
    const int64_t it = blockIdx.x + static_cast<int64_t>(n) * gridDim.x;
    table[n] = it < a.items ? item_at(a, it) : Item{0, 0, 0, 0};
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  Items items{a, table};

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (elect_one()) {
      int q_phase = -1, phase[kSlots];
#pragma unroll
      for (int i = 0; i < kSlots; ++i) phase[i] = -1;
      bool ok = true;
      int slot = 0;
      uint32_t round = 0;  // of the ring
      Item item;
      for (int m = 0; ok && items.next<true>(item); ++m) {
        const int tiles = item.nq > kBQ ? 2 : 1;
        if (m > 0 && !mbar_wait<true>(q_empty, static_cast<uint32_t>(m - 1) & 1u, abort_flag, err, kDevTimeoutAttn)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(q_full, tiles * kTile);
        for (int i = 0; i < tiles; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) tma_load_2d(smem + i * kTile + c * kAtom, &tm_q, q_full, items.head * dim + 64 * c, item.q + i * kBQ);
        q_phase = m & 1;
        const int x = items.head / group * dim, nkv = (item.nk + kBK - 1) / kBK;
        for (int j = 0; j < 2 * nkv; ++j) {  // K_0, V_0, K_1, V_1, ..
          if (!mbar_wait<true>(&empty[slot], (round & 1u) ^ 1u, abort_flag, err, kDevTimeoutAttn)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[slot], kTile);
#pragma unroll
          for (int c = 0; c < 2; ++c)
            tma_load_2d(smem + kOffRing + slot * kTile + c * kAtom, j & 1 ? &tm_v : &tm_k, &full[slot], x + 64 * c, item.k + (j >> 1) * kBK);
          phase[slot] = static_cast<int>(round & 1u);
          if (++slot == kSlots) {
            slot = 0;
            ++round;
          }
        }
      }
      // Normally everything has been consumed. After an abort, let issued copies land (bounded) before the CTA can exit.
      if (!ok) {
        const unsigned long long t0 = globaltimer();
        if (q_phase >= 0)
          while (!mbar_try_wait(smem_u32(q_full), static_cast<uint32_t>(q_phase)) && globaltimer() - t0 < kWaitLimitNs) {
          }
        for (int i = 0; i < kSlots; ++i)
          if (phase[i] >= 0)
            while (!mbar_try_wait(smem_u32(&full[i]), static_cast<uint32_t>(phase[i])) && globaltimer() - t0 < kWaitLimitNs) {
            }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs
    if (elect_one()) {
      constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);  // both operands fp16 or bf16
      const uint32_t id_o = idesc_f16(128, dim) | fmt | (1u << 16);  // B = V is MN-major
      const int steps = dim / 16;
      const uint32_t ring = smem_u32(smem) + kOffRing;
      // Keys of a tile that its products cover: all, or the sequence's last ones rounded up to 16.
      auto width = [](int nk, int j) { return min(kBK, (nk - j * kBK + 15) & ~15); };
      auto issue_s = [&](int i, int tile, int slot, int keys) {
        const uint32_t id = idesc_f16(128, keys) | fmt;
        const uint64_t qd = sdesc_k_sw128(smem_u32(smem) + tile * kTile);
        const uint64_t kd = sdesc_k_sw128(ring + slot * kTile);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < steps) {
            const uint64_t o = (k >> 2) * (kAtom >> 4) + (k & 3) * 2;
            mma_f16(tmem + t_s(i), qd + o, kd + o, id, k > 0);
          }
        tc_commit(&s_full[i]);
      };
      auto issue_pv = [&](int i, int slot, int keys, bool first) {
        const uint64_t vd = sdesc_v(ring + slot * kTile);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (16 * k < keys) mma_ts(tmem + t_o(i), tmem + t_s(i) + 8 * k, vd + static_cast<uint64_t>(k * 128), id_o, (first && k == 0) ? 0u : 1u);
      };
      bool ok = true;
      auto wait = [&](uint64_t* b, uint32_t parity) {
        if (ok) ok = mbar_wait<true>(b, parity, abort_flag, err, kDevTimeoutAttn);
        return ok;
      };
      // Ring positions: key tile t over all items has K at 2 t, V at 2 t + 1.
      auto arrived = [&](uint32_t at) {
        const bool r = wait(&full[at % kSlots], at / kSlots & 1u);
        tc_fence_after();
        return r;
      };
      int m = 0, s_left = 0;  // item; its S that are to be issued, after which its queries may go
      uint32_t g0 = 0, count[2] = {0, 0};
      // S of stream i for key tile t of an item; its keys and queries are there. keys_done: no other stream needs them.
      auto scores = [&](int i, int tile, int slot, int keys, bool keys_done) {
        issue_s(i, tile, slot, keys);
        if (keys_done) tc_commit(&empty[slot]);
        if (--s_left == 0) tc_commit(q_empty);
      };
      Item cur{}, nxt{};
      int first_done = 0;  // bits: streams whose first S of the next item has been issued
      // The same for its first key tile, of item `k`, if it has one.
      auto first_scores = [&](int i, const Item& item, int k, uint32_t g) {
        if (i == 1 && !pair_of(item) && !split_of(item)) return;
        if (first_done == 0) {
          if (!wait(q_full, static_cast<uint32_t>(k) & 1u)) return;
          s_left = tiles_of(item) * (pair_of(item) ? 2 : 1);
        }
        const int t = split_of(item) ? i : 0;
        if (!arrived(2 * (g + t))) return;
        scores(i, pair_of(item) ? i : 0, 2 * (g + t) % kSlots, width(item.nk, t), !pair_of(item) || first_done != 0);
        first_done |= 1 << i;
      };
      bool have = items.next<true>(cur);
      if (have) {
        first_scores(0, cur, 0, 0);
        if (ok) first_scores(1, cur, 0, 0);
      }
      while (have && ok) {
        const bool more = items.next<true>(nxt), two = pair_of(cur), split = split_of(cur);
        const int nkv = tiles_of(cur), stride = split ? 2 : 1;
        first_done = 0;
        for (int t = 0; t < nkv && ok; ++t) {
          // All that the issuing after a wait for P needs, worked out before it.
          const int keys = width(cur.nk, t), next_keys = width(cur.nk, t + stride);
          const bool on = t + stride < nkv;
          const uint32_t v = 2 * (g0 + t) + 1;
          const int v_slot = v % kSlots, k_slot = (v_slot + 2 * stride - 1) % kSlots;
          auto turn = [&](int i) {
            if ((!two || i == 0) && ((on && !arrived(2 * (g0 + t + stride))) || !arrived(v))) return;  // of a pair, stream 0 has waited
            if (!wait(&p_full[i], count[i] & 1u)) return;
            tc_fence_after();
            issue_pv(i, v_slot, keys, t < stride);
            ++count[i];
            if (on)  // before anything else: the softmax waits for it
              scores(i, two ? i : 0, k_slot, next_keys, !two || i == 1);
            else
              tc_commit(&o_full[i]);
            if (!two || i == 1) tc_commit(&empty[v_slot]);
            if (!on && more) first_scores(i, nxt, m + 1, g0 + nkv);
          };
          if (!split || (t & 1) == 0) turn(0);
          if (ok && (two || (split && (t & 1)))) turn(1);
        }
        if (ok && more && !two && !split) first_scores(1, nxt, m + 1, g0 + nkv);  // stream 1 had nothing here
        g0 += nkv;
        cur = nxt;
        have = more;
        ++m;
      }
      tc_commit(drain);
      const unsigned long long t0 = globaltimer();
      while (!mbar_try_wait(smem_u32(drain), 0)) {
        if (globaltimer() - t0 > kWaitLimitNs) {
          atomicCAS(err, 0, kDevTimeoutDrain);
          break;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax and results
    const int g = (warp - 2) >> 2, quarter = warp & 3;
    const uint32_t ts = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + t_s(g);
    const uint32_t to = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + t_o(g);
    float* const join = reinterpret_cast<float*>(smem + kOffJoin) + quarter * 32 + lane;
    bool ok = true;
    uint32_t g0 = 0, tiles = 0, worked = 0, splits = 0, freed = 0;  // key tiles of the items before; of this stream, and its items; split ones, and waited for
    Item item;
    while (ok && items.next<false>(item)) {
      const bool two = pair_of(item), split = split_of(item);
      const int first_row = (two ? g * kBQ : 0) + quarter * 32;  // of this warp, in the item
      const int64_t row = item.q + first_row + lane;
      const bool store = first_row + lane < item.nq, active = first_row < item.nq;
      T* const out = static_cast<T*>(p.out) + row * p.ldo + static_cast<int64_t>(items.head) * dim;
      if (item.nk == 0) {
        if (store && (two || g == 0))
          for (int c = 0; c < dim; c += 8) *reinterpret_cast<uint4*>(out + c) = make_uint4(0, 0, 0, 0);
        continue;
      }
      const int nkv = tiles_of(item), stride = split ? 2 : 1, first = split ? g : 0;
      const uint32_t g1 = g0;
      g0 += nkv;
      if (g == 1 && !two && !split) continue;  // nothing for this stream
      const uint8_t* const mask = p.mask != nullptr ? p.mask + item.k : nullptr;
      uint32_t ahead[4];  // mask bytes of the next tile's keys 32 c + lane
      auto fetch = [&](int j) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = j * kBK + 32 * c + lane;
          ahead[c] = key < item.nk ? __ldg(mask + key) : 0;
        }
      };
      if (mask != nullptr) fetch(first);
      Maximum m{0.f, 0.f, false};
      float use = 0.f;  // m.shift, or such a one that all scores seem to have grown
      float2 sum = make_float2(0.f, 0.f);
      for (int j = first; j < nkv; j += stride, ++tiles) {
        const int left = item.nk - j * kBK;
        uint32_t bits[4];  // keys that take part
        bool every = left >= kBK;
        if (mask != nullptr) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            bits[c] = __ballot_sync(0xffffffffu, ahead[c] != 0);
            every = every && bits[c] == 0xffffffffu;
          }
          fetch(j + stride);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) bits[c] = left >= 32 * c + 32 ? 0xffffffffu : left <= 32 * c ? 0u : (1u << (left - 32 * c)) - 1u;
        }
        if (!mbar_wait(&s_full[g], tiles & 1u, abort_flag, err, kDevTimeoutAttn)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (!every) {  // zeros for the values of keys left out but within the product: warp i has keys [32 i, +32)
          const uint32_t mine = quarter == 0 ? bits[0] : quarter == 1 ? bits[1] : quarter == 2 ? bits[2] : bits[3];
          const int within = ((left + 15) & ~15) - 32 * quarter;
          const uint32_t out_of = within <= 0 ? 0u : ~mine & (within >= 32 ? 0xffffffffu : (1u << within) - 1u);
          if (out_of != 0) {
            const uint32_t at = 2 * (g1 + j) + 1, v_slot = at % kSlots;
            if (!mbar_wait(&full[v_slot], at / kSlots & 1u, abort_flag, err, kDevTimeoutAttn)) {
              ok = false;
              break;
            }
            zero_values(smem + kOffRing + v_slot * kTile + quarter * 32 * 128, out_of, lane);
            fence_async_smem();
          }
        }
        if (active) {
          const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
          uint32_t s[2][32];
          tmem_ld32(ts, s[0]);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c < 3) tmem_ld32(ts + 32 * (c + 1), s[(c + 1) & 1]);
            uint32_t(&sc)[32] = s[c & 1];
            if (bits[c] != 0xffffffffu) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(bits[c] >> e & 1u)) sc[e] = 0xff800000u;  // -inf
            }
            if (c == 0 && j == first) {  // a first maximum
              const float at = largest(sc) * p.scale_log2;
              m.set = fabsf(at) < kFarScore;  // else below
              if (m.set) use = m.shift = kUp<T> - floorf(at);
            }
            uint32_t pk[16];
            float2 part;
            auto exponentials = [&](float shift) -> float {  // -> the largest exponent
              const float2 sh2 = make_float2(shift, shift);
              float mx[2] = {-INFINITY, -INFINITY};
              float2 ps[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float2 x = fma2(make_float2(__uint_as_float(sc[2 * e]), __uint_as_float(sc[2 * e + 1])), sc2, sh2);
                mx[e & 1] = max3(mx[e & 1], x.x, x.y);
                const float2 w = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                ps[e & 1] = add2(ps[e & 1], w);
                pk[e] = Pair16<T>::pack(w.x, w.y);
              }
              part = add2(ps[0], ps[1]);
              return fmaxf(mx[0], mx[1]);
            };
            const float mx = exponentials(use);
            const bool grown = mx > kUp<T> + kGrowth || (!m.set && bits[c] != 0);
            if (__any_sync(0xffffffffu, grown)) {
              if (c < 3) tmem_ld_wait();  // nothing on its way into registers across the calls
              tmem_st_wait();  // what the calls read back (P of the chunks before, O after an earlier growth) has been written
              const float top = largest(sc);
              const float corr = below<T>(m, top, p.scale_log2) ? raise<T>(m, top, p.scale_log2) : 1.f;
              use = m.ref != 0.f ? kSeemsGrown : m.shift;
              if (__any_sync(0xffffffffu, m.ref != 0.f)) {
#pragma unroll
                for (int e = 0; e < 32; ++e) sc[e] = __float_as_uint(__uint_as_float(sc[e]) - m.ref);
              }
              if (j > first) rescale(to, dim, corr);
              if (c > 0) rescale_p<T>(ts, c, corr);
              sum.x *= corr;
              sum.y *= corr;
              exponentials(m.shift);
              if (part.x != part.x || part.y != part.y) {
                m = {0.f, 0.f, true};
                use = 0.f;
              }
            }
            sum = add2(sum, part);
            tmem_st16(ts + 16 * c, pk);
            if (c < 3) tmem_ld_wait();
          }
        }
        if (g == 1 && freed != splits) {  // before the first product into this O: stream 0 has read it
          if (!mbar_wait(o_free, (splits - 1) & 1u, abort_flag, err, kDevTimeoutAttn)) {
            ok = false;
            break;
          }
          freed = splits;
        }
        __syncwarp();
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
      }
      if (!ok) break;
      if (!mbar_wait(&o_full[g], worked++ & 1u, abort_flag, err, kDevTimeoutAttn)) break;
      tc_fence_after();
      float l = sum.x + sum.y, mine = 1.f, other = 0.f;  // what both streams' outputs count
      if (split) {  // a stream's O is 2^shift times what it stands for; stream 0 writes the result
        if (g == 1) {
          join[0] = m.ref;
          join[128] = m.set ? m.shift : INFINITY;
          join[256] = l;
          __syncwarp();
          if (lane == 0) mbar_arrive(joined);
          ++splits;
          continue;
        }
        if (!mbar_wait(joined, splits & 1u, abort_flag, err, kDevTimeoutAttn)) break;
        ++splits;
        tc_fence_after();
        const Maximum theirs{join[0], join[128], join[128] < INFINITY};
        if (m.set && theirs.set) {  // else one has zeros, or NaN, which counts as well
          const float up = above(theirs, m, p.scale_log2);
          mine = up > 0.f ? ex2_approx(-up) : 1.f;
          other = up > 0.f ? 1.f : ex2_approx(up);
        } else {
          other = 1.f;
        }
        l = l * mine + join[256] * other;
      }
      if (active) {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // no key took part: zeros
        mine *= inv;
        other *= inv;
        for (int c = 0; c < dim; c += 16) {
          uint32_t o[16];
          tmem_ld16(to + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * mine);
          if (split) {
            uint32_t o1[16];
            tmem_ld16(to + t_o(1) - t_o(0) + c, o1);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(fmaf(__uint_as_float(o1[e]), other, __uint_as_float(o[e])));
          }
          if (store) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = Pair16<T>::pack(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
            store_columns(out + c, w);
          }
        }
      }
      if (split) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_free);
      }
      // The next item's first product into O waits for this group's next P, which comes after these reads.
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

template <class T>
int launch_tc(const TcArgs& a, int grid, cudaStream_t s) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(cross_tc_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmem) != cudaSuccess)
      return check_launch("cross_tc: cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  CUtensorMap maps[3];
  const int rc = cross_maps(a.p, std::is_same<T, __nv_bfloat16>::value, kBK, maps);
  if (rc != FF_OK) return rc;
  launch(cross_tc_kernel<T>, dim3(grid), dim3(kTcThreads), kTcSmem, s, maps[0], maps[1], maps[2], a);
  return check_launch("cross_tc_kernel");
}

}  // namespace

int cross_maps(const CrossArgs& p, bool bf16, int key_rows, CUtensorMap (&maps)[3]) {
  const void* base[3] = {p.q, p.k, p.v};
  const int64_t ld[3] = {p.ldq, p.ldk, p.ldv};
  for (int i = 0; i < 3; ++i) {
    const uint64_t cols = static_cast<uint64_t>(i == 0 ? p.heads : p.kv_heads) * p.dim, rows = i == 0 ? p.q_rows : p.k_rows;
    const int rc = make_tmap_2d_pitched(&maps[i], base[i], bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, cols, rows,
                                        2 * (rows > 1 ? static_cast<uint64_t>(ld[i]) : cols), 64, i == 0 ? kBQ : key_rows, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != FF_OK) return rc;
  }
  return FF_OK;
}

int cross_tc(const CrossArgs& p, bool bf16, cudaStream_t s) {
  TcArgs a{};
  a.p = p;
  a.tiles_per_seq = p.q_start == nullptr ? (p.q_rows / p.sequences + 255) / 256 : 0;
  const int64_t slots = p.q_start == nullptr ? static_cast<int64_t>(p.sequences) * a.tiles_per_seq : static_cast<int64_t>(p.q_rows) / 256 + p.sequences;
  FF_REQUIRE(slots <= 0x3fffffff, "ff_cross_attention: %lld query tiles", static_cast<long long>(slots));
  a.items = slots * p.heads;
  a.err = device_error_word();
  FF_REQUIRE(a.err != nullptr, "ff_cross_attention: no device error word");
  // Sequences that may differ in length: a CTA per item, so that whoever is done takes the next, the longest first; but where
  // these are short and many, CTAs that walk them, since the start of a CTA (3.5 us) counts then and their sums even out.
  // Walking and a CTA each (heads of 64 and 128, lengths alike to differing by 100% either way): 400 sequences of 140 queries over
  // 64 keys 233 to 330 and 429 to 491 us, 64 of 256 over 384: 77 to 150 and 102 to 149, over 512: 90 to 191 and 114 to
  // 178, over 1300: 175 to 413 and 188 to 318. Where there are fewer items, 24 of 200 over 256: 37 to 48 and 31 to 42, over 64: 22 to
  // 28 and 23 to 32.
  const bool even = p.q_start == nullptr && p.k_start == nullptr && p.k_len == nullptr;
  const int64_t keys = (static_cast<int64_t>(p.k_rows) + p.sequences - 1) / p.sequences;
  const bool walk = even || keys <= 64 || (keys <= 384 && a.items > 5 * sm_count());
  const int grid = static_cast<int>(std::min<int64_t>(a.items, walk ? sm_count() : 0x7fffffff));
  a.by_cost = !walk && grid == a.items && p.sequences <= kTcThreads;
  if (p.dim <= 64) return cross_tc64(a, bf16, grid, s);
  return bf16 ? launch_tc<__nv_bfloat16>(a, grid, s) : launch_tc<__half>(a, grid, s);
}

}  // namespace ff
