// Attention of many queries per sequence to its keys and values on the 5th-generation tensor cores (tcgen05), heads of up to
// 64 columns.
//   out = softmax(scale q k^T) v, head by head, keys that do not take part left out
//
// Bound by the exponentials (one per query, key and head). With one softmax warp per scheduler and query tile their chains of
// dependent instructions left the unit 60% busy, so four streams share an SM, each with its scores S [128 queries x 64
// keys], weights P (over S) and output O in TMEM (64 + 64 columns) and four softmax warps: an item's two tiles of 128
// queries with every second step of 64 keys, or its only tile with every fourth. Streams of one tile keep a maximum, a sum
// and an output each, which are joined at the item's end.
//
// Persistent CTAs (one per SM, 640 threads, all 512 TMEM columns) walk items: up to 256 queries of one sequence and head
// against that sequence's keys; consecutive items overlap in the pipeline.
//   warp 0      loads, by TMA: an item's queries into one of two buffers, and 64 keys and their values in turn through one
//               ring of 8 steps. Their rows are rows of the whole matrix, whatever sequence they belong to.
//   warps 1, 2  MMAs, by an elected thread each: warp 1 for streams 0 and 1, warp 2 for 2 and 3. Per step of a stream: O += P V
//               (P read from TMEM), then S = Q K^T of the stream's next step, which finds P consumed, since MMAs of one
//               thread execute in order.
//   warps 4-19  softmax, four warps per stream, a query per thread: P = 2^(s - m + 7) (bf16: s - m - 28) in 16 bits, the sum of P in f32 before
//               that rounding. m is the maximum at some earlier time: the exponentials start at once, and the new maximum
//               is found beside them. Only where it has grown by more than 2^8 (P could pass 2^15, fp16's range) are m, O
//               and the sum rescaled and the step's exponentials repeated, out of line (372 us with that in the loop).
// Keys that take no part (past the sequence's end, or masked) get P = 0, and their rows of the value tile are overwritten
// with zeros in shared memory before the product, so that nothing they hold (NaN, infinities) counts. Streams of both
// tiles write the same zeros, each before it lets its own product start.
//
// Measured (at 1965 MHz): 2592 queries over 5184 keys of 4 images, 16 heads, fp16: 359 us, 614 TFLOP/s, exponentials 61% of the
// unit's rate (a quarter of them as polynomials on the other units 421 where this took 372: the issue slots are half taken
// already); 128 queries over 1025 keys of 64 images 93 us; 1845 queries over 16 keys of 6 sequences, 32 heads over 8: 43 us.
#include <algorithm>

#include "common.h"
#include "cross_tc.cuh"

namespace ff {

namespace {

constexpr int kStep = 64;                 // keys
constexpr int kRing = 8;                  // steps
constexpr int kSlot = kStep * 128;        // bytes of a K or V tile
constexpr int kThreads64 = 640;
constexpr int kOffRing = 4 * kAtom;       // two buffers of two query tiles
constexpr int kOffJoin = kOffRing + 2 * kRing * kSlot;          // [2][4 streams][128 rows] (ref, shift, sum, nothing)
constexpr int kOffTable = kOffJoin + 2 * 4 * 128 * 16;
constexpr int kOffBars = kOffTable + kTable * static_cast<int>(sizeof(Item));
constexpr int kSmem64 = 1024 + kOffBars + 512;
static_assert(kSmem64 <= 232448, "shared memory of a CTA");

__host__ __device__ constexpr uint32_t t_s64(int s) { return 64u * s; }
__host__ __device__ constexpr uint32_t t_o64(int s) { return 256u + 64u * s; }

// Which steps are whose: step t of an item belongs to its tiles' streams of phase t % ways. Two tiles: streams 0, 1 and 2, 3, two
// ways each; one tile: all four.
__device__ __forceinline__ int ways_of(const Item& i) { return i.nq > kBQ ? 2 : 4; }
__device__ __forceinline__ int phase_of(const Item& i, int stream) { return i.nq > kBQ ? stream & 1 : stream; }
__device__ __forceinline__ int steps_of(const Item& i) { return (i.nk + kStep - 1) / kStep; }

// The way of a step whose scores have grown, or seem to: out of line, it is rare. S in TMEM from `ts` becomes P. -> What all
// before has to be scaled by, the sum of the weights, the shift and whether there has been a key. Where the weights are
// relative to a ref, the shift is kSeemsGrown, and (ref, shift) are in the query's place of the join.
struct Grown {
  float corr, sum, shift;
  bool set;
};
template <class T>
__device__ __noinline__ Grown grown_step(uint32_t ts, uint32_t bits0, uint32_t bits1, float4* place, float shift, bool set, float scale_log2) {
  const bool far = shift == kSeemsGrown;
  Maximum m{far ? place->x : 0.f, far ? place->y : shift, set};
  float top = -INFINITY;
  uint32_t s[32];
  auto scores = [&](int c) {
    const uint32_t bits = c ? bits1 : bits0;
    tmem_ld32(ts + 32 * c, s);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (!(bits >> e & 1u)) s[e] = 0xff800000u;  // -inf
  };
  for (int c = 0; c < 2; ++c) {
    scores(c);
    top = fmaxf(top, largest(s));
  }
  Grown r{};
  r.corr = below<T>(m, top, scale_log2) ? raise<T>(m, top, scale_log2) : 1.f;
  for (int c = 0; c < 2; ++c) {
    scores(c);  // P is over the first half's
    uint32_t pk[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[i] = ex2_approx(fmaf(__uint_as_float(s[2 * e + i]) - m.ref, scale_log2, m.shift));
        r.sum += w[i];
      }
      pk[e] = Pair16<T>::pack(w[0], w[1]);
    }
    tmem_st16(ts + 16 * c, pk);
  }
  const bool nan = r.sum != r.sum, away = m.ref != 0.f && !nan;
  r.set = m.set || nan;
  r.shift = nan ? 0.f : away ? kSeemsGrown : m.shift;
  if (away) *place = make_float4(m.ref, m.shift, 0.f, 0.f);
  return r;
}

template <class T>
__global__ void __launch_bounds__(kThreads64, 1)
    cross_tc64_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ TcArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Item* const table = reinterpret_cast<Item*>(smem + kOffTable);
  auto join = reinterpret_cast<float4(*)[4][128]>(smem + kOffJoin);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint64_t* q_full = bar;               // [2]
  uint64_t* q_empty = q_full + 2;       // [2], by both MMA threads
  uint64_t* full = q_empty + 2;         // [2 kRing]: K, V of a step
  uint64_t* empty = full + 2 * kRing;   // [2 kRing], by both MMA threads
  uint64_t* s_full = empty + 2 * kRing;  // [4]
  uint64_t* p_full = s_full + 4;        // [4], by four warps
  uint64_t* o_full = p_full + 4;        // [4]: a stream's last product of an item
  uint64_t* joined = o_full + 4;        // maxima and sums of an item are there: 16 warps
  uint64_t* o_free = joined + 1;        // O of an item has been read: 16 warps
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
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 2);
    }
    for (int i = 0; i < 2 * kRing; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(joined, 16);
    mbar_init(o_free, 16);
    mbar_init(drain, 2);
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
  for (int n = a.by_cost ? kTable : threadIdx.x; n < kTable; n += kThreads64) {
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
      int q_phase[2] = {-1, -1}, phase[2 * kRing];
#pragma unroll
      for (int i = 0; i < 2 * kRing; ++i) phase[i] = -1;
      bool ok = true;
      uint32_t g = 0;  // step, over all items
      Item item;
      for (int m = 0; ok && items.next<true>(item); ++m) {
        const int qb = m & 1, tiles = item.nq > kBQ ? 2 : 1;
        if (m >= 2 && !mbar_wait<true>(&q_empty[qb], static_cast<uint32_t>((m >> 1) - 1) & 1u, abort_flag, err, kDevTimeoutAttn)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&q_full[qb], tiles * kAtom);
        for (int i = 0; i < tiles; ++i) tma_load_2d(smem + (2 * qb + i) * kAtom, &tm_q, &q_full[qb], items.head * dim, item.q + i * kBQ);
        q_phase[qb] = (m >> 1) & 1;
        const int x = items.head / group * dim, steps = steps_of(item);
        for (int t = 0; ok && t < steps; ++t, ++g)
          for (int v = 0; v < 2; ++v) {
            const uint32_t slot = 2 * (g % kRing) + v, round = g / kRing;
            if (!mbar_wait<true>(&empty[slot], (round & 1u) ^ 1u, abort_flag, err, kDevTimeoutAttn)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&full[slot], kSlot);
            tma_load_2d(smem + kOffRing + slot * kSlot, v ? &tm_v : &tm_k, &full[slot], x, item.k + t * kStep);
            phase[slot] = static_cast<int>(round & 1u);
          }
      }
      // Normally everything has been consumed. After an abort, let issued copies land (bounded) before the CTA can exit.
      if (!ok) {
        const unsigned long long t0 = globaltimer();
        for (int i = 0; i < 2; ++i)
          if (q_phase[i] >= 0)
            while (!mbar_try_wait(smem_u32(&q_full[i]), static_cast<uint32_t>(q_phase[i])) && globaltimer() - t0 < kWaitLimitNs) {
            }
        for (int i = 0; i < 2 * kRing; ++i)
          if (phase[i] >= 0)
            while (!mbar_try_wait(smem_u32(&full[i]), static_cast<uint32_t>(phase[i])) && globaltimer() - t0 < kWaitLimitNs) {
            }
      }
    }
  } else if (warp == 1 || warp == 2) {
    // ------------------------------------------------------------ MMAs
    if (elect_one()) {
      constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);  // both operands fp16 or bf16
      const uint32_t id_o = idesc_f16(128, dim) | fmt | (1u << 16);  // B = V is MN-major
      const int k_steps = dim / 16, base = 2 * (warp - 1);           // this thread's streams: base, base + 1
      const uint32_t ring = smem_u32(smem) + kOffRing;
      bool ok = true;
      auto wait = [&](uint64_t* b, uint32_t parity) {
        if (ok) ok = mbar_wait<true>(b, parity, abort_flag, err, kDevTimeoutAttn);
        return ok;
      };
      // Keys that a step's products cover: all, or the sequence's last ones rounded up to 16.
      auto width = [](const Item& i, int t) { return min(kStep, (i.nk - t * kStep + 15) & ~15); };
      uint32_t count[2] = {0, 0};  // steps of the streams
      auto keys_there = [&](uint32_t g) {
        const bool r = wait(&full[2 * (g % kRing)], (g / kRing) & 1u);
        tc_fence_after();
        return r;
      };
      // S of step t (g over all items) of item m for a stream, whose keys and queries are there.
      auto issue_s = [&](int i, const Item& item, int m, int t, uint32_t g) {
        const uint32_t slot = 2 * (g % kRing);
        const int stream = base + i, tile = item.nq > kBQ ? stream >> 1 : 0;
        const uint32_t id = idesc_f16(128, width(item, t)) | fmt;
        const uint64_t qd = sdesc_k_sw128(smem_u32(smem) + (2 * (m & 1) + tile) * kAtom), kd = sdesc_k_sw128(ring + slot * kSlot);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < k_steps) mma_f16(tmem + t_s64(stream), qd + 2 * k, kd + 2 * k, id, k > 0);
        tc_commit(&s_full[stream]);
        tc_commit(&empty[slot]);
      };
      Item cur{}, nxt{};
      int m = 0;
      uint32_t g0 = 0;  // first step of cur
      bool have = items.next<true>(cur);
      if (have && wait(&q_full[0], 0)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (ok && phase_of(cur, base + i) < steps_of(cur) && keys_there(phase_of(cur, base + i))) issue_s(i, cur, 0, phase_of(cur, base + i), phase_of(cur, base + i));
      }
      while (have && ok) {
        const bool more = items.next<true>(nxt);
        const int steps = steps_of(cur), ways = ways_of(cur);
        bool waiting = more;  // for the next item's queries
        bool first[2] = {false, false};  // its first S has been issued
        // Waits for what the stream's first S of the next item reads; whether there is one.
        auto first_there = [&](int i) {
          const int t = phase_of(nxt, base + i);
          if (!more || t >= steps_of(nxt)) return false;
          if (waiting && !wait(&q_full[(m + 1) & 1], static_cast<uint32_t>((m + 1) >> 1) & 1u)) return false;
          waiting = false;
          return keys_there(g0 + steps + t);
        };
        auto first_s = [&](int i) { issue_s(i, nxt, m + 1, phase_of(nxt, base + i), g0 + steps + phase_of(nxt, base + i)); };
        for (int t = 0; t < steps && ok; ++t) {
          const uint32_t g = g0 + t, slot = 2 * (g % kRing), round = (g / kRing) & 1u;
          bool mine = false;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (t % ways != phase_of(cur, base + i)) continue;
            mine = true;
            const int stream = base + i, keys = width(cur, t);
            const bool on = t + ways < steps;  // the stream goes on in this item
            const bool next = on ? keys_there(g + ways) : first_there(i);  // waited for before P, whose way through here counts
            if (!wait(&full[slot + 1], round) || !wait(&p_full[stream], count[i] & 1u)) break;
            ++count[i];
            tc_fence_after();
            const uint64_t vd = sdesc_v(ring + (slot + 1) * kSlot);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (16 * k < keys) mma_ts(tmem + t_o64(stream), tmem + t_s64(stream) + 8 * k, vd + static_cast<uint64_t>(k * 128), id_o, (t >= ways || k > 0) ? 1u : 0u);
            if (on) {  // before anything else: the softmax waits for it
              issue_s(i, cur, m, t + ways, g + ways);
            } else {
              tc_commit(&o_full[stream]);
              first[i] = true;
              if (next) first_s(i);
            }
            tc_commit(&empty[slot + 1]);
          }
          if (!mine && ok) {  // the other thread's, which needs this one's consent to load over it
            if (!wait(&full[slot], round) || !wait(&full[slot + 1], round)) break;
            mbar_arrive(&empty[slot]);
            mbar_arrive(&empty[slot + 1]);
          }
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (ok && !first[i] && first_there(i)) first_s(i);  // a stream without a step in this item
        tc_commit(&q_empty[m & 1]);
        g0 += steps;
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
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax and results
    const int stream = (warp - 4) >> 2, quarter = warp & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t ts = lanes + t_s64(stream), to = lanes + t_o64(stream);
    const int in_tile = quarter * 32 + lane;
    bool ok = true;
    uint32_t g0 = 0, count = 0, worked = 0, m = 0;  // first step of the item; steps, items with steps of this stream; items with keys
    Item item;
    while (ok && items.next<false>(item)) {
      const bool two = item.nq > kBQ;
      const int tile = two ? stream >> 1 : 0, ways = ways_of(item), phase = phase_of(item, stream), steps = steps_of(item);
      const int first_row = tile * kBQ + quarter * 32;
      const bool store = first_row + lane < item.nq, active = first_row < item.nq;
      T* const out = static_cast<T*>(p.out) + static_cast<int64_t>(item.q + first_row + lane) * p.ldo + static_cast<int64_t>(items.head) * dim;
      if (item.nk == 0) {
        if (store && (stream & (ways - 1)) == 0)
          for (int c = 0; c < dim; c += 8) *reinterpret_cast<uint4*>(out + c) = make_uint4(0, 0, 0, 0);
        continue;
      }
      const uint8_t* const mask = p.mask != nullptr ? p.mask + item.k : nullptr;
      uint32_t ahead[2] = {0, 0};  // mask bytes of the next step's keys lane and lane + 32
      auto fetch = [&](int t) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int key = t * kStep + 32 * c + lane;
          ahead[c] = key < item.nk ? __ldg(mask + key) : 0;
        }
      };
      if (mask != nullptr) fetch(phase);
      float shift = 0.f;  // once there is a maximum
      bool set = false;
      float4* const place = &join[m & 1][stream][in_tile];
      float2 sum = make_float2(0.f, 0.f);
      for (int t = phase; t < steps; t += ways, ++count) {
        const uint32_t g = g0 + t, v_slot = 2 * (g % kRing) + 1;
        const int left = item.nk - t * kStep;
        uint32_t bits[2];  // keys that take part
        if (mask != nullptr) {
          bits[0] = __ballot_sync(0xffffffffu, ahead[0] != 0);
          bits[1] = __ballot_sync(0xffffffffu, ahead[1] != 0);
          fetch(t + ways);
        } else {
          bits[0] = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
          bits[1] = left >= 64 ? 0xffffffffu : left <= 32 ? 0u : (1u << (left - 32)) - 1u;
        }
        const bool every = (bits[0] & bits[1]) == 0xffffffffu;
        if (!mbar_wait(&s_full[stream], count & 1u, abort_flag, err, kDevTimeoutAttn)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (!every) {  // zeros for the values of keys left out but within the product: warp i has keys [16 i, +16)
          const uint32_t mine = (quarter & 2 ? bits[1] : bits[0]) >> (16 * (quarter & 1));
          const uint32_t out_of = 16 * quarter < left ? ~mine & 0xffffu : 0u;
          if (out_of != 0) {
            if (!mbar_wait(&full[v_slot], (g / kRing) & 1u, abort_flag, err, kDevTimeoutAttn)) {
              ok = false;
              break;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = 4 * i + (lane >> 3);  // 8 lanes, 128 bytes: no two on a bank
              if (out_of >> key & 1u)
                *reinterpret_cast<uint4*>(smem + kOffRing + v_slot * kSlot + (quarter * 16 + key) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();
          }
        }
        if (active) {
          const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
          float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          float mx[2] = {-INFINITY, -INFINITY};
          uint32_t pk[2][16];
          bool slow = false;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t s[32];
            tmem_ld32(ts + 32 * c, s);
            tmem_ld_wait();
            if (bits[c] != 0xffffffffu) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(bits[c] >> e & 1u)) s[e] = 0xff800000u;  // -inf
            }
            if (c == 0 && t < ways) {  // a first maximum, from these 32
              const float top = largest(s), at = top * p.scale_log2;
              set = fabsf(at) < kFarScore;  // else with its second half
              if (set) shift = kUp<T> - floorf(at);
            }
            const float2 sh2 = make_float2(shift, shift);
            float2 x[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              x[e] = fma2(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), sc2, sh2);
              mx[e & 1] = max3(mx[e & 1], x[e].x, x[e].y);
            }
            if (c == 1) {
              const bool grown = fmaxf(mx[0], mx[1]) > kUp<T> + kGrowth || (!set && (bits[0] | bits[1]) != 0);
              if (__any_sync(0xffffffffu, grown)) {
                slow = true;
                break;
              }
              tmem_st16(ts, pk[0]);  // all of S is in registers
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 w = make_float2(ex2_approx(x[e].x), ex2_approx(x[e].y));
              part[e & 1] = add2(part[e & 1], w);
              pk[c][e] = Pair16<T>::pack(w.x, w.y);
            }
          }
          if (!slow) {
            tmem_st16(ts + 16, pk[1]);
          } else {
            const Grown r = grown_step<T>(ts, bits[0], bits[1], place, shift, set, p.scale_log2);
            if (t >= ways) rescale(to, dim, r.corr);
            sum.x *= r.corr;
            sum.y *= r.corr;
            part[0] = make_float2(r.sum, 0.f);
            part[1] = make_float2(0.f, 0.f);
            shift = r.shift;
            set = r.set;
          }
          sum = add2(sum, add2(part[0], part[1]));
        }
        if (t < ways && m > 0) {  // before the first product into O: the last item's has been read by all
          if (!mbar_wait(o_free, (m - 1) & 1u, abort_flag, err, kDevTimeoutAttn)) {
            ok = false;
            break;
          }
        }
        __syncwarp();
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[stream]);
      }
      if (!ok) break;
      if (phase < steps) {
        if (!mbar_wait(&o_full[stream], worked & 1u, abort_flag, err, kDevTimeoutAttn)) break;
        ++worked;
      }
      // The tile's streams are joined: each takes every ways-th 16 columns.
      if (shift != kSeemsGrown) *place = make_float4(0.f, set ? shift : INFINITY, 0.f, 0.f);
      place->z = sum.x + sum.y;
      __syncwarp();
      if (lane == 0) mbar_arrive(joined);
      if (!mbar_wait(joined, m & 1u, abort_flag, err, kDevTimeoutAttn)) break;
      tc_fence_after();
      if (active) {
        const int base = stream & ~(ways - 1), with = min(ways, steps);  // streams of this tile, and those that had a step
        float weight[4], l = 0.f;
        Maximum most{0.f, INFINITY, false};  // the highest
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < with) {
            const float4 v = join[m & 1][base + i][in_tile];
            const Maximum other{v.x, v.y, v.y < INFINITY};
            if (other.set && (!most.set || above(other, most, p.scale_log2) > 0.f)) most = other;
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          weight[i] = 0.f;
          if (i < with) {
            const float4 v = join[m & 1][base + i][in_tile];
            weight[i] = v.y < INFINITY ? ex2_approx(above({v.x, v.y, true}, most, p.scale_log2)) : 1.f;  // without a key: zeros, or NaN, which counts
            l = fmaf(v.z, weight[i], l);
          }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;  // no key took part: zeros
        for (int c = 16 * (stream - base); c < dim; c += 16 * ways) {
          float o[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < with) {
              uint32_t w[16];
              tmem_ld16(lanes + t_o64(base + i) + c, w);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = fmaf(__uint_as_float(w[e]), weight[i], o[e]);
            }
          if (store) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = Pair16<T>::pack(o[2 * e] * inv, o[2 * e + 1] * inv);
            store_columns(out + c, w);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      g0 += steps;
      ++m;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

template <class T>
int launch_tc64(const TcArgs& a, int grid, cudaStream_t s) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(cross_tc64_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem64) != cudaSuccess)
      return check_launch("cross_tc64: cudaFuncSetAttribute");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  CUtensorMap maps[3];
  const int rc = cross_maps(a.p, std::is_same<T, __nv_bfloat16>::value, kStep, maps);
  if (rc != FF_OK) return rc;
  launch(cross_tc64_kernel<T>, dim3(grid), dim3(kThreads64), kSmem64, s, maps[0], maps[1], maps[2], a);
  return check_launch("cross_tc64_kernel");
}

}  // namespace

int cross_tc64(const TcArgs& a, bool bf16, int grid, cudaStream_t s) {
  return bf16 ? launch_tc64<__nv_bfloat16>(a, grid, s) : launch_tc64<__half>(a, grid, s);
}

}  // namespace ff
