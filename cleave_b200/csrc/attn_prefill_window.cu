// Causal prefill over a sliding window with sinks, ragged or paged, on the tcgen05 tensor cores.
//
// The query at position p of its request sees key j <= p when j > p - window or j < sinks. An item is two blocks of 128
// query rows with one list of key tiles (128 keys): the tiles of the sinks, then ceil((window + 127) / 128) tiles that
// start at the first key of the first row's window, wherever that is; where the two ranges come close they are one. The
// blocks are two heads of a group, which see the same keys, or two neighbouring query tiles where a group has an odd
// number of heads; a block that does not exist is not computed.
//
//   S_g = Q_g K^T, P_g = 2^(scale S_g - m_g), O_g += P_g V     for the blocks g = 0, 1, key tile after key tile
//
// Why two: one block is a chain - scores, softmax, value product - in which the tensor cores idle during the softmax and
// the softmax warps during the products. With two blocks in turn the one's softmax runs beside the other's products, and a
// CTA asks L2 for half as many keys per row. Measured for one prompt of 8191 tokens, window 1024, 32/8 heads of 128:
// 206 .. 208 us where the same tiles on the one-block kernel of the plain prefill take 232 (five chunks of 1 .. 130 rows, where most
// items are one short chain and half of the SMs have none, take 25 where one block an item took 22: one kernel serves both); a step of both blocks takes 4200
// cycles, of which the tensor cores work 2050 and the exponentials' unit as much. What remains is latency: a softmax warp
// has its scheduler nearly to itself while the other block's products run, and issues an exponential every 16
// cycles where two warps at work issue one every 9.
//
// Tensor memory (512 columns of 128 lanes): S_0 | S_1 | O_0 | O_1. P_g takes the place of S_g (16-bit pairs, the first 64
// columns), so S_g of the next tile is issued only when the value product that reads P_g has completed.
// Warps: 0 loads Q and K, 1 issues the MMAs, 2 loads V, 3 hands out items; 4..7 and 8..11 are the softmax of block 0 and
// 1, a thread per row (no exchange between threads), with the registers that the first four give up; 12..15, where the
// keys are gathered row by row, copy K and V.
// The softmax keeps a reference maximum per row and rescales O (in tensor memory) only when the maximum has grown by
// more than 2^8; the factor is applied to O and to the row sum alike. P is rounded to the storage type, as the operand of
// a 16-bit product must be, and in fp16 scaled by 2^7 before (weight_headroom); everything else is held in 32 bits.
// CTAs are persistent: one per SM, items from a counter in the workspace header that clears itself.
// Keys that no row of an item sees (behind the last row, between the sinks and the window) add nothing whatever their
// rows hold: their scores are masked, and their rows of V are zero.

#include "common.cuh"

#include <algorithm>
#include <climits>
#include <cstring>
#include <type_traits>

namespace cb200 {
namespace {

constexpr int kBM = 128, kBN = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.f;  // log2 units
constexpr uint32_t kColS = 0, kColO = 256;  // block g: + 128 g

template <bool PAGED>
struct Roles {
  static constexpr int kThreads = PAGED ? 512 : 384;
  // registers a thread: launched with, softmax warps (256 threads), the others
  static constexpr int kRegsLaunch = PAGED ? 128 : 168;
  static constexpr int kRegsSoftmax = PAGED ? 176 : 208;
  static constexpr int kRegsOther = PAGED ? 80 : 88;
  static_assert(256 * kRegsSoftmax + (kThreads - 256) * kRegsOther <= kThreads * kRegsLaunch, "setmaxnreg would wait for good");
};

template <int D>
struct Cfg {
  static constexpr int kChunks = D / 64;         // 64-column chunks (128 bytes)
  static constexpr int kChunkBytes = 128 * 128;  // 128 rows of 128 bytes
  static constexpr int kTileBytes = kChunks * kChunkBytes;
  static constexpr int kStages = D == 64 ? 3 : 2;  // per K ring and per V ring
  static constexpr int kSmemBytes = (2 + 2 * kStages) * kTileBytes + 1024 /*barriers, items*/ + 1024;
};

struct Params {
  int* status;
  const void* k;  // paged: the caches
  const void* v;
  void* out;
  float* lse;
  const int* qo_indptr;
  const int* kv_indptr;
  const int* kv_indices;
  float scale_log2;
  int hq, hkv, num_pages, n_idx, batch, total_q;
  int fill;  // bit 0 / 1: rows of out / lse that belong to no request become 0 / -inf
  int window, sinks;
};

// A bounded wait in few instructions: there are two dozen of them in the kernel, and its code has to stay in the
// instruction cache. A wait that fails suspends the thread for a while in hardware; after 2^22 of those, or once another
// wait of the launch has given up, it returns and the status word says so.
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, int* status, int fault) {
  uint32_t n = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++n & 1023) == 0 && (n >= (1u << 22) || *reinterpret_cast<volatile int*>(status) != 0)) {
      atomicCAS(status, 0, fault);
      return;
    }
  }
}

// What the warps have to know of an item; found by warp 3, handed to the others through a ring in shared memory.
struct Item {
  int nt;             // key tiles; 0: no row sees a key; -1: there are no more items
  int two;            // the second block exists
  int head, row0;     // head and first query row (inside the request) of block 0; of block 1: head_of, row_of
  int hk;             // kv head
  int q_base, kv_base, sq, skv, off;                 // the request
  int last_key, first_key, n_sink, win_key, window;  // which keys the tiles hold
};

// A thread's row is written in whole 32-byte sectors: neighbouring lanes write rows that are far apart.
__device__ __forceinline__ void store_32_bytes(bool aligned, void* dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f, uint32_t g, uint32_t h) {
  if (!aligned) {  // a result of the caller's that starts on a 16-byte boundary only
    static_cast<uint4*>(dst)[0] = make_uint4(a, b, c, d);
    static_cast<uint4*>(dst)[1] = make_uint4(e, f, g, h);
    return;
  }
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h) : "memory");
}
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* m, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}

__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_of_32(const uint32_t (&x)[32]) {
  float a = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])), b = fmaxf(__uint_as_float(x[2]), __uint_as_float(x[3]));
#pragma unroll
  for (int i = 4; i < 32; i += 4) {
    a = max3(a, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
    b = max3(b, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
  }
  return fmaxf(a, b);
}

template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(Roles<PAGED>::kThreads, 1)
window_prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using C = Cfg<D>;
  using R = Roles<PAGED>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;                         // [2 blocks]
  uint8_t* k_smem = q_smem + 2 * C::kTileBytes;   // [stages]
  uint8_t* v_smem = k_smem + kStages * C::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_smem + kStages * C::kTileBytes);
  uint64_t* k_full = bars;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* v_land = v_empty + kStages;  // the load of a V tile whose rows are cleared before it is handed on
  uint64_t* q_full = v_land + kStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;   // [2] S_g complete
  uint64_t* p_half = s_full + 2;    // [2] the first 64 keys of P_g stored (and O_g rescaled if needed)
  uint64_t* p_full = p_half + 2;    // [2] all of P_g stored
  uint64_t* pv_done = p_full + 2;   // [2] the value product that reads P_g has completed
  uint64_t* o_done = pv_done + 2;   // [2] O_g of the item complete
  uint64_t* o_free = o_done + 2;    // [2] O_g has been read
  uint64_t* t_full = o_free + 2;    // [2] an item number is in the ring
  uint64_t* t_empty = t_full + 2;   // [2] every warp has read it
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(t_empty + 2);
  Item* item_ring = reinterpret_cast<Item*>(tmem_holder + 4);  // [2]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kWarps = R::kThreads / 32;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], PAGED ? 128 : 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], PAGED ? 128 : 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&v_land[s], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_half[g], 4);
      mbar_init(&p_full[g], 4);
      mbar_init(&pv_done[g], 1);
      mbar_init(&o_done[g], 1);
      mbar_init(&o_free[g], 4);
      mbar_init(&t_full[g], 1);
      mbar_init(&t_empty[g], kWarps - 1);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tm_q);
    if (!PAGED) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_holder);
  pdl_wait();
  pdl_launch_dependents();

  // ---- the work list. Row offsets are caller data: clipped to the rows there are, so no row outside `out` is written.
  auto q_row = [&](int r) { return min(max(__ldg(p.qo_indptr + r), 0), p.total_q); };
  int pre_lo = 0, pre_hi = 0, pre_klo = 0, pre_khi = 0;  // the ranges of the first 32 requests (lane = request)
  const bool heads_pair = (p.hq / p.hkv) % 2 == 0;  // the blocks are two heads; otherwise two query tiles
  const int unit = heads_pair ? kBM : 2 * kBM;                 // query rows of a request that an item covers
  const int head_units = heads_pair ? p.hq / 2 : p.hq;
  int q_units;
  {
    if (lane < p.batch) {
      pre_lo = q_row(lane);
      pre_hi = q_row(lane + 1);
      pre_klo = __ldg(p.kv_indptr + lane);
      pre_khi = __ldg(p.kv_indptr + lane + 1);
    }
    int mine = pre_hi > pre_lo ? ceil_div(pre_hi - pre_lo, unit) : 0;
#pragma unroll 4
    for (int r = 32 + lane; r < p.batch; r += 32) {
      const int lo = q_row(r), hi = q_row(r + 1);
      mine += hi > lo ? ceil_div(hi - lo, unit) : 0;
    }
    q_units = __reduce_add_sync(0xffffffffu, mine);
    // rows in front of the first request and behind the last, shared out over the grid
    if (p.fill) {
      const int head = q_row(0), rest = max(q_row(p.batch), head);
      const long long none = head + (p.total_q - rest), step = static_cast<long long>(gridDim.x) * blockDim.x;
      const long long i0 = static_cast<long long>(blockIdx.x) * blockDim.x + tid;
      auto row_of = [&](long long r) { return static_cast<size_t>(r < head ? r : r - head + rest); };
      if (p.fill & 1) {
        const int chunks = p.hq * (D / 8);  // 16 bytes each
        uint4* o = reinterpret_cast<uint4*>(p.out);
        for (long long i = i0; i < none * chunks; i += step) o[row_of(i / chunks) * chunks + i % chunks] = make_uint4(0u, 0u, 0u, 0u);
      }
      if ((p.fill & 2) && p.lse)
        for (long long i = i0; i < none * p.hq; i += step) p.lse[row_of(i / p.hq) * p.hq + i % p.hq] = -INFINITY;
    }
  }

  const int n_items = head_units * q_units;
  auto row_of = [&](const Item& w, int g) { return w.row0 + (heads_pair ? 0 : g * kBM); };
  auto head_of = [&](const Item& w, int g) { return w.head + (heads_pair ? g : 0); };

  // Item number -> item
  auto find_item = [&](int item, Item& w) {
    const int hu = item % head_units;
    int t = q_units - 1 - item / head_units;  // late query tiles first
    bool found = false;
    for (int r0 = 0; r0 < p.batch && !found; r0 += 32) {  // 32 requests a step, lane = request
      const int rr = r0 + lane;
      int lo = pre_lo, hi = pre_hi, klo = pre_klo, khi = pre_khi;
      if (r0 > 0) {
        lo = rr < p.batch ? q_row(rr) : 0;
        hi = rr < p.batch ? q_row(rr + 1) : 0;
        klo = rr < p.batch ? __ldg(p.kv_indptr + rr) : 0;
        khi = rr < p.batch ? __ldg(p.kv_indptr + rr + 1) : 0;
      }
      const int tiles = hi > lo ? ceil_div(hi - lo, unit) : 0;
      int incl = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const int all = __shfl_sync(0xffffffffu, incl, 31);
      if (t < all) {
        const int first = __ffs(__ballot_sync(0xffffffffu, incl > t)) - 1;
        t -= __shfl_sync(0xffffffffu, incl - tiles, first);
        w.q_base = __shfl_sync(0xffffffffu, lo, first);
        w.sq = __shfl_sync(0xffffffffu, hi, first) - w.q_base;
        w.kv_base = __shfl_sync(0xffffffffu, klo, first);
        w.skv = max(__shfl_sync(0xffffffffu, khi, first) - w.kv_base, 0);
        found = true;
      } else {
        t -= all;
      }
    }
    if (!found) return;  // not for the exact counts above
    if (PAGED && p.n_idx > 0) {
      // the page table is caller data: a range that runs past its stated length is read as a shorter request
      w.kv_base = min(max(w.kv_base, 0), p.n_idx);
      w.skv = min(w.skv, p.n_idx - w.kv_base);
    }
    w.row0 = t * unit;
    w.head = heads_pair ? 2 * hu : hu;
    w.hk = w.head / (p.hq / p.hkv);
    w.two = row_of(w, 1) < w.sq;
    w.off = w.skv - w.sq;  // row r of the request sits at position r + off
    // KV tile j starts at key tile_key(j): the sinks' tiles, then those of the window, which starts at first_key; or
    // tiles from key 0 on, where that takes no more of them
    w.window = min(p.window, w.skv);
    w.last_key = min(w.sq, w.row0 + unit) - 1 + w.off;             // last key any row of the item sees
    w.first_key = max(w.row0 + w.off - w.window + 1, 0);           // first key of the first row's window
    w.nt = w.last_key < 0 || w.skv == 0 ? 0 : w.last_key / kBN + 1;
    w.n_sink = w.win_key = 0;
    const int sink_tiles = ceil_div(min(p.sinks, w.first_key), kBN), win_tiles = ceil_div(w.last_key + 1 - w.first_key, kBN);
    if (w.nt > 0 && (sink_tiles + win_tiles < w.nt || sink_tiles == 0)) {
      w.n_sink = sink_tiles;
      w.win_key = w.first_key;
      w.nt = sink_tiles + win_tiles;
    }
  };
  auto tile_key = [&](const Item& w, int j) { return j < w.n_sink ? j * kBN : w.win_key + (j - w.n_sink) * kBN; };
  // whether no row of the item sees key `key` of KV tile j, and whether a KV tile holds such a key
  auto dead_key = [&](const Item& w, int j, int key) { return key > w.last_key || (key >= p.sinks && (j < w.n_sink || key < w.first_key)); };
  auto has_dead = [&](const Item& w, int j) {
    const int k0 = tile_key(w, j), k1 = k0 + kBN - 1;
    return k1 > w.last_key || (j < w.n_sink ? k1 >= p.sinks : max(k0, p.sinks) <= min(k1, w.first_key - 1));
  };

  // ---- items: the first of a CTA is its block index, the others come from a counter, one ahead of their use
  int* ticket = p.status + 8;
  int* finished = p.status + 9;
  int n_taken = 0;
  auto next_item = [&](Item& w) -> bool {
    const int s = n_taken & 1;
    wait(&t_full[s], (n_taken >> 1) & 1, p.status, kFaultFullBarrier);
    w = item_ring[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(&t_empty[s]);
    ++n_taken;
    return w.nt >= 0;
  };

  if (warp < 4 || warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::kRegsOther));
    if (warp == 3) {
      // ================================================================ items
      for (int k = 0;; ++k) {
        // with no more items than CTAs every item is somebody's first: no counter, nothing to clear at the end
        int item = k == 0 ? static_cast<int>(blockIdx.x) : n_items;
        if (k > 0 && n_items > static_cast<int>(gridDim.x)) {
          if (lane == 0) item = static_cast<int>(gridDim.x) + atomicAdd(ticket, 1);
          item = __shfl_sync(0xffffffffu, item, 0);
        }
        Item w{};
        w.nt = -1;
        if (item < n_items) find_item(item, w);
        const int s = k & 1;
        wait(&t_empty[s], ((k >> 1) & 1) ^ 1, p.status, kFaultEmptyBarrier);
        if (lane == 0) {
          item_ring[s] = w;
          mbar_arrive(&t_full[s]);
        }
        __syncwarp();
        if (w.nt < 0) break;
        // Q of an item that is about one item away is asked into L2: nothing else can hide that load, which waits for
        // the item before to be done with its Q
        if (k > 0 && w.nt > 0 && lane == 0) {
          for (int g = 0; g <= w.two; ++g)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c) tma_prefetch_3d(&tm_q, c * 64, head_of(w, g), w.q_base + row_of(w, g));
        }
      }
    } else if (warp == 0) {
      // ================================================================ TMA producer: Q, then K tiles
      int st = 0, ph = 0, it = 0;
      Item w;
      while (next_item(w)) {
        if (w.nt == 0) continue;
        auto load_q = [&]() {
          wait(q_empty, (it & 1) ^ 1, p.status, kFaultEmptyBarrier);
          if (lane == 0) {
            mbar_arrive_expect_tx(q_full, (1 + w.two) * C::kTileBytes);
            for (int g = 0; g <= w.two; ++g) {
  #pragma unroll
              for (int c = 0; c < C::kChunks; ++c) {
                uint8_t* dst = q_smem + g * C::kTileBytes + c * C::kChunkBytes;
                tma_load_3d(dst, &tm_q, q_full, c * 64, head_of(w, g), w.q_base + row_of(w, g));
              }
            }
          }
          __syncwarp();
          ++it;
        };
        if constexpr (PAGED) load_q();
        if constexpr (!PAGED) {
          for (int j = 0; j < w.nt; ++j) {
            wait(&k_empty[st], ph ^ 1, p.status, kFaultEmptyBarrier);
            uint8_t* dst = k_smem + st * C::kTileBytes;
            const int k0 = tile_key(w, j);
            if (elect_one()) {
              mbar_arrive_expect_tx(&k_full[st], C::kTileBytes);
#pragma unroll
              for (int c = 0; c < C::kChunks; ++c) tma_load_3d(dst + c * C::kChunkBytes, &tm_k, &k_full[st], c * 64, w.hk, w.kv_base + k0);
            }
            __syncwarp();
            if (j == 0) load_q();  // the first K tile does not have to wait for Q's place
            if (++st == kStages) { st = 0; ph ^= 1; }
          }
        }
      }
    } else if (warp == 2) {
      // ================================================================ TMA producer: V tiles
      // Rows of V that no query of the item sees meet P = 0, and 0 * V is 0 only for finite V: they are cleared once
      // the tile has landed, after the load of the tile behind it has been asked for, and only then is the tile handed on.
      int st = 0, ph = 0, land_ph = 0;  // land_ph: one bit a stage
      Item w;
      while (next_item(w)) {
        if (w.nt == 0) continue;
        if constexpr (!PAGED) {
          int unclear = -1, unclear_st = 0;
          auto clear_rows = [&]() {
            if (unclear < 0) return;
            wait(&v_land[unclear_st], land_ph >> unclear_st & 1, p.status, kFaultFullBarrier);
            land_ph ^= 1 << unclear_st;
            const int k0 = tile_key(w, unclear);
            uint8_t* dst = v_smem + unclear_st * C::kTileBytes;
            for (int i = lane; i < kBN * 8; i += 32) {
              if (!dead_key(w, unclear, k0 + (i >> 3))) continue;
#pragma unroll
              for (int c = 0; c < C::kChunks; ++c) *reinterpret_cast<uint4*>(dst + c * C::kChunkBytes + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[unclear_st]);
            unclear = -1;
          };
          for (int j = 0; j < w.nt; ++j) {
            wait(&v_empty[st], ph ^ 1, p.status, kFaultEmptyBarrier);
            uint8_t* dst = v_smem + st * C::kTileBytes;
            const int k0 = tile_key(w, j);
            const bool clear = has_dead(w, j);
            uint64_t* bar = clear ? &v_land[st] : &v_full[st];
            if (elect_one()) {
              mbar_arrive_expect_tx(bar, C::kTileBytes);
#pragma unroll
              for (int c = 0; c < C::kChunks; ++c) tma_load_3d(dst + c * C::kChunkBytes, &tm_v, bar, c * 64, w.hk, w.kv_base + k0);
            }
            __syncwarp();
            clear_rows();
            if (clear) {
              unclear = j;
              unclear_st = st;
            }
            if (++st == kStages) { st = 0; ph ^= 1; }
          }
          clear_rows();
        }
      }
    } else if (warp == 1) {
      // ================================================================ MMA issuer
      constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
      constexpr uint32_t idesc_s = umma_idesc(kBf16, /*b_mn_major=*/false, kBM, kBN);
      constexpr uint32_t idesc_pv = umma_idesc(kBf16, /*b_mn_major=*/true, kBM, D);
      // descriptors of the first stage; the others are a sum away (addresses count 16 bytes). Built anew for every MMA they
      // cost the issuing thread as long as the MMA takes.
      const uint64_t q_desc = umma_smem_desc(smem_u32(q_smem), 16, 8 * 128);
      const uint64_t k_desc = umma_smem_desc(smem_u32(k_smem), 16, 8 * 128);
      const uint64_t v_desc = umma_smem_desc(smem_u32(v_smem), C::kChunkBytes, 8 * 128);
      int kst = 0, kph = 0, vst = 0, vph = 0, it = 0;
      int n_s0 = 0, n_s1 = 0, n_it0 = 0, n_it1 = 0;  // tiles and items of each block so far
      Item w;
      while (next_item(w)) {
        if (w.nt == 0) continue;
        wait(q_full, it & 1, p.status, kFaultFullBarrier);
        // the blocks take turns: value product of tile j, scores of tile j + 1. One copy of the code for both.
#pragma unroll 1
        for (int j = -1; j < w.nt; ++j) {
#pragma unroll 1
          for (int g = 0; g <= w.two; ++g) {
            const uint32_t s_tmem = tmem_base + kColS + g * 128, o_tmem = tmem_base + kColO + g * 128;
            const int n = g ? n_s1 : n_s0;  // scores issued so far; those of tile j were the latest, and their P has the same number
            if (j >= 0) {
              wait(&v_full[vst], vph, p.status, kFaultFullBarrier);
              if constexpr (PAGED) fence_proxy_async_smem();
              // the first value product of an item overwrites O: the epilogue of the item before must have read it
              if (j == 0) wait(&o_free[g], ((g ? n_it1 : n_it0) & 1) ^ 1, p.status, kFaultTmemBarrier);
              const uint64_t vd = v_desc + vst * (C::kTileBytes >> 4);
              // the product over the first 64 keys starts while the softmax warps are on the others
#pragma unroll
              for (int part = 0; part < 2; ++part) {
                wait(part ? &p_full[g] : &p_half[g], (n - 1) & 1, p.status, kFaultTmemBarrier);
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                  for (int ks = part * 4; ks < part * 4 + 4; ++ks)  // B: MN-major, 16 token rows of 128 bytes per step
                    umma_f16_ts(o_tmem, s_tmem + ks * 8, vd + ((ks * 16 * 128) >> 4), idesc_pv, (j > 0 || ks > 0) ? 1u : 0u);
                  if (part == 1) {
                    umma_commit(&pv_done[g]);
                    if (g == w.two) umma_commit(&v_empty[vst]);
                    if (j == w.nt - 1) umma_commit(&o_done[g]);
                  }
                }
                __syncwarp();
              }
              if (g == w.two && ++vst == kStages) { vst = 0; vph ^= 1; }
            }
            if (j + 1 < w.nt) {
              wait(&k_full[kst], kph, p.status, kFaultFullBarrier);
              if constexpr (PAGED) fence_proxy_async_smem();
              // P of the tile before lies where S goes: the value product that reads it must have completed
              if (n > 0) wait(&pv_done[g], (n - 1) & 1, p.status, kFaultMmaBarrier);
              tc_fence_after();
              if (elect_one()) {
                const uint64_t qd = q_desc + g * (C::kTileBytes >> 4), kd = k_desc + kst * (C::kTileBytes >> 4);
#pragma unroll
                for (int c = 0; c < C::kChunks; ++c) {
#pragma unroll
                  for (int kk = 0; kk < 4; ++kk)
                    umma_f16(s_tmem, qd + ((c * C::kChunkBytes + kk * 32) >> 4), kd + ((c * C::kChunkBytes + kk * 32) >> 4), idesc_s, (c > 0 || kk > 0) ? 1u : 0u);
                }
                umma_commit(&s_full[g]);
                if (g == w.two) {
                  umma_commit(&k_empty[kst]);
                  if (j + 1 == w.nt - 1) umma_commit(q_empty);  // the item's last use of Q
                }
              }
              __syncwarp();
              if (g) ++n_s1; else ++n_s0;
              if (g == w.two && ++kst == kStages) { kst = 0; kph ^= 1; }
            }
          }
        }
        ++it;
        ++n_it0;
        n_it1 += w.two;
      }
    } else if constexpr (PAGED) {
      // ================================================================ row gather of K and V
      // Consecutive lanes copy consecutive 16-byte chunks of a row, so one warp instruction moves whole rows; rows that
      // no query sees are filled with zeros.
      const int gtid = tid - 12 * 32;  // 0..127
      constexpr int kChunksPerRow = D / 8;
      constexpr int kRowsPerRound = 128 / kChunksPerRow;
      constexpr int kRounds = kBN / kRowsPerRound;
      const int c = gtid % kChunksPerRow, r_in = gtid / kChunksPerRow;
      const uint32_t row_bytes = static_cast<uint32_t>(p.hkv) * D * 2;
      int st = 0, ph = 0;
      Item w;
      while (next_item(w)) {
        if (w.nt == 0) continue;
        const char* kc = static_cast<const char*>(p.k) + (w.hk * D + c * 8) * 2;
        const char* vc = static_cast<const char*>(p.v) + (w.hk * D + c * 8) * 2;
        const int* table = p.kv_indices + w.kv_base;
        const int last = w.skv - 1;
        auto load_pages = [&](int j, int (&pg)[kRounds]) {
          const int k0 = tile_key(w, j);
#pragma unroll
          for (int r = 0; r < kRounds; ++r) {
            const int tok = min(k0 + r * kRowsPerRound + r_in, last);
            pg[r] = __ldg(table + tok);
          }
        };
        int pg[kRounds];
        load_pages(0, pg);
        for (int j = 0; j < w.nt; ++j) {
          const int k0 = tile_key(w, j);
          uint32_t at[kRounds];  // the rows' places in the pool
          uint32_t alive = 0xffffffffu;
#pragma unroll
          for (int r = 0; r < kRounds; ++r) {
            at[r] = static_cast<uint32_t>(min(max(pg[r], 0), p.num_pages - 1));
          }
          if (has_dead(w, j)) {
#pragma unroll
            for (int r = 0; r < kRounds; ++r)
              if (dead_key(w, j, k0 + r * kRowsPerRound + r_in)) alive &= ~(1u << r);
          }
          if (j + 1 < w.nt) load_pages(j + 1, pg);  // one tile ahead: the index latency stays off the critical path
          auto copy = [&](const char* from, uint32_t to) {
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
              const int row = r * kRowsPerRound + r_in;
              const uint32_t o = (c >> 3) * C::kChunkBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4);
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + o), "l"(from + static_cast<uint64_t>(at[r]) * row_bytes),
                           "r"((alive >> r & 1u) * 16u)
                           : "memory");
            }
          };
          wait(&k_empty[st], ph ^ 1, p.status, kFaultEmptyBarrier);
          copy(kc, smem_u32(k_smem + st * C::kTileBytes));
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&k_full[st])) : "memory");
          wait(&v_empty[st], ph ^ 1, p.status, kFaultEmptyBarrier);
          copy(vc, smem_u32(v_smem + st * C::kTileBytes));
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&v_full[st])) : "memory");
          if (++st == kStages) { st = 0; ph ^= 1; }
        }
      }
    }
  } else {
    // ================================================================ softmax / epilogue: warps 4..7 block 0, 8..11 block 1
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R::kRegsSoftmax));
    const int g = warp >= 8 ? 1 : 0, quarter = warp & 3;
    const int row = quarter * 32 + lane;  // row of the block = tensor memory lane
    const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t s_col = lanes + kColS + g * 128, o_col = lanes + kColO + g * 128;
    const float scale = p.scale_log2;
    constexpr float kHeadroom = weight_headroom<T>(kRescaleThreshold);  // P is at most 2^8
    const bool negative = scale < 0.f;  // the largest score is then the smallest product
    int n = 0, it = 0;  // tiles and items of this block so far
    Item w;
    while (next_item(w)) {
      if (g == 1 && !w.two) continue;
      // ---- what the row sees: keys lo .. limit, and those in front of `sinks`; what all rows of the warp see
      const int qrow = row_of(w, g) + row, limit = qrow + w.off, lo = limit - w.window + 1;
      const bool live_row = qrow < w.sq;
      // rows behind the request's last are left out: they see whatever the others see
      const int warp_limit = __reduce_min_sync(0xffffffffu, live_row ? limit : INT_MAX);
      const int warp_lo = __reduce_max_sync(0xffffffffu, live_row ? lo : INT_MIN);
      float m_ref = -INFINITY;
      uint64_t l2 = pack_f32x2(0.f, 0.f);  // the row sum, in two halves
      for (int j = 0; j < w.nt; ++j, ++n) {
        const int k0 = tile_key(w, j);
        const bool sink_tile = j < w.n_sink;  // keys behind the sinks belong to the window's tiles
        wait(&s_full[g], n & 1, p.status, kFaultMmaBarrier);
        tc_fence_after();
        const bool edge = !(k0 + kBN - 1 <= warp_limit && ((k0 >= warp_lo && !sink_tile) || k0 + kBN - 1 < p.sinks));
        // P of 32 keys from their scores, into tensor memory
        auto put_p = [&](const uint32_t (&x)[32], int q, uint64_t scale2, uint64_t shift2) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x0, x1;
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale2, shift2), x0, x1);
            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
            l2 = add_f32x2(l2, pack_f32x2(p0, p1));
            pk[i] = pack2<T>(p0, p1);
          }
          tmem_st_32x16(s_col + q * 16, pk);
        };
        auto hand_on = [&](uint64_t* bar) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar);
        };
        // A tile at the edge of what the rows see, 32 keys at a time in a loop that is not unrolled, with the scores read
        // twice (pass 0: their maximum, pass 1: P): there are two or three such tiles an item, and unrolled four times
        // over, the code of this path did not stay in the instruction cache beside the other's (7000 cycles a tile).
        // P of 32 keys goes where scores already used were.
        auto edge_pass = [&](int pass, float m_use) -> float {
          float top = -INFINITY;
          const uint64_t one2 = pack_f32x2(1.f, 1.f), shift2 = pack_f32x2(-m_use, -m_use);
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            const int c0 = k0 + q * 32, above = limit - c0, below = sink_tile ? 64 : lo - c0, sink = p.sinks - c0;
            // bit i: the row sees key c0 + i; keys 0 .. above, from `below` on or in front of `sink`
            uint32_t see = below <= 0 ? 0xffffffffu : below > 31 ? 0u : 0xffffffffu << below;
            see |= sink > 31 ? 0xffffffffu : sink <= 0 ? 0u : (1u << sink) - 1;
            see &= above >= 31 ? 0xffffffffu : above < 0 ? 0u : (2u << above) - 1;
            uint32_t x[32];
            if (__any_sync(0xffffffffu, see != 0)) {
              tmem_ld_32x32(s_col + q * 32, x);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = see >> i & 1 ? __float_as_uint(__uint_as_float(x[i]) * scale) : 0xff800000u;
              if (pass == 0) top = fmaxf(top, max_of_32(x));
              else put_p(x, q, one2, shift2);
            } else if (pass == 1) {
              uint32_t none[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) none[i] = 0u;
              tmem_st_32x16(s_col + q * 16, none);
            }
            if (pass == 1 && q == 1) hand_on(&p_half[g]);
          }
          return top;
        };
        uint32_t r[4][32];
        float m_tile = -INFINITY;
        if (!edge) {
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld_32x32(s_col + q * 32, r[q]);
          tmem_ld_wait();
          if (!negative) {
            float mx[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) mx[q] = max_of_32(r[q]);
            m_tile = max3(mx[0], mx[1], fmaxf(mx[2], mx[3])) * scale;
          }
        }
        if (edge || negative) m_tile = edge_pass(0, 0.f);
        // the maximum of the row has grown: O and the sum follow. A row may see its first key in any tile; until then m_ref
        // is -inf, and O and the sum are worth nothing
        float alpha = 1.f;
        const bool grown = m_tile > m_ref + kRescaleThreshold;
        if (grown) {
          alpha = fast_exp2(m_ref - m_tile);
          m_ref = m_tile;
        }
        if (__any_sync(0xffffffffu, grown)) {
          l2 = mul_f32x2(l2, pack_f32x2(alpha, alpha));
          if (j > 0) {  // S of this tile was issued after the value product of the tile before had completed: O is at rest
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
              uint32_t o[32];
              tmem_ld_32x32(o_col + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = alpha == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x32(o_col + c0, o);
            }
          }
        }
        const float m_use = m_ref == -INFINITY ? 0.f : m_ref - kHeadroom;
        if (!edge) {
          const uint64_t scale2 = pack_f32x2(scale, scale), shift2 = pack_f32x2(-m_use, -m_use);
          put_p(r[0], 0, scale2, shift2);
          put_p(r[1], 1, scale2, shift2);
          hand_on(&p_half[g]);
          put_p(r[2], 2, scale2, shift2);
          put_p(r[3], 3, scale2, shift2);
        } else {
          edge_pass(1, m_use);
        }
        hand_on(&p_full[g]);
      }
      // ---- epilogue
      float l_a, l_b;
      unpack_f32x2(l2, l_a, l_b);
      const float l_run = l_a + l_b;
      // (an item without keys: its rows are 0 / -inf, and O is not looked at)
      if (w.nt > 0) {
        wait(&o_done[g], it & 1, p.status, kFaultMmaBarrier);
        tc_fence_after();
        ++it;
      }
      const float inv = l_run != 0.f ? 1.f / l_run : 0.f;  // the sum of a row with a NaN score is NaN, and so is the row
      const bool aligned = (reinterpret_cast<uintptr_t>(p.out) & 31) == 0;
      const size_t orow = static_cast<size_t>(w.q_base + row_of(w, g) + row) * p.hq + head_of(w, g);
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t o[32];
        if (w.nt > 0) {
          tmem_ld_32x32(o_col + c0, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (w.nt > 0 && c0 + 32 >= D) {  // O is out of tensor memory: the next item's value product may start
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_free[g]);
        }
        if (live_row) {
          T* dst = reinterpret_cast<T*>(p.out) + orow * D + c0;
          const float* v = reinterpret_cast<const float*>(o);
#pragma unroll
          for (int i = 0; i < 32; i += 16)
            store_32_bytes(aligned, dst + i, pack2<T>(v[i] * inv, v[i + 1] * inv), pack2<T>(v[i + 2] * inv, v[i + 3] * inv),
                           pack2<T>(v[i + 4] * inv, v[i + 5] * inv), pack2<T>(v[i + 6] * inv, v[i + 7] * inv),
                           pack2<T>(v[i + 8] * inv, v[i + 9] * inv), pack2<T>(v[i + 10] * inv, v[i + 11] * inv),
                           pack2<T>(v[i + 12] * inv, v[i + 13] * inv), pack2<T>(v[i + 14] * inv, v[i + 15] * inv));
        }
      }
      if (live_row && l_run == 0.f) {  // no key seen: what the tile's other rows see may hold Inf, and 0 * Inf is in O
#pragma unroll 1
        for (int i = 0; i < D / 8; ++i) reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + orow * D)[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      if (live_row && p.lse) p.lse[orow] = l_run != 0.f ? m_ref - kHeadroom + fast_log2(l_run) : -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (tid == 0 && n_items > static_cast<int>(gridDim.x) && atomicAdd(finished, 1) == static_cast<int>(gridDim.x) - 1) {
    // every CTA has fetched its last item number: the counters are clear for the next launch
    atomicExch(ticket, 0);
    atomicExch(finished, 0);
  }
}

// ------------------------------------------------------------------------------------- host side
template <typename T, int D, bool PAGED>
int launch_kernel(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const Params& p, long long items, cudaStream_t stream) {
  auto kern = window_prefill_kernel<T, D, PAGED>;
  static bool ready[16] = {false};  // per device
  int dev = 0;
  CB200_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 16 || !ready[dev]) {
    cudaFuncAttributes attr;
    CB200_CUDA_TRY(cudaFuncGetAttributes(&attr, kern));
    if (attr.numRegs < Roles<PAGED>::kRegsLaunch) return CB200_ERR_UNSUPPORTED;  // the softmax warps would wait for registers for good
    CB200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmemBytes));
    if (dev < 16) ready[dev] = true;
  }
  const int sms = sm_count();
  if (sms <= 0) return CB200_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>(items, sms)), 1, 1);
  cfg.blockDim = dim3(Roles<PAGED>::kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg<D>::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  // scheduled while the preceding kernel of the stream drains; the kernel waits before its first global access
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm_q, tm_k, tm_v, p));
  CB200_CUDA_TRY(cudaGetLastError());
  return CB200_OK;
}

int check_window(const cb200_attn_prefill_ragged_args* a) {
  if (!a) return CB200_ERR_BAD_ARG;
  if (a->num_qo_heads <= 0 || a->num_kv_heads <= 0 || a->batch <= 0 || a->total_q <= 0 || a->total_kv <= 0) return CB200_ERR_BAD_ARG;
  if (a->num_qo_heads % a->num_kv_heads) return CB200_ERR_BAD_ARG;
  if (a->head_dim != 64 && a->head_dim != 128) return CB200_ERR_UNSUPPORTED;
  if (a->dtype != CB200_F16 && a->dtype != CB200_BF16) return CB200_ERR_UNSUPPORTED;
  if (static_cast<long long>(a->num_qo_heads) * (ceil_div(a->total_q, kBM) + a->batch) >= (1LL << 31)) return CB200_ERR_UNSUPPORTED;
  if (a->total_q > (1 << 30) || (a->kv_indices ? a->num_kv_indices : a->total_kv) > (1 << 30)) return CB200_ERR_UNSUPPORTED;  // rows and keys, rounded up to tiles, in 32 bits
  if (!a->q || !a->k || !a->v || !a->out || !a->qo_indptr || !a->kv_indptr) return CB200_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
       reinterpret_cast<uintptr_t>(a->out)) & 15)
    return CB200_ERR_ALIGNMENT;
  if (!a->workspace || a->workspace_bytes < kWsHeaderBytes) return CB200_ERR_WORKSPACE;
  return CB200_OK;
}

template <typename T, int D>
int launch_window(const cb200_attn_prefill_ragged_args* a, int window, int sinks, int fill, cudaStream_t stream) {
  Params p{};
  p.status = reinterpret_cast<int*>(a->workspace);
  p.k = a->k;
  p.v = a->v;
  p.scale_log2 = a->sm_scale * kLog2e;
  p.hq = a->num_qo_heads;
  p.hkv = a->num_kv_heads;
  p.num_pages = a->total_kv;
  p.out = a->out;
  p.lse = a->lse;
  p.qo_indptr = a->qo_indptr;
  p.kv_indptr = a->kv_indptr;
  p.kv_indices = a->kv_indices;
  p.n_idx = a->kv_indices ? a->num_kv_indices : 0;
  p.batch = a->batch;
  p.total_q = a->total_q;
  p.fill = fill;
  p.window = window;
  p.sinks = sinks;
  const CUtensorMapDataType dt = a->dtype == CB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  CUtensorMap tm_q, tm_k, tm_v;
  memset(&tm_k, 0, sizeof(tm_k));
  memset(&tm_v, 0, sizeof(tm_v));
  // a box is 64 columns of one head for 128 consecutive tokens
  const uint32_t box[3] = {64u, 1u, 128u};
  const uint64_t row = static_cast<uint64_t>(D) * 2;
  const uint64_t dq[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a->num_qo_heads), static_cast<uint64_t>(a->total_q)};
  const uint64_t sq[2] = {row, row * a->num_qo_heads};
  if (!encode_tensor_map(&tm_q, dt, 3, const_cast<void*>(a->q), dq, sq, box, sw)) return CB200_ERR_CUDA;
  if (!a->kv_indices) {
    const uint64_t dk[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a->num_kv_heads), static_cast<uint64_t>(a->total_kv)};
    const uint64_t sk[2] = {row, row * a->num_kv_heads};
    if (!encode_tensor_map(&tm_k, dt, 3, const_cast<void*>(a->k), dk, sk, box, sw) ||
        !encode_tensor_map(&tm_v, dt, 3, const_cast<void*>(a->v), dk, sk, box, sw))
      return CB200_ERR_CUDA;
  }
  // an upper bound on the items: every request has at most ceil(its rows / unit) <= its rows / unit + 1 of them per head
  const bool heads_pair = (p.hq / p.hkv) % 2 == 0;
  const long long items = heads_pair ? static_cast<long long>(p.hq / 2) * (ceil_div(a->total_q, kBM) + a->batch)
                                     : static_cast<long long>(p.hq) * (ceil_div(a->total_q, 2 * kBM) + a->batch);
  return a->kv_indices ? launch_kernel<T, D, true>(tm_q, tm_k, tm_v, p, items, stream)
                       : launch_kernel<T, D, false>(tm_q, tm_k, tm_v, p, items, stream);
}

}  // namespace
}  // namespace cb200

extern "C" int cb200_attn_prefill_ragged_window(const cb200_attn_prefill_ragged_args* a, int window, int sinks, int fill, void* stream) {
  using namespace cb200;
  if (window <= 0 || sinks < 0 || fill < 0 || fill > 3) return CB200_ERR_BAD_ARG;
  const int rc = check_window(a);
  if (rc != CB200_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f16 = a->dtype == CB200_F16;
  if (a->head_dim == 64)
    return f16 ? launch_window<__half, 64>(a, window, sinks, fill, st) : launch_window<__nv_bfloat16, 64>(a, window, sinks, fill, st);
  return f16 ? launch_window<__half, 128>(a, window, sinks, fill, st) : launch_window<__nv_bfloat16, 128>(a, window, sinks, fill, st);
}

