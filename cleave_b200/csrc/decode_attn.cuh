// Decode attention (MHA / GQA / MQA; contiguous or paged KV) for sm_100a.
//
// One persistent launch, one CTA per SM. The KV cache is cut into tiles of 64 tokens; the tiles of
// all (request, kv head) items form one stream that is split evenly over the CTAs, so a CTA's
// share may start or end in the middle of an item. A producer warp streams its share of tiles
// into a ring of shared-memory stages (TMA tiled loads with the 128-byte swizzle when a tile maps
// to whole boxes of the cache; otherwise eight producer warps gather the token rows with 16-byte
// cp.async into the same swizzled layout) and the
// consumer warps run QK^T and PV on m16n8k16 tensor-core MMAs with a warp-shuffle online softmax
// in the exp2 domain. An item finished inside one CTA is written directly; an item cut across
// CTAs leaves fp32 partials (O, m, l) in the workspace and the last CTA to arrive does the
// log-sum-exp combine (no second launch, nobody waits).
//
// Semantics follow python/cleave/dynamic/reference.py:143-200 of the reference (paged) and
// demo/attention.py:5-8 (static); the valid-length clamp follows
// python/cleave/dynamic/paging/builders/slab.py:132-142.
//
// Three more operators on paged caches run on the same stream of tiles (template parameter MODE):
//   kWindow   token j of a request with n tokens takes part when j >= n - window or j < sinks. Only the tiles that
//             hold such a token are in the stream: the tiles of the sinks, then those of the window.
//   kWeights  the scores (log2 units, fp32) are also left in a scratch buffer, from which a second kernel forms
//             the attention weights once the row's log-sum-exp is known: 4 bytes a (query head, token) written and
//             read against 4 D bytes of K and V a (kv head, token), where a second pass over K would read 2 D.
//   kSuffix   every request continues a prefix whose attention another kernel has left as fp32 partials (O, m, l):
//             they are merged where the row's result is stored.
// In these modes a token that takes no part adds nothing whatever its cache row holds (the plain mode multiplies
// the rows behind a request's last token by zero), and P enters P V as the sum of two 16-bit numbers, scaled where that keeps
// them out of fp16's subnormal range: the warp MMAs have the room (the kernel is bound by the stream of K and V), and the
// error of the output is then the rounding of the output alone.

#pragma once

#include "common.cuh"
#include "stream_walk.cuh"

#include <cstring>
#include <type_traits>

namespace cb200 {

constexpr int kTile = 64;          // tokens per KV tile
constexpr int kRowsMax = 16;       // query rows one item carries (M of the MMA tile)
constexpr int kConsumerWarps = 4;  // each owns 16 tokens of every tile
constexpr int kPieceUnits = 5;     // what starting and finishing a piece costs, in tiles: the stream of a paged launch is cut by cost
constexpr int kPrefetchTiles = 16; // tiles a CTA asks into L2 while it waits for the preceding kernel (contiguous caches)
constexpr float kLog2e = 1.4426950408889634f;

enum DecodeMode { kPlain = 0, kWindow = 1, kWeights = 2, kSuffix = 3 };

// The modes find the next piece and load its Q while the one before is merged, so a piece costs them less. 64 requests with
// windows of 1004 tokens / 64 behind 8192 / 128 behind 32768: 53.7 / 45.7 / 192.0 us with 5, 52.9 / 45.2 / 190.6 with 3,
// 52.9 / 45.5 / 197.0 with 2, 53.8 / 51.0 / 200.3 with 1.
// Three shapes are what this constant rests on. Where the page table has no more tiles than there are CTAs, every tile is a
// CTA's whole share and nothing is left to balance: no units then, so that the working CTAs are the first ones, which find SMs
// beside the prefix's (4 requests behind 1000 tokens: 14.3 -> 11.3 us). The rule knows the table, not the stream: a short
// window over a long table keeps the units although its tiles are few.
constexpr int kPieceUnitsModes = 3;

struct DecodeParams {
  const void* q;
  const void* k;
  const void* v;
  const int* kv_indptr;
  const int* kv_indices;
  const int* kv_last;
  void* out;
  float* lse;
  int* status;     // workspace header
  int* counters;   // one arrival counter per item, zero between launches
  float* partials; // gridDim.x * 2 slots
  int batch, hkv, vblk, rows, page_size, num_pages, n_idx, kv_len, paged, box_tok;
  float scale_log2;
  int page_shift;  // log2 of page_size, or -1 where it is not a power of two
  int piece_units; // modes: what starting and finishing a piece costs, in tiles
  // kWindow
  int window, sinks;
  // kWeights: scores, one row of raw_pitch floats per (request, query head); tokens beyond raw_len are not kept
  float* raw;
  int raw_len;
  long long raw_pitch;
  // kSuffix: partials of the prefix, pre_splits of them per (kv head, block of 128 query rows), see prefix_attn.cu
  const float* pre_o;   // [kv head][row block][split][128][D], relative to the split's reference maximum
  const float* pre_ml;  // [kv head][row block][split][2][128]: reference maximum (log2 units; -inf: no score is finite), sum
  int pre_splits, pre_blocks, pre_batch;  // pre_batch: requests per row block
};

// Boxes of 16 tokens, for the tiles of which only some such groups are needed (TMA path of the modes on paged caches)
struct GroupMaps {
  CUtensorMap k, v;
};

template <int D, bool GATHER, int MODE>
struct SmemPlan {
  // Both paths use the same tile layout: per 64-column half, 64 rows of 128 bytes with the
  // 128-byte swizzle (what TMA writes; the gather path reproduces it with 16-byte cp.async).
  static constexpr int kMatBytes = kTile * D * 2;
  static constexpr int kStageBytes = 2 * kMatBytes;
  static constexpr int kStages = 5;
  // gather: eight copying warps - the bytes an SM keeps in flight are bounded per issuing warp (a gather-only kernel
  // over random 1 KB rows moved 4.0 TB/s with four warps per SM whatever their depth, 6.0 with eight)
  static constexpr int kProducerWarps = GATHER ? 8 : 1;
  static constexpr int kThreads = (kConsumerWarps + kProducerWarps) * 32;
  // A warp's state in the merge buffer. In the modes the rows are eight floats apart in the banks, so that the fragments'
  // rows meet no bank twice when they are written (the plain kernel's rows of D floats leave room for more requests).
  static constexpr int kMergePitch = MODE == kPlain ? D : D + 8;
  static constexpr int kMergeFloats = kRowsMax * kMergePitch + 2 * kRowsMax;
  static constexpr int kSlotFloats = kRowsMax * D + 2 * kRowsMax;  // a partial in the workspace
  static constexpr int kMergeBytes = kConsumerWarps * kMergeFloats * 4;
  static constexpr int kFixedBytes = kStages * kStageBytes + kMergeBytes + 256;  // + barriers/flags
};

// Pages of request b that the page table really holds: kv_indptr is caller data, so the range it names is
// clipped to [0, n_idx) and every later read of kv_indices stays inside the array whatever it says.
__device__ __forceinline__ int item_pages(const DecodeParams& p, int b) {
  const int base = p.kv_indptr[b];
  if (base < 0 || base >= p.n_idx) return 0;
  return max(min(p.kv_indptr[b + 1] - base, p.n_idx - base), 0);
}

__device__ __forceinline__ int item_valid_len(const DecodeParams& p, int b) {
  if (!p.paged) return p.kv_len;
  const int n_pages = item_pages(p, b);
  if (p.page_size == 1 || p.kv_last == nullptr) return n_pages * p.page_size;
  // the count is caller data: clipped before it is added, so that the sum stays in 32 bits (and loaded whatever n_pages is, so
  // that the load does not wait for the page table's)
  const int v = max(n_pages - 1, 0) * p.page_size + min(max(p.kv_last[b], 0), p.page_size);
  return min(v, n_pages * p.page_size);
}

// The tiles of a request with n tokens that are in the stream. Whole boxes of the cache (TMA): tile t of the item is tile t
// of the cache while t < n_sink, and tile t + skip behind that; tokens from `lo` on are inside the window, and the tiles
// at the edges hold others too. Gathered rows: the stream holds the tokens that take part and no others; its token v is
// the cache's v while v < head, and v + jump behind that.
struct ItemView {
  int valid;               // tokens up to which the stream's count runs
  int lo, n_sink, skip;    // whole boxes
  int head, jump;          // gathered rows
  __device__ __forceinline__ int tile(int t) const { return t < n_sink ? t : t + skip; }
  __device__ __forceinline__ int token(int v) const { return v < head ? v : v + jump; }
  __device__ __forceinline__ int n_tiles() const { return ceil_div(valid, kTile) - skip; }
};

template <int MODE, bool GATHER>
__device__ __forceinline__ ItemView item_view(const DecodeParams& p, int n) {
  ItemView v{n, 0, 0, 0, 0, 0};
  if constexpr (MODE == kWindow) {
    const int lo = max(n - p.window, 0), sinks = min(p.sinks, lo);
    if constexpr (GATHER) {
      v.head = sinks;
      v.jump = lo - sinks;
      v.valid = n - v.jump;
    } else {
      const int first = lo / kTile;
      v.lo = lo;
      v.n_sink = min(ceil_div(sinks, kTile), first);
      v.skip = first - v.n_sink;
    }
  }
  return v;
}

// The modes read a tile in groups of 16 tokens, a consumer warp's share: whether token `tok` takes part, whether any of the
// group from `tok` on does, and whether all 64 of the tile from `tok` on do
template <int MODE, bool GATHER>
__device__ __forceinline__ bool token_lives(const DecodeParams& p, const ItemView& v, int tok) {
  return tok < v.valid && (MODE != kWindow || GATHER || tok >= v.lo || tok < p.sinks);
}
template <int MODE, bool GATHER>
__device__ __forceinline__ bool group_lives(const DecodeParams& p, const ItemView& v, int tok) {
  return tok < v.valid && (MODE != kWindow || GATHER || tok + 15 >= v.lo || tok < p.sinks);
}
template <int MODE, bool GATHER>
__device__ __forceinline__ bool tile_whole(const DecodeParams& p, const ItemView& v, int tok) {
  return tok + kTile <= v.valid && (MODE != kWindow || GATHER || tok >= v.lo || tok + kTile <= p.sinks);
}

template <typename T, int D, bool GATHER, int MODE = kPlain>
__global__ void __launch_bounds__(SmemPlan<D, GATHER, MODE>::kThreads, 1)
decode_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ GroupMaps tm_group, const DecodeParams p) {
  using Plan = SmemPlan<D, GATHER, MODE>;
  constexpr int kStages = Plan::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stages = smem;
  float* merge = reinterpret_cast<float*>(smem + kStages * Plan::kStageBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kStages * Plan::kStageBytes + Plan::kMergeBytes);
  uint64_t* empty_bar = full_bar + kStages;
  int* flags = reinterpret_cast<int*>(empty_bar + kStages);  // [0] last-arriver flag, [1..] scan scratch
  int* P = reinterpret_cast<int*>(smem + Plan::kFixedBytes);
  int* V = P + p.batch + 1;  // modes: tokens per request, so that a piece is found without a trip to memory

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nthreads = blockDim.x;
  const int hkvv = p.hkv * p.vblk;
  const int w = MODE == kPlain ? kPieceUnits : p.piece_units;  // of a paged launch

  // The launch carries the programmatic-serialization attribute: this CTA may start while the kernel
  // before it in the stream is still draining. Nothing that kernel may have written (page tables, the
  // caches, Q, the workspace) is touched before pdl_wait(); what precedes it is shared-memory set-up.
  // ---- tile prefix over requests (every CTA computes the same table)
  int tiles_per_req = 0;
  if (p.paged) {
    // Behind a prefix the kernel before this one is the prefix's, which reads what this one reads, lets this one start
    // only once its own predecessor is done, and writes nothing but the partials: they are waited for where they
    // are merged, and CTAs that find an SM stream their requests' own tokens beside it.
    if (MODE != kSuffix || p.pre_splits == 0) pdl_wait();
    int* scratch = reinterpret_cast<int*>(merge);  // merge buffer is free at this point
    const int per = ceil_div(p.batch, nthreads);
    const int i0 = min(tid * per, p.batch), i1 = min(i0 + per, p.batch);
    int sum = 0;
    for (int i = i0; i < i1; ++i) {
      const int n = item_valid_len(p, i);
      if (MODE != kPlain) V[i] = n;
      sum += Walker::units(item_view<MODE, GATHER>(p, n).n_tiles(), w);
    }
    scratch[tid] = sum;
    __syncthreads();
    if (tid < 32) {
      const int all = warp_scan_in_place(scratch, nthreads, tid);
      if (tid == 0) P[p.batch] = all;
    }
    __syncthreads();
    int run = scratch[tid];
    for (int i = i0; i < i1; ++i) {
      P[i] = run;
      run += Walker::units(item_view<MODE, GATHER>(p, MODE != kPlain ? V[i] : item_valid_len(p, i)).n_tiles(), w);
    }
  } else {
    tiles_per_req = ceil_div(p.kv_len, kTile);
  }
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], GATHER ? Plan::kProducerWarps * 32 : 1);  // gather: one arrival per copying thread
      mbar_init(&empty_bar[s], kConsumerWarps);
    }
    mbar_fence_init();
    if (!GATHER) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
  }
  __syncthreads();

  const int total_per_head = p.paged ? P[p.batch] : p.batch * tiles_per_req;
  const int total = hkvv * total_per_head;
  const int G = gridDim.x;
  const int span = total > 0 ? ceil_div(total, G) : 1;
  const int u0 = min(static_cast<int>(blockIdx.x) * span, total);
  const int u1 = min(u0 + span, total);
  Walker walker{p.paged ? P : nullptr, p.batch, hkvv, tiles_per_req, p.paged ? w : 0};
  if (!p.paged) {
    // Contiguous caches: where this CTA's first tiles lie follows from the launch parameters alone, so
    // while the preceding kernel still runs the TMA unit is asked to bring them into L2 (a hint: nothing
    // reaches the SM, and L2 is where that kernel's writes land too). The first ring fill then comes from
    // L2 with warm address translations instead of paying the cold 2.3 us.
    if (!GATHER && warp == kConsumerWarps && lane == 0 && u0 < u1) {
      int uf = u0;
      const Piece pc = walker.at(uf, u1);
      const int h = pc.hv / p.vblk;
      for (int t = pc.tile0; t < pc.tile0 + min(pc.count, kPrefetchTiles); ++t) {
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
          tma_prefetch_4d(&tm_k, hf * 64, 0, t * kTile, pc.b * p.hkv + h);
          tma_prefetch_4d(&tm_v, hf * 64, 0, t * kTile, pc.b * p.hkv + h);
        }
      }
    }
    pdl_wait();
  }
  pdl_launch_dependents();  // the next kernel's CTAs may take SMs as this grid's CTAs retire

  if (warp >= kConsumerWarps) {
    // ================================================================= producer warp(s)
    int stage = 0, phase = 0;
    Piece pc{};
    for (int u = u0; u < u1;) {
      pc = MODE == kPlain || u == u0 ? walker.at(u, u1) : walker.after(pc, u, u1);
      if (pc.count == 0) break;  // the share ends in front of the next item's tiles
      const int h = MODE != kPlain && p.vblk == 1 ? pc.hv : pc.hv / p.vblk;
      const ItemView view = item_view<MODE, GATHER>(p, MODE != kPlain ? V[pc.b] : item_valid_len(p, pc.b));
      const int valid = view.valid;
      const int page_base = p.paged ? p.kv_indptr[pc.b] : 0;
      const int n_pages = p.paged ? ceil_div(valid, p.page_size) : 0;
      if constexpr (!GATHER) {
        int win = -1, cur_idx = 0, next_idx = 0;
        for (int ti = pc.tile0; ti < pc.tile0 + pc.count; ++ti) {
          const int t = view.tile(ti);
          mbar_wait(&empty_bar[stage], phase ^ 1, p.status, kFaultEmptyBarrier);
          uint8_t* kdst = stages + stage * Plan::kStageBytes;
          uint8_t* vdst = kdst + Plan::kMatBytes;
          // an edge tile of the modes: only the groups of 16 tokens that hold one that takes part
          uint32_t groups = 15;
          if constexpr (MODE != kPlain) {
            if (!tile_whole<MODE, GATHER>(p, view, t * kTile)) {
#pragma unroll
              for (int g = 0; g < 4; ++g)
                if (!group_lives<MODE, GATHER>(p, view, t * kTile + g * 16)) groups ^= 1u << g;
            }
          }
          if (lane == 0) mbar_arrive_expect_tx(&full_bar[stage], MODE == kPlain ? Plan::kStageBytes : __popc(groups) * (Plan::kStageBytes / 4));
          __syncwarp();
          if (p.paged) {
            const int nbox = kTile / p.box_tok;
            for (int j = 0; j < nbox; ++j) {
              const int tok = t * kTile + j * p.box_tok;
              const int pord = min(tok / p.page_size, n_pages - 1);
              const int slot = tok - (tok / p.page_size) * p.page_size;
              const int w = pord >> 5;
              if (w != win) {  // warp-uniform: refill the 32-entry window of page ids
                if (w == win + 1 && win >= 0) {
                  cur_idx = next_idx;
                } else {
                  cur_idx = __ldg(p.kv_indices + page_base + min(w * 32 + lane, n_pages - 1));
                }
                next_idx = __ldg(p.kv_indices + page_base + min((w + 1) * 32 + lane, n_pages - 1));
                win = w;
              }
              int page = __shfl_sync(0xffffffffu, cur_idx, pord & 31);
              page = min(max(page, 0), p.num_pages - 1);
              if (MODE != kPlain && groups != 15) {
                if (lane == 0) {
                  for (int g = 0; g < 4; ++g) {
                    if (!(groups >> g & 1)) continue;
#pragma unroll
                    for (int hf = 0; hf < D / 64; ++hf) {
                      const int off = hf * (kTile * 128) + g * 16 * 128;
                      tma_load_4d(kdst + off, &tm_group.k, &full_bar[stage], hf * 64, h, slot + g * 16, page);
                      tma_load_4d(vdst + off, &tm_group.v, &full_bar[stage], hf * 64, h, slot + g * 16, page);
                    }
                  }
                }
              } else if (lane == 0) {
#pragma unroll
                for (int hf = 0; hf < D / 64; ++hf) {
                  const int off = hf * (kTile * 128) + j * p.box_tok * 128;
                  tma_load_4d(kdst + off, &tm_k, &full_bar[stage], hf * 64, h, slot, page);
                  tma_load_4d(vdst + off, &tm_v, &full_bar[stage], hf * 64, h, slot, page);
                }
              }
            }
          } else if (lane == 0) {
#pragma unroll
            for (int hf = 0; hf < D / 64; ++hf) {
              const int off = hf * (kTile * 128);
              tma_load_4d(kdst + off, &tm_k, &full_bar[stage], hf * 64, 0, t * kTile, pc.b * p.hkv + h);
              tma_load_4d(vdst + off, &tm_v, &full_bar[stage], hf * 64, 0, t * kTile, pc.b * p.hkv + h);
            }
          }
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      } else {
        // Row gather (pages smaller than a tile): eight producer warps copy the 64 token
        // rows of a tile with 16-byte cp.async into the swizzled layout. Consecutive lanes copy
        // consecutive 16-byte chunks of a row, so one warp instruction moves whole rows (full 128-byte
        // lines) instead of a sliver of 32 rows; a thread's arrival on the full barrier fires when its
        // copies have landed. Page ids are read one tile ahead so their latency stays off the
        // critical path.
        const T* kc = reinterpret_cast<const T*>(p.k);
        const T* vc = reinterpret_cast<const T*>(p.v);
        constexpr int kPThreads = Plan::kProducerWarps * 32;
        const int ptid = tid - kConsumerWarps * 32;   // 0..kPThreads-1
        constexpr int kChunks = D / 8;                // 16-byte chunks per row
        constexpr int kRowsPerRound = kPThreads / kChunks;  // rows the copying threads cover at once
        constexpr int kRounds = kTile / kRowsPerRound;
        const int c = ptid % kChunks, r_in = ptid / kChunks;
        if constexpr (MODE == kPlain) {
          auto load_pages = [&](int t, int (&pg)[kRounds]) {
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
              const int tok = min(t * kTile + r * kRowsPerRound + r_in, valid - 1);
              pg[r] = __ldg(p.kv_indices + page_base + tok / p.page_size);
            }
          };
          int pg[kRounds];
          load_pages(pc.tile0, pg);
          for (int t = pc.tile0; t < pc.tile0 + pc.count; ++t) {
            int cur[kRounds];
#pragma unroll
            for (int r = 0; r < kRounds; ++r) cur[r] = pg[r];
            if (t + 1 < pc.tile0 + pc.count) load_pages(t + 1, pg);
            mbar_wait(&empty_bar[stage], phase ^ 1, p.status, kFaultEmptyBarrier);
            const uint32_t kdst = smem_u32(stages + stage * Plan::kStageBytes);
            const uint32_t vdst = kdst + Plan::kMatBytes;
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
              const int row = r * kRowsPerRound + r_in;
              const int tok = min(t * kTile + row, valid - 1);
              const int slot = tok - (tok / p.page_size) * p.page_size;
              const long long page = min(max(cur[r], 0), p.num_pages - 1);
              const long long off = ((page * p.page_size + slot) * p.hkv + h) * D + c * 8;
              const uint32_t dst_off = (c >> 3) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(kdst + dst_off), "l"(kc + off) : "memory");
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(vdst + dst_off), "l"(vc + off) : "memory");
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full_bar[stage])) : "memory");
            if (++stage == kStages) { stage = 0; phase ^= 1; }
          }
        } else {
          // The copying warps are bound by the instructions they issue for an address, not by the memory: pages of a
          // power of two of tokens are found by a shift (a division a row cost a third of the rate), a token's place in
          // the pool is a 32-bit number (the host has checked), and only tiles at an edge look at which groups live.
          const uint32_t row_bytes = static_cast<uint32_t>(p.hkv) * D * 2;
          const char* kcol = reinterpret_cast<const char*>(kc + h * D + c * 8);
          const char* vcol = reinterpret_cast<const char*>(vc + h * D + c * 8);
          auto stream = [&](auto pow2) {
            constexpr bool POW2 = decltype(pow2)::value;
            auto load_pages = [&](int t, int (&pg)[kRounds]) {
#pragma unroll
              for (int r = 0; r < kRounds; ++r) {
                const int tok = view.token(min(t * kTile + r * kRowsPerRound + r_in, valid - 1));
                pg[r] = __ldg(p.kv_indices + page_base + (POW2 ? tok >> p.page_shift : tok / p.page_size));
              }
            };
            int pg[kRounds];
            load_pages(view.tile(pc.tile0), pg);
            for (int ti = pc.tile0; ti < pc.tile0 + pc.count; ++ti) {
              const int t = view.tile(ti);
              uint32_t at[kRounds];  // the rows' places in the pool
#pragma unroll
              for (int r = 0; r < kRounds; ++r) {
                const int tok = view.token(min(t * kTile + r * kRowsPerRound + r_in, valid - 1)), page = min(max(pg[r], 0), p.num_pages - 1);
                at[r] = POW2 ? (static_cast<uint32_t>(page) << p.page_shift) + (tok & (p.page_size - 1))
                             : static_cast<uint32_t>(page) * p.page_size + tok % p.page_size;
              }
              if (ti + 1 < pc.tile0 + pc.count) load_pages(view.tile(ti + 1), pg);
              mbar_wait(&empty_bar[stage], phase ^ 1, p.status, kFaultEmptyBarrier);
              const uint32_t kdst = smem_u32(stages + stage * Plan::kStageBytes);
              const uint32_t vdst = kdst + Plan::kMatBytes;
              auto copy = [&](int r) {
                const int row = r * kRowsPerRound + r_in;
                const uint64_t off = static_cast<uint64_t>(at[r]) * row_bytes;
                const uint32_t dst_off = (c >> 3) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(kdst + dst_off), "l"(kcol + off) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(vdst + dst_off), "l"(vcol + off) : "memory");
              };
              if (tile_whole<MODE, GATHER>(p, view, t * kTile)) {
#pragma unroll
                for (int r = 0; r < kRounds; ++r) copy(r);
              } else {
#pragma unroll
                for (int r = 0; r < kRounds; ++r)
                  if (group_lives<MODE, GATHER>(p, view, t * kTile + ((r * kRowsPerRound + r_in) & ~15))) copy(r);
              }
              asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full_bar[stage])) : "memory");
              if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
          };
          if (p.page_shift >= 0) stream(std::true_type{});
          else stream(std::false_type{});
        }
      }
      u += pc.count;
    }
    return;
  }

  // =================================================================== consumer warps
  const int ctid = tid;  // 0 .. kConsumerWarps*32-1
  constexpr int kCThreads = kConsumerWarps * 32;
  T* outp = reinterpret_cast<T*>(p.out);

  // Requests without any live token: out = 0, lse = -inf (behind a prefix: the prefix alone, further down).
  if (MODE != kSuffix && p.paged) {
    const int rows_all = p.hkv * p.rows;  // query rows per request
    for (int b = blockIdx.x; b < p.batch; b += G) {
      if (P[b + 1] - P[b] != 0) continue;
      for (int i = ctid; i < rows_all * D; i += kCThreads) outp[static_cast<size_t>(b) * rows_all * D + i] = T(0.f);
      if (p.lse)
        for (int i = ctid; i < rows_all; i += kCThreads) p.lse[static_cast<size_t>(b) * rows_all + i] = -INFINITY;
    }
  }

  constexpr float kHeadroom = MODE == kPlain ? 0.f : weight_headroom<T>(0.f);  // P is at most 1

  const int ws = warp;  // token slice of this warp inside a tile
  const int r0 = lane >> 2, c2 = (lane & 3) * 2;
  const uint32_t stages_u32 = smem_u32(stages);
  float* my_merge = merge + warp * Plan::kMergeFloats;
  const int slot_floats = Plan::kSlotFloats;

  constexpr int kColsPerThread = kRowsMax * D / kCThreads;  // 16 (D=128) or 8 (D=64)
  constexpr int kThreadsPerRow = kCThreads / kRowsMax;      // 8
  // a thread's columns of its row: four from mcol on, and from mcol + 32, mcol + 64 ... on
  const int mrow = ctid / kThreadsPerRow, mcol = (ctid % kThreadsPerRow) * 4;
  constexpr int kQuads = kColsPerThread / 4;
  // Writes one row's columns of a thread: `of` relative to the maximum Mf, with the sum Lf.
  auto store_final = [&](int b, int h, int blk, int rows_here, float Mf, float Lf, float* of) {
    if (mrow >= rows_here) return;
    const size_t row = (static_cast<size_t>(b) * p.hkv + h) * p.rows + blk * kRowsMax + mrow;
    if constexpr (MODE == kSuffix) {
      if (p.pre_splits > 0) {  // merge_prefix has left the prefix's sum for the item's rows in the merge buffer
        const float Mp = merge[kRowsMax * D + mrow], Lp = merge[kRowsMax * D + kRowsMax + mrow];
        const float Mn = fmaxf(Mf, Mp), Mu = Mn == -INFINITY ? 0.f : Mn;
        const float fa = fast_exp2(Mf - Mu), fb = fast_exp2(Mp - Mu);
        Lf = fa * Lf + fb * Lp;
#pragma unroll
        for (int c = 0; c < kColsPerThread; ++c) of[c] = fa * of[c] + fb * merge[mrow * D + mcol + (c >> 2) * 32 + (c & 3)];
        Mf = Mn;
      }
    }
    const bool some = MODE == kPlain ? Lf > 0.f : Lf != 0.f;  // modes: the sum of a row with a NaN score is NaN, and so is the row
    const float inv = some ? 1.f / Lf : 0.f;
    T* dst = outp + row * D + mcol;
#pragma unroll
    for (int k = 0; k < kQuads; ++k)
      *reinterpret_cast<uint2*>(dst + 32 * k) = make_uint2(pack2<T>(of[4 * k] * inv, of[4 * k + 1] * inv), pack2<T>(of[4 * k + 2] * inv, of[4 * k + 3] * inv));
    if (p.lse && mcol == 0) p.lse[row] = some ? Mf + fast_log2(Lf) : -INFINITY;
  };
  // kSuffix, all consumer threads: the partials of the prefix for an item's rows, summed into the merge buffer (rows of
  // O, then maxima and sums). A thread takes four columns of one row through all parts of the prefix, eight parts in
  // flight, so that a group of four query heads costs one or two round trips to L2 with every thread at work.
  auto merge_prefix = [&](int b, int h, int blk, int rows_here) {
    if (p.pre_splits == 0) return;
    pdl_wait();
    named_bar_sync(1, kCThreads);  // nobody reads the buffer any more
    const size_t part0 = (static_cast<size_t>(h) * p.pre_blocks + b / p.pre_batch) * p.pre_splits;
    const int prow0 = (b % p.pre_batch) * p.rows + blk * kRowsMax;
    constexpr int kGroup = 8;
    for (int i = ctid; i < rows_here * (D / 4); i += kCThreads) {
      const int row = i / (D / 4), col = i % (D / 4) * 4;
      const float* ml = p.pre_ml + part0 * 256 + prow0 + row;
      const float* o = p.pre_o + (part0 * 128 + prow0 + row) * D + col;
      float M = -INFINITY, L = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s0 = 0; s0 < p.pre_splits; s0 += kGroup) {
        float m[kGroup], l[kGroup];
        float4 x[kGroup];
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
          const int s = min(s0 + g, p.pre_splits - 1);
          m[g] = __ldcg(ml + s * 256);
          l[g] = __ldcg(ml + s * 256 + 128);
          x[g] = __ldcg(reinterpret_cast<const float4*>(o + static_cast<size_t>(s) * 128 * D));
        }
        float Mn = M;
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
          if (s0 + g >= p.pre_splits) m[g] = -INFINITY;  // a part that was loaded twice
          Mn = fmaxf(Mn, m[g]);
        }
        const float Mu = Mn == -INFINITY ? 0.f : Mn, f = fast_exp2(M - Mu);
        L *= f;
        sum.x *= f, sum.y *= f, sum.z *= f, sum.w *= f;
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
          const float w = fast_exp2(m[g] - Mu);
          L += w * l[g];
          sum.x += w * x[g].x;
          sum.y += w * x[g].y;
          sum.z += w * x[g].z;
          sum.w += w * x[g].w;
        }
        M = Mn;
      }
      *reinterpret_cast<float4*>(merge + row * D + col) = sum;
      if (col == 0) {
        merge[kRowsMax * D + row] = M;
        merge[kRowsMax * D + kRowsMax + row] = L;
      }
    }
    named_bar_sync(1, kCThreads);
  };

  // Q fragments (A operand) of a piece's rows; those beyond its last are zero
  uint32_t qf[D / 16][4];
  auto load_q = [&](const Piece& piece) {
    const int h = MODE != kPlain && p.vblk == 1 ? piece.hv : piece.hv / p.vblk, blk = piece.hv - h * p.vblk;
    const int rows_here = min(kRowsMax, p.rows - blk * kRowsMax);
    const size_t row_base = (static_cast<size_t>(piece.b) * p.hkv + h) * p.rows + blk * kRowsMax;
    const T* qrow0 = reinterpret_cast<const T*>(p.q) + (row_base + r0) * D;
    const T* qrow1 = qrow0 + 8 * D;
    const bool ok0 = r0 < rows_here, ok1 = r0 + 8 < rows_here;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const int d = kk * 16 + c2;
      qf[kk][0] = ok0 ? *reinterpret_cast<const uint32_t*>(qrow0 + d) : 0u;
      qf[kk][1] = ok1 ? *reinterpret_cast<const uint32_t*>(qrow1 + d) : 0u;
      qf[kk][2] = ok0 ? *reinterpret_cast<const uint32_t*>(qrow0 + d + 8) : 0u;
      qf[kk][3] = ok1 ? *reinterpret_cast<const uint32_t*>(qrow1 + d + 8) : 0u;
    }
  };

  int stage = 0, phase = 0;
  Piece pc{}, next{};
  int u_next = u0;
  for (int u = u0; u < u1; u = u_next) {
    if (MODE == kPlain || u == u0) {
      pc = walker.at(u, u1);
      if (pc.count > 0) load_q(pc);
    } else {
      pc = next;
    }
    if (pc.count == 0) break;  // the share ends in front of the next item's tiles
    u_next = u + pc.count;
    const int h = MODE != kPlain && p.vblk == 1 ? pc.hv : pc.hv / p.vblk, blk = pc.hv - h * p.vblk;
    const ItemView view = item_view<MODE, GATHER>(p, MODE != kPlain ? V[pc.b] : item_valid_len(p, pc.b));
    const int valid = view.valid;
    const int rows_here = min(kRowsMax, p.rows - blk * kRowsMax);
    const size_t row_base = (static_cast<size_t>(pc.b) * p.hkv + h) * p.rows + blk * kRowsMax;

    float acc[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

    for (int t = pc.tile0; MODE == kPlain && t < pc.tile0 + pc.count; ++t) {
      mbar_wait(&full_bar[stage], phase, p.status, kFaultFullBarrier);
      const int tok0 = t * kTile + ws * 16;
      if (tok0 < valid) {
        const uint32_t kbase = stages_u32 + stage * Plan::kStageBytes;
        const uint32_t vbase = kbase + Plan::kMatBytes;
        const int mi = lane >> 3, rr = lane & 7;
        // ---- S = Q K^T for this warp's 16 tokens
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        {
          const int row = ws * 16 + (mi >> 1) * 8 + rr;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const int d = kk * 16 + (mi & 1) * 8;
            const uint32_t addr = kbase + (d >> 6) * (kTile * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4);
            uint32_t b0, b1, b2, b3;
            ldmatrix_x4(b0, b1, b2, b3, addr);
            mma_16816<T>(s[0], qf[kk], b0, b1);
            mma_16816<T>(s[1], qf[kk], b2, b3);
          }
        }
        // ---- online softmax (exp2 domain)
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = tok0 + nb * 8 + c2 + (e & 1);
            const float x = tok < valid ? s[nb][e] * p.scale_log2 : -INFINITY;
            s[nb][e] = x;
            if (e < 2) mx0 = fmaxf(mx0, x); else mx1 = fmaxf(mx1, x);
          }
        }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float mn0 = fmaxf(m_run[0], mx0), mn1 = fmaxf(m_run[1], mx1);
        const float mu0 = mn0 == -INFINITY ? 0.f : mn0, mu1 = mn1 == -INFINITY ? 0.f : mn1;
        const float sc0 = fast_exp2(m_run[0] - mu0), sc1 = fast_exp2(m_run[1] - mu1);
        m_run[0] = mn0;
        m_run[1] = mn1;
        uint32_t pf[4];
        float ps0 = 0.f, ps1 = 0.f;
        {
          const float p00 = fast_exp2(s[0][0] - mu0), p01 = fast_exp2(s[0][1] - mu0);
          const float p02 = fast_exp2(s[0][2] - mu1), p03 = fast_exp2(s[0][3] - mu1);
          const float p10 = fast_exp2(s[1][0] - mu0), p11 = fast_exp2(s[1][1] - mu0);
          const float p12 = fast_exp2(s[1][2] - mu1), p13 = fast_exp2(s[1][3] - mu1);
          ps0 = p00 + p01 + p10 + p11;
          ps1 = p02 + p03 + p12 + p13;
          pf[0] = pack2<T>(p00, p01);
          pf[1] = pack2<T>(p02, p03);
          pf[2] = pack2<T>(p10, p11);
          pf[3] = pack2<T>(p12, p13);
        }
        l_run[0] = l_run[0] * sc0 + ps0;
        l_run[1] = l_run[1] * sc1 + ps1;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          acc[n][0] *= sc0;
          acc[n][1] *= sc0;
          acc[n][2] *= sc1;
          acc[n][3] *= sc1;
        }
        // ---- O += P V
        {
          const int row = ws * 16 + (mi & 1) * 8 + rr;
#pragma unroll
          for (int dp = 0; dp < D / 16; ++dp) {
            const int d = dp * 16 + (mi >> 1) * 8;
            const uint32_t addr = vbase + (d >> 6) * (kTile * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4);
            uint32_t b0, b1, b2, b3;
            ldmatrix_x4_trans(b0, b1, b2, b3, addr);
            mma_16816<T>(acc[2 * dp], pf, b0, b1);
            mma_16816<T>(acc[2 * dp + 1], pf, b2, b3);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[stage]);
      if (++stage == kStages) { stage = 0; phase ^= 1; }
    }

    // The other modes. A warp takes its 16 tokens of TWO tiles a step where all of them take part, and of one otherwise
    // (a request's last tile, the edges of a window): with 32 tokens in hand the two chains of score MMAs overlap, and
    // the reductions of the maximum cost half as much a token. O is rescaled only when a maximum has grown, which
    // after the first tiles is rare; the factor would be exactly 1. (64 requests of 512..8192 tokens in 16-token pages,
    // weights mode: 274 us a tile at a time with a rescale each, 248 so.)
    if constexpr (MODE != kPlain) {
      const int mi = lane >> 3, rr = lane & 7;
      auto takes_part = [&](int tok) { return token_lives<MODE, GATHER>(p, view, tok); };
      auto step = [&](int ti, auto tiles, auto edge) {
        constexpr int N = decltype(tiles)::value;
        constexpr bool EDGE = decltype(edge)::value;  // some of the tokens may not take part
        uint32_t kbase[N];
        int tok0[N];
        uint64_t* freed[N];
        bool some = !EDGE;
#pragma unroll
        for (int u = 0; u < N; ++u) {
          tok0[u] = view.tile(ti + u) * kTile + ws * 16;
          if (EDGE) some = group_lives<MODE, GATHER>(p, view, tok0[u]);
          kbase[u] = stages_u32 + stage * Plan::kStageBytes;
          freed[u] = &empty_bar[stage];
          mbar_wait(&full_bar[stage], phase, p.status, kFaultFullBarrier);
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        if (some) {
          // ---- S = Q K^T
          float s[N][2][4];
#pragma unroll
          for (int u = 0; u < N; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[u][0][e] = s[u][1][e] = 0.f;
          {
            const int row = ws * 16 + (mi >> 1) * 8 + rr;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const int d = kk * 16 + (mi & 1) * 8;
              const uint32_t at = (d >> 6) * (kTile * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4);
#pragma unroll
              for (int u = 0; u < N; ++u) {
                uint32_t b0, b1, b2, b3;
                ldmatrix_x4(b0, b1, b2, b3, kbase[u] + at);
                mma_16816<T>(s[u][0], qf[kk], b0, b1);
                mma_16816<T>(s[u][1], qf[kk], b2, b3);
              }
            }
          }
          // ---- online softmax (exp2 domain)
          float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
          for (int u = 0; u < N; ++u)
#pragma unroll
            for (int nb = 0; nb < 2; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float x = s[u][nb][e] * p.scale_log2;
                if (EDGE && !takes_part(tok0[u] + nb * 8 + c2 + (e & 1))) x = -INFINITY;
                s[u][nb][e] = x;
                if (e < 2) mx0 = fmaxf(mx0, x); else mx1 = fmaxf(mx1, x);
              }
          if constexpr (MODE == kWeights) {
            // a warp instruction writes 32-byte runs of eight rows; the scratch rows are padded to whole runs
#pragma unroll
            for (int u = 0; u < N; ++u) {
              float* raw = p.raw + (row_base + r0) * p.raw_pitch + tok0[u] + c2;
#pragma unroll
              for (int nb = 0; nb < 2; ++nb) {
                if (tok0[u] + nb * 8 < p.raw_len) {
                  if (r0 < rows_here) *reinterpret_cast<float2*>(raw + nb * 8) = make_float2(s[u][nb][0], s[u][nb][1]);
                  if (r0 + 8 < rows_here) *reinterpret_cast<float2*>(raw + 8 * p.raw_pitch + nb * 8) = make_float2(s[u][nb][2], s[u][nb][3]);
                }
              }
            }
          }
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
          if (__any_sync(0xffffffffu, mx0 > m_run[0] || mx1 > m_run[1])) {
            const float mn0 = fmaxf(m_run[0], mx0), mn1 = fmaxf(m_run[1], mx1);
            const float sc0 = mn0 == -INFINITY ? 0.f : fast_exp2(m_run[0] - mn0), sc1 = mn1 == -INFINITY ? 0.f : fast_exp2(m_run[1] - mn1);
            m_run[0] = mn0;
            m_run[1] = mn1;
            l_run[0] *= sc0;
            l_run[1] *= sc1;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              acc[n][0] *= sc0;
              acc[n][1] *= sc0;
              acc[n][2] *= sc1;
              acc[n][3] *= sc1;
            }
          }
          const float mu0 = m_run[0] == -INFINITY ? 0.f : m_run[0] - kHeadroom, mu1 = m_run[1] == -INFINITY ? 0.f : m_run[1] - kHeadroom;
#pragma unroll
          for (int u = 0; u < N; ++u) {
            // ---- P, as the sum of two 16-bit numbers
            uint32_t hi[4], rest[4];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
              const float p0 = fast_exp2(s[u][nb][0] - mu0), p1 = fast_exp2(s[u][nb][1] - mu0);
              const float p2 = fast_exp2(s[u][nb][2] - mu1), p3 = fast_exp2(s[u][nb][3] - mu1);
              l_run[0] += p0 + p1;
              l_run[1] += p2 + p3;
              hi[2 * nb] = pack2<T>(p0, p1);
              hi[2 * nb + 1] = pack2<T>(p2, p3);
              rest[2 * nb] = pack2_rest<T>(p0, p1, hi[2 * nb]);
              rest[2 * nb + 1] = pack2_rest<T>(p2, p3, hi[2 * nb + 1]);
            }
            // ---- O += P V. Values of tokens that take no part become zero: 0 * V is not 0 where the row holds Inf or
            // NaN. A register of the V fragment holds two tokens (c2, c2 + 1, or those plus 8) of one column.
            uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
            if constexpr (EDGE) {
              const int tk = tok0[u] + c2;
              keep0 = (takes_part(tk) ? 0xffffu : 0u) | (takes_part(tk + 1) ? 0xffff0000u : 0u);
              keep1 = (takes_part(tk + 8) ? 0xffffu : 0u) | (takes_part(tk + 9) ? 0xffff0000u : 0u);
            }
            const uint32_t vbase = kbase[u] + Plan::kMatBytes;
            const int row = ws * 16 + (mi & 1) * 8 + rr;
#pragma unroll
            for (int dp = 0; dp < D / 16; ++dp) {
              const int d = dp * 16 + (mi >> 1) * 8;
              uint32_t b0, b1, b2, b3;
              ldmatrix_x4_trans(b0, b1, b2, b3, vbase + (d >> 6) * (kTile * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4));
              if constexpr (EDGE) {
                b0 &= keep0;
                b1 &= keep1;
                b2 &= keep0;
                b3 &= keep1;
              }
              mma_16816<T>(acc[2 * dp], hi, b0, b1);
              mma_16816<T>(acc[2 * dp + 1], hi, b2, b3);
              mma_16816<T>(acc[2 * dp], rest, b0, b1);
              mma_16816<T>(acc[2 * dp + 1], rest, b2, b3);
            }
          }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < N; ++u)
          if (lane == 0) mbar_arrive(freed[u]);
      };
      auto whole = [&](int ti) {  // every token of the tile takes part (the same for the four warps)
        return tile_whole<MODE, GATHER>(p, view, view.tile(ti) * kTile);
      };
      for (int ti = pc.tile0; ti < pc.tile0 + pc.count;) {
        if (ti + 1 < pc.tile0 + pc.count && whole(ti) && whole(ti + 1)) {
          step(ti, std::integral_constant<int, 2>{}, std::false_type{});
          ti += 2;
        } else {
          step(ti, std::integral_constant<int, 1>{}, std::true_type{});
          ti += 1;
        }
      }
    }

    if constexpr (MODE != kPlain) {
      // The next piece's rows of Q are on their way while this one's states are merged (128 requests of 100 .. 2048 tokens,
      // 16-token pages: 108.7 -> 104.2 us)
      next = walker.after(pc, u_next, u1);
      if (next.count > 0) load_q(next);
    }

    // ---- merge the four warps' states through shared memory
    l_run[0] += __shfl_xor_sync(0xffffffffu, l_run[0], 1);
    l_run[0] += __shfl_xor_sync(0xffffffffu, l_run[0], 2);
    l_run[1] += __shfl_xor_sync(0xffffffffu, l_run[1], 1);
    l_run[1] += __shfl_xor_sync(0xffffffffu, l_run[1], 2);
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      *reinterpret_cast<float2*>(my_merge + r0 * Plan::kMergePitch + n * 8 + c2) = make_float2(acc[n][0], acc[n][1]);
      *reinterpret_cast<float2*>(my_merge + (r0 + 8) * Plan::kMergePitch + n * 8 + c2) = make_float2(acc[n][2], acc[n][3]);
    }
    if ((lane & 3) == 0) {
      my_merge[kRowsMax * Plan::kMergePitch + r0] = m_run[0] - kHeadroom;
      my_merge[kRowsMax * Plan::kMergePitch + r0 + 8] = m_run[1] - kHeadroom;
      my_merge[kRowsMax * Plan::kMergePitch + kRowsMax + r0] = l_run[0];
      my_merge[kRowsMax * Plan::kMergePitch + kRowsMax + r0 + 8] = l_run[1];
    }
    named_bar_sync(1, kCThreads);

    float M = -INFINITY, L = 0.f, o[kColsPerThread];
    {
      float mw[kConsumerWarps];
#pragma unroll
      for (int w = 0; w < kConsumerWarps; ++w) {
        mw[w] = merge[w * Plan::kMergeFloats + kRowsMax * Plan::kMergePitch + mrow];
        M = fmaxf(M, mw[w]);
      }
      const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int c = 0; c < kColsPerThread; ++c) o[c] = 0.f;
#pragma unroll
      for (int w = 0; w < kConsumerWarps; ++w) {
        const float cf = fast_exp2(mw[w] - Mu);
        L += cf * merge[w * Plan::kMergeFloats + kRowsMax * Plan::kMergePitch + kRowsMax + mrow];
        const float* src = merge + w * Plan::kMergeFloats + mrow * Plan::kMergePitch + mcol;
#pragma unroll
        for (int c = 0; c < kColsPerThread; c += 4) {
          const float4 x = *reinterpret_cast<const float4*>(src + 8 * c);
          o[c] += cf * x.x;
          o[c + 1] += cf * x.y;
          o[c + 2] += cf * x.z;
          o[c + 3] += cf * x.w;
        }
      }
    }

    const bool starts_here = (u == pc.unit0);
    const bool whole = starts_here && pc.count == pc.n_tiles;
    if (whole) {
      if constexpr (MODE == kSuffix) merge_prefix(pc.b, h, blk, rows_here);
      store_final(pc.b, h, blk, rows_here, M, L, o);
    } else {
      // ---- leave a partial, then let the last arriver combine
      float* slot = p.partials + (static_cast<size_t>(blockIdx.x) * 2 + (starts_here ? 1 : 0)) * slot_floats;
      if (mrow < rows_here) {
#pragma unroll
        for (int c = 0; c < kColsPerThread; c += 4)
          *reinterpret_cast<float4*>(slot + mrow * D + mcol + 8 * c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        if (mcol == 0) {
          slot[kRowsMax * D + mrow] = M;
          slot[kRowsMax * D + kRowsMax + mrow] = L;
        }
      }
      __threadfence();
      named_bar_sync(1, kCThreads);
      const int c_first = pc.unit0 / span, c_last = (pc.unit0 + pc.n_tiles - 1) / span;
      int* counter = p.counters + pc.b * hkvv + pc.hv;
      if (ctid == 0) {
        const int old = atomicAdd(counter, 1);
        flags[0] = (old == c_last - c_first) ? 1 : 0;
      }
      named_bar_sync(1, kCThreads);
      if (flags[0]) {
        __threadfence();
        float Mc = -INFINITY, Lc = 0.f, oc[kColsPerThread];
#pragma unroll
        for (int c = 0; c < kColsPerThread; ++c) oc[c] = 0.f;
        if (mrow < rows_here) {
          // the partials of up to four CTAs are fetched together: one L2 round trip per group instead of
          // one per CTA (an item of a long request can span every CTA of the grid)
          constexpr int kGroup = 4, kVec = kColsPerThread / 4;
          for (int cta0 = c_first; cta0 <= c_last; cta0 += kGroup) {
            float mi_[kGroup], li_[kGroup];
            float4 x[kGroup][kVec];
#pragma unroll
            for (int g = 0; g < kGroup; ++g) {
              const int cta = min(cta0 + g, c_last);  // a repeated slot is given weight zero below
              const float* src = p.partials + (static_cast<size_t>(cta) * 2 + (cta == c_first ? 1 : 0)) * slot_floats;
              mi_[g] = __ldcg(src + kRowsMax * D + mrow);
              li_[g] = __ldcg(src + kRowsMax * D + kRowsMax + mrow);
#pragma unroll
              for (int c = 0; c < kVec; ++c) x[g][c] = __ldcg(reinterpret_cast<const float4*>(src + mrow * D + mcol + 32 * c));
            }
#pragma unroll
            for (int g = 0; g < kGroup; ++g) {
              if (cta0 + g > c_last) continue;
              const float Mn = fmaxf(Mc, mi_[g]);
              const float Mu = Mn == -INFINITY ? 0.f : Mn;
              const float a = fast_exp2(Mc - Mu), bb = fast_exp2(mi_[g] - Mu);
              Lc = a * Lc + bb * li_[g];
#pragma unroll
              for (int c = 0; c < kVec; ++c) {
                oc[4 * c] = a * oc[4 * c] + bb * x[g][c].x;
                oc[4 * c + 1] = a * oc[4 * c + 1] + bb * x[g][c].y;
                oc[4 * c + 2] = a * oc[4 * c + 2] + bb * x[g][c].z;
                oc[4 * c + 3] = a * oc[4 * c + 3] + bb * x[g][c].w;
              }
              Mc = Mn;
            }
          }
        }
        if constexpr (MODE == kSuffix) merge_prefix(pc.b, h, blk, rows_here);
        store_final(pc.b, h, blk, rows_here, Mc, Lc, oc);
        if (ctid == 0) *counter = 0;  // ready for the next launch
      }
    }
    named_bar_sync(1, kCThreads);  // merge buffer and flag are free again
  }
  if constexpr (MODE == kSuffix) {
    // requests with nothing behind the prefix; their (request, kv head) pairs are shared out over the CTAs
    for (int i = blockIdx.x; i < p.batch * hkvv; i += G) {
      const int b = i / hkvv, hv = i - b * hkvv, h = hv / p.vblk, blk = hv - h * p.vblk;
      if (P[b + 1] - P[b] != 0) continue;
      float none[kColsPerThread];
#pragma unroll
      for (int c = 0; c < kColsPerThread; ++c) none[c] = 0.f;
      const int rows_here = min(kRowsMax, p.rows - blk * kRowsMax);
      merge_prefix(b, h, blk, rows_here);
      store_final(b, h, blk, rows_here, -INFINITY, 0.f, none);
    }
    pdl_wait();  // a CTA that merged nothing: the grid is not done before the prefix's is
  }
}

// ------------------------------------------------------------------------------------- host side
namespace {

struct DecodeSetup {
  DecodeParams p;
  bool gather;
  bool overlap;  // the launch may start while its predecessor drains; not for a caller that bounds the grid, see bounded()
  int grid, smem_bytes;
  size_t ws_needed, counters_off, partials_off;
  CUtensorMap tm_k, tm_v;
  GroupMaps tm_group;
};

// Whether max_ctas leaves less than the device. An operator of two kernels then keeps each of them to the bound and does not
// let the second start beside the first.
bool bounded(const cb200_attn_decode_args* a) { return a->max_ctas > 0 && a->max_ctas < sm_count(); }

int plan_decode(const cb200_attn_decode_args* a, DecodeSetup* s, bool need_maps, bool modes = false) {
  if (!a) return CB200_ERR_BAD_ARG;
  if (a->batch <= 0 || a->num_qo_heads <= 0 || a->num_kv_heads <= 0) return CB200_ERR_BAD_ARG;
  if (a->num_qo_heads % a->num_kv_heads) return CB200_ERR_BAD_ARG;
  if (a->head_dim != 64 && a->head_dim != 128) return CB200_ERR_UNSUPPORTED;
  if (a->dtype != CB200_F16 && a->dtype != CB200_BF16) return CB200_ERR_UNSUPPORTED;
  const bool paged = a->kv_indptr != nullptr;
  const int D = a->head_dim;
  const int q_rows = a->q_rows > 1 ? a->q_rows : 1;
  const int rows = (a->num_qo_heads / a->num_kv_heads) * q_rows;
  DecodeParams& p = s->p;
  p = DecodeParams{};
  p.batch = a->batch;
  p.hkv = a->num_kv_heads;
  p.rows = rows;
  p.vblk = ceil_div(rows, kRowsMax);
  p.paged = paged ? 1 : 0;
  p.scale_log2 = a->sm_scale * kLog2e;
  long long tiles_ub;
  if (paged) {
    if (a->page_size <= 0 || a->num_pages <= 0 || a->num_kv_indices < 0) return CB200_ERR_BAD_ARG;
    p.page_size = a->page_size;
    p.num_pages = a->num_pages;
    p.n_idx = a->num_kv_indices;
    const int ps = a->page_size;
    // Pages of a whole tile (64 tokens) or more are fetched as TMA boxes; smaller pages would need several
    // small boxes per tile (measured 2.8 TB/s at 16 tokens, 4.3 at 32, 6.0 at 64) and take the row gather
    // instead (5.3 - 5.5 TB/s at any page size).
    s->gather = !(ps >= kTile && ps % kTile == 0);
    p.page_shift = -1;
    if ((ps & (ps - 1)) == 0)
      for (p.page_shift = 0; (1 << p.page_shift) < ps;) ++p.page_shift;
    p.box_tok = kTile;
    tiles_ub = (static_cast<long long>(a->num_kv_indices) * ps + kTile - 1) / kTile + static_cast<long long>(a->batch) * (1 + kPieceUnits);
  } else {
    if (a->kv_len <= 0) return CB200_ERR_BAD_ARG;
    p.kv_len = a->kv_len;
    s->gather = false;
    p.box_tok = kTile;
    tiles_ub = static_cast<long long>(a->batch) * ceil_div(a->kv_len, kTile);
  }
  const long long units_ub = tiles_ub * p.hkv * p.vblk;
  // The kernel counts tiles in 32 bits. Requests may share pages (overlapping kv_indptr ranges), so the
  // bound for that count is every request spanning the whole table, not the table's own size.
  const long long tiles_max = paged ? static_cast<long long>(a->batch) * ((static_cast<long long>(a->num_kv_indices) * a->page_size + kTile - 1) / kTile + 1 + kPieceUnits)
                                    : tiles_ub;
  if (tiles_max * p.hkv * p.vblk >= (1LL << 31)) return CB200_ERR_UNSUPPORTED;
  // the modes hold a token's place in the pool in 32 bits (2^31 tokens would be 256 GB of the narrowest rows), and its
  // place in its request, rounded up to whole tiles, with a sign
  if (modes && paged && (static_cast<long long>(a->num_pages) * a->page_size >= (1LL << 31) ||
                         static_cast<long long>(a->num_kv_indices) * a->page_size > (1LL << 30)))
    return CB200_ERR_UNSUPPORTED;
  const int sms = sm_count();
  if (sms <= 0) return CB200_ERR_CUDA;
  int grid = sms;
  if (a->max_ctas > 0 && a->max_ctas < grid) grid = a->max_ctas;
  // The workspace is sized for a full grid so that one allocation serves every launch.
  const int fixed = modes ? (D == 128 ? SmemPlan<128, false, kWindow>::kFixedBytes : SmemPlan<64, false, kWindow>::kFixedBytes)
                          : (D == 128 ? SmemPlan<128, false, kPlain>::kFixedBytes : SmemPlan<64, false, kPlain>::kFixedBytes);
  s->smem_bytes = fixed + (paged ? (a->batch + 1 + (modes ? a->batch : 0)) * 4 : 0) + 1024 + 16;
  if (s->smem_bytes > 227 * 1024) return CB200_ERR_UNSUPPORTED;  // too many requests for one launch
  // Layout: header | partial slots (two per SM, sized for head_dim 128) | arrival counters.
  // The counters sit at an offset that does not depend on the problem shape: launches of
  // different shapes may share one workspace, and a region that one launch used for partials
  // is never read as counters by the next.
  constexpr size_t kSlotBytesMax = (kRowsMax * 128 + 2 * kRowsMax) * 4;
  s->partials_off = kWsHeaderBytes;
  s->counters_off = align_up(s->partials_off + static_cast<size_t>(sms) * 2 * kSlotBytesMax, 256);
  s->ws_needed = s->counters_off + static_cast<size_t>(a->batch) * p.hkv * p.vblk * 4;
  p.piece_units = (tiles_ub - static_cast<long long>(a->batch) * kPieceUnits) * p.hkv * p.vblk <= grid ? 0 : kPieceUnitsModes;
  s->grid = static_cast<int>(units_ub < grid ? (units_ub > 0 ? units_ub : 1) : grid);
  s->overlap = true;
  if (!need_maps) return CB200_OK;

  if (!a->q || !a->k_cache || !a->v_cache || !a->out) return CB200_ERR_BAD_ARG;
  if (paged && !a->kv_indices && a->num_kv_indices > 0) return CB200_ERR_BAD_ARG;
  if (paged && a->page_size != 1 && !a->kv_last_page_len) return CB200_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k_cache) |
       reinterpret_cast<uintptr_t>(a->v_cache) | reinterpret_cast<uintptr_t>(a->out)) & 15)
    return CB200_ERR_ALIGNMENT;
  if (!a->workspace || a->workspace_bytes < s->ws_needed) return CB200_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 255) return CB200_ERR_ALIGNMENT;
  p.q = a->q;
  p.k = a->k_cache;
  p.v = a->v_cache;
  p.kv_indptr = a->kv_indptr;
  p.kv_indices = a->kv_indices;
  p.kv_last = a->kv_last_page_len;
  p.out = a->out;
  p.lse = a->lse;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.status = reinterpret_cast<int*>(ws);
  p.counters = reinterpret_cast<int*>(ws + s->counters_off);
  p.partials = reinterpret_cast<float*>(ws + s->partials_off);

  if (!s->gather) {
    const CUtensorMapDataType dt = a->dtype == CB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    uint64_t dims[4], strides[3];
    uint32_t box[4] = {64u, 1u, static_cast<uint32_t>(p.box_tok), 1u};
    const uint64_t rowb = static_cast<uint64_t>(D) * 2;
    if (paged) {
      dims[0] = D; dims[1] = p.hkv; dims[2] = p.page_size; dims[3] = p.num_pages;
      strides[0] = rowb; strides[1] = rowb * p.hkv; strides[2] = rowb * p.hkv * p.page_size;
    } else {
      dims[0] = D; dims[1] = 1; dims[2] = p.kv_len; dims[3] = static_cast<uint64_t>(p.batch) * p.hkv;
      strides[0] = rowb; strides[1] = rowb; strides[2] = rowb * p.kv_len;
    }
    if (!encode_tensor_map(&s->tm_k, dt, 4, const_cast<void*>(a->k_cache), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tensor_map(&s->tm_v, dt, 4, const_cast<void*>(a->v_cache), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return CB200_ERR_CUDA;
    memset(&s->tm_group, 0, sizeof(GroupMaps));
    box[2] = 16u;
    if (modes && (!encode_tensor_map(&s->tm_group.k, dt, 4, const_cast<void*>(a->k_cache), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B) ||
                   !encode_tensor_map(&s->tm_group.v, dt, 4, const_cast<void*>(a->v_cache), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)))
      return CB200_ERR_CUDA;
  } else {
    memset(&s->tm_group, 0, sizeof(GroupMaps));
    memset(&s->tm_k, 0, sizeof(CUtensorMap));
    memset(&s->tm_v, 0, sizeof(CUtensorMap));
  }
  return CB200_OK;
}

template <typename T, int D, bool GATHER, int MODE>
int launch_decode(const DecodeSetup& s, cudaStream_t stream) {
  auto kern = decode_attn_kernel<T, D, GATHER, MODE>;
  static int configured_smem[16] = {0};  // per device
  int dev = 0;
  CB200_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 16 && configured_smem[dev] < s.smem_bytes) {
    CB200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    configured_smem[dev] = 227 * 1024;
  } else if (dev >= 16) {
    CB200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.grid, 1, 1);
  cfg.blockDim = dim3(SmemPlan<D, GATHER, MODE>::kThreads, 1, 1);
  cfg.dynamicSmemBytes = s.smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  // the grid may be scheduled while the preceding kernel of the stream drains; it waits (griddepcontrol.wait)
  // before its first global access
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.overlap ? 1 : 0;
  CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, s.tm_k, s.tm_v, s.tm_group, s.p));
  CB200_CUDA_TRY(cudaGetLastError());
  return CB200_OK;
}

template <int MODE>
int launch_decode_mode(const DecodeSetup& s, const cb200_attn_decode_args* a, cudaStream_t st) {
  const bool f16 = a->dtype == CB200_F16;
  if (a->head_dim == 128) {
    if (s.gather) return f16 ? launch_decode<__half, 128, true, MODE>(s, st) : launch_decode<__nv_bfloat16, 128, true, MODE>(s, st);
    return f16 ? launch_decode<__half, 128, false, MODE>(s, st) : launch_decode<__nv_bfloat16, 128, false, MODE>(s, st);
  }
  if (s.gather) return f16 ? launch_decode<__half, 64, true, MODE>(s, st) : launch_decode<__nv_bfloat16, 64, true, MODE>(s, st);
  return f16 ? launch_decode<__half, 64, false, MODE>(s, st) : launch_decode<__nv_bfloat16, 64, false, MODE>(s, st);
}

}  // namespace
}  // namespace cb200
