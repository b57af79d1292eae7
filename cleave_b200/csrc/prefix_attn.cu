// Decode of a batch whose requests share a long prefix: attention over prefix ++ own tokens, with the prefix's keys
// and values read once for the whole batch instead of once per request.
//
// softmax over a set of keys splits over any partition of it: with (O, m, l) = (sum 2^(x - m) v, max x, sum 2^(x - m))
// of each part, the whole is the sum of the parts' O and l after scaling them to a common maximum. Two kernels:
//   1. prefix_attn_kernel, here: the query rows of all requests that read one kv head (batch * HQ / HKV rows) attend the
//      prefix as ONE problem on the tcgen05 tensor cores. An item is (kv head, block of 128 query rows, part of the
//      prefix's tiles of 128 tokens); the prefix is cut into as many parts as fill the SMs. Each item leaves fp32
//      (O, m, l) in the scratch buffer. P is one 16-bit operand here, in fp16 scaled by 2^7 (weight_headroom), so this
//      kernel sets the error of the result: the two-part P of the second one helps where a request's own tokens weigh most.
//   2. decode_attn_kernel in its suffix mode: the stream over the requests' own tokens; where a row's result is
//      stored, the row's prefix parts are merged in. No third launch, and the requests' own part may be empty.
// The prefix costs max(its bytes / bandwidth, 4 D flop per (query head, token) / tensor rate); up to 128 query rows per kv
// head it is bound by the bytes, beyond that by the tensor cores and the exponentials.
// Measured: 128 requests of 32 query and 8 kv heads of 128 over 32768 tokens 74 us (0.57 of the tensor rate; a tile takes
// 1.15 us of an SM, most of it the latency of scores - softmax - value product), the whole with 1074 own tokens each 188 us.
//
// The structure of the kernel (warp roles, tensor memory layout, lazy rescale) is that of attn_prefill_tc.cu with no mask
// inside a tile but the prefix's end, keys from a page table, and partial results.

#include "decode_attn.cuh"

#include <algorithm>
#include <type_traits>

namespace cb200 {
namespace pre {

constexpr int kBM = 128, kBN = 128;
constexpr int kThreads = 384;        // pages of whole 64-token boxes: TMA
constexpr int kThreadsGather = 512;  // other pages: four more warps copy token rows
constexpr float kRescaleThreshold = 8.f;  // log2 units
constexpr uint32_t kColS = 0, kColO = 256, kColP = 384;  // tensor memory: S0 | S1 | O | P0 | P1

template <int D>
struct Cfg {
  static constexpr int kChunks = D / 64;
  static constexpr int kChunkBytes = 128 * 128;  // 128 rows of 128 bytes
  static constexpr int kTileBytes = kChunks * kChunkBytes;
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kSmemBytes = (1 + 2 * kStages) * kTileBytes + 4096 + 1024;
};

struct Params {
  const int* indices;  // the prefix's pages
  const void* k;
  const void* v;
  float* o;
  float* ml;
  int* status;
  int len, page_size, num_pages, batch, hkv, group, per_block, blocks, splits, n_tiles;
  int item0;  // the first of this launch's items
  float scale_log2;
};

template <typename T, int D, bool GATHER>
__global__ void __launch_bounds__(GATHER ? kThreadsGather : kThreads, 1)
prefix_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using C = Cfg<D>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;
  uint8_t* k_smem = q_smem + C::kTileBytes;
  uint8_t* v_smem = k_smem + kStages * C::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_smem + kStages * C::kTileBytes);
  uint64_t* k_full = bars;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* q_full = v_empty + kStages;
  uint64_t* s_full = q_full + 1;   // [2] S complete in tensor memory
  uint64_t* s_empty = s_full + 2;  // [2] the softmax warps have read S
  uint64_t* p_full = s_empty + 2;  // [2] P stored (and O rescaled if needed)
  uint64_t* p_empty = p_full + 2;  // [2] the PV MMAs that read the P buffer have completed
  uint64_t* o_done = p_empty + 2;
  uint64_t* v_tail = o_done + 1;   // the boxes of the prefix's last, partial V tile have landed
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(v_tail + 1);
  float* mx_exch = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 1024);  // [2 tiles][2 halves][128 rows]
  float* l_exch = mx_exch + 2 * 2 * kBM;                                               // [128 rows]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // row blocks of one part are neighbours: they read the same keys at the same time
  const int item = p.item0 + static_cast<int>(blockIdx.x);
  const int blk = item % p.blocks;
  const int split = item / p.blocks % p.splits;
  const int h = item / (p.blocks * p.splits);
  const int t0 = static_cast<int>(static_cast<long long>(p.n_tiles) * split / p.splits);
  const int nt = static_cast<int>(static_cast<long long>(p.n_tiles) * (split + 1) / p.splits) - t0;  // at least 1

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], GATHER ? 128 : 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], GATHER ? 128 : 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 8);
      mbar_init(&p_full[s], 8);
      mbar_init(&p_empty[s], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(o_done, 1);
    mbar_init(v_tail, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tm_q);
    if (!GATHER) {
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
  pdl_launch_dependents();  // not before the wait: the suffix kernel relies on what precedes this kernel being done

  // The 64-token boxes of tile `t` from tensor map `tm` into `dst`; boxes behind the prefix's end are not fetched.
  // Page ids come from a window of 32 that the lanes of the warp hold.
  int win = -1, ids = 0;
  const int n_pages = ceil_div(p.len, p.page_size);
  auto load_tile = [&](const CUtensorMap* tm, uint8_t* dst, uint64_t* bar, int t) {
    const int boxes = min(2, ceil_div(p.len - t * kBN, 64));
    if (lane == 0) mbar_arrive_expect_tx(bar, boxes * C::kChunks * 64 * 128);
    __syncwarp();
    for (int j = 0; j < boxes; ++j) {
      const int tok = t * kBN + j * 64, pord = tok / p.page_size;
      if ((pord >> 5) != win) {
        win = pord >> 5;
        ids = __ldg(p.indices + min(win * 32 + lane, n_pages - 1));
      }
      const int page = min(max(__shfl_sync(0xffffffffu, ids, pord & 31), 0), p.num_pages - 1);
      if (lane == 0) {
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) tma_load_4d(dst + c * C::kChunkBytes + j * 64 * 128, tm, bar, c * 64, h, tok - pord * p.page_size, page);
      }
    }
  };

  if (warp == 0) {
    // ================================================================ TMA producer: Q, then K tiles
    if (lane == 0) {
      // one box is the 64 columns of the group's heads of `per_block` requests; requests past the batch read as zero
      mbar_arrive_expect_tx(q_full, C::kChunks * p.group * p.per_block * 128);
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) tma_load_3d(q_smem + c * C::kChunkBytes, &tm_q, q_full, c * 64, h * p.group, blk * p.per_block);
    }
    __syncwarp();
    if constexpr (!GATHER) {
      int st = 0, ph = 0;
      for (int j = 0; j < nt; ++j) {
        mbar_wait(&k_empty[st], ph ^ 1, p.status, kFaultEmptyBarrier);
        load_tile(&tm_k, k_smem + st * C::kTileBytes, &k_full[st], t0 + j);
        if (++st == kStages) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 6) {
    // ================================================================ TMA producer: V tiles
    if constexpr (!GATHER) {
      int st = 0, ph = 0;
      for (int j = 0; j < nt; ++j) {
        mbar_wait(&v_empty[st], ph ^ 1, p.status, kFaultEmptyBarrier);
        uint8_t* dst = v_smem + st * C::kTileBytes;
        const int live = p.len - (t0 + j) * kBN;
        if (live >= kBN) {
          load_tile(&tm_v, dst, &v_full[st], t0 + j);
        } else {
          // The rows behind the prefix's end meet P = 0, and 0 * V is 0 only for finite V: they are cleared here,
          // once the boxes have landed, before the tile is handed on.
          load_tile(&tm_v, dst, v_tail, t0 + j);
          mbar_wait(v_tail, 0, p.status, kFaultFullBarrier);
          for (int i = live * 8 + lane; i < kBN * 8; i += 32) {
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c) *reinterpret_cast<uint4*>(dst + c * C::kChunkBytes + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[st]);
        }
        if (++st == kStages) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp >= 12) {
    // ================================================================ row gather (pages that are not whole boxes)
    if constexpr (GATHER) {
      // consecutive lanes copy consecutive 16-byte chunks of a row; rows behind the end are filled with zeros
      const int gtid = tid - 12 * 32;
      constexpr int kChunksPerRow = D / 8;
      constexpr int kRowsPerRound = 128 / kChunksPerRow;
      constexpr int kRounds = kBN / kRowsPerRound;
      const int c = gtid % kChunksPerRow, r_in = gtid / kChunksPerRow;
      const T* kc = reinterpret_cast<const T*>(p.k);
      const T* vc = reinterpret_cast<const T*>(p.v);
      auto load_pages = [&](int t, int (&pg)[kRounds]) {
#pragma unroll
        for (int r = 0; r < kRounds; ++r) pg[r] = __ldg(p.indices + min(t * kBN + r * kRowsPerRound + r_in, p.len - 1) / p.page_size);
      };
      int pg[kRounds];
      load_pages(t0, pg);
      int st = 0, ph = 0;
      for (int j = 0; j < nt; ++j) {
        long long src[kRounds];
        uint32_t live = 0;
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
          const int tok = (t0 + j) * kBN + r * kRowsPerRound + r_in;
          const int at = min(tok, p.len - 1);
          const long long page = min(max(pg[r], 0), p.num_pages - 1);
          src[r] = ((page * p.page_size + at % p.page_size) * p.hkv + h) * D + c * 8;
          live |= (tok < p.len ? 1u : 0u) << r;
        }
        if (j + 1 < nt) load_pages(t0 + j + 1, pg);
        const uint32_t kdst = smem_u32(k_smem + st * C::kTileBytes), vdst = smem_u32(v_smem + st * C::kTileBytes);
        auto copy = [&](const T* from, uint32_t to) {
#pragma unroll
          for (int r = 0; r < kRounds; ++r) {
            const int row = r * kRowsPerRound + r_in;
            const uint32_t o = (c >> 3) * C::kChunkBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + o), "l"(from + src[r]), "r"((live >> r & 1u) * 16u) : "memory");
          }
        };
        mbar_wait(&k_empty[st], ph ^ 1, p.status, kFaultEmptyBarrier);
        copy(kc, kdst);
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&k_full[st])) : "memory");
        mbar_wait(&v_empty[st], ph ^ 1, p.status, kFaultEmptyBarrier);
        copy(vc, vdst);
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&v_full[st])) : "memory");
        if (++st == kStages) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ================================================================ MMA issuer
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t idesc_s = umma_idesc(kBf16, /*b_mn_major=*/false, kBM, kBN);
    constexpr uint32_t idesc_pv = umma_idesc(kBf16, /*b_mn_major=*/true, kBM, D);
    const uint32_t q_addr = smem_u32(q_smem), k_addr = smem_u32(k_smem), v_addr = smem_u32(v_smem);
    int kst = 0, kph = 0, vst = 0, vph = 0;
    auto issue_s = [&](int j) {
      const int sb = j & 1;
      mbar_wait(&k_full[kst], kph, p.status, kFaultFullBarrier);
      if constexpr (GATHER) fence_proxy_async_smem();
      mbar_wait(&s_empty[sb], ((j >> 1) & 1) ^ 1, p.status, kFaultTmemBarrier);
      tc_fence_after();
      if (elect_one()) {
        const uint32_t d = tmem_base + kColS + sb * kBN;
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint64_t adesc = umma_smem_desc(q_addr + c * C::kChunkBytes + kk * 32, 16, 8 * 128);
            const uint64_t bdesc = umma_smem_desc(k_addr + kst * C::kTileBytes + c * C::kChunkBytes + kk * 32, 16, 8 * 128);
            umma_f16(d, adesc, bdesc, idesc_s, (c > 0 || kk > 0) ? 1u : 0u);
          }
        }
        umma_commit(&k_empty[kst]);
        umma_commit(&s_full[sb]);
      }
      __syncwarp();
      if (++kst == kStages) { kst = 0; kph ^= 1; }
    };
    mbar_wait(q_full, 0, p.status, kFaultFullBarrier);
    issue_s(0);
    for (int j = 0; j < nt; ++j) {
      if (j + 1 < nt) issue_s(j + 1);  // the tensor pipe works on the next scores beside the softmax of these
      const int pb = j & 1;
      mbar_wait(&v_full[vst], vph, p.status, kFaultFullBarrier);
      if constexpr (GATHER) fence_proxy_async_smem();
      mbar_wait(&p_full[pb], (j >> 1) & 1, p.status, kFaultTmemBarrier);
      tc_fence_after();
      if (elect_one()) {
        const uint32_t va = v_addr + vst * C::kTileBytes;
#pragma unroll
        for (int ks = 0; ks < kBN / 16; ++ks) {
          const uint64_t bdesc = umma_smem_desc(va + ks * 16 * 128, C::kChunkBytes, 8 * 128);
          umma_f16_ts(tmem_base + kColO, tmem_base + kColP + pb * 64 + ks * 8, bdesc, idesc_pv, (j > 0 || ks > 0) ? 1u : 0u);
        }
        umma_commit(&v_empty[vst]);
        umma_commit(&p_empty[pb]);
        if (j == nt - 1) umma_commit(o_done);
      }
      __syncwarp();
      if (++vst == kStages) { vst = 0; vph ^= 1; }
    }
  } else if (warp != 7) {
    // ================================================================ softmax / epilogue (warps 2..5 and 8..11)
    const int quarter = warp & 3;
    const int half = warp >= 8 ? 1 : 0;   // which 64 of a tile's 128 scores this thread takes
    const int row = quarter * 32 + lane;  // query row of the block = tensor memory lane
    const uint32_t lane_field = static_cast<uint32_t>(quarter * 32) << 16;
    const int pair_bar = 1 + quarter;     // named barrier of the two warps that share the rows
    constexpr float kHeadroom = weight_headroom<T>(kRescaleThreshold);  // P is at most 2^8
    float m_ref = -INFINITY, l_run = 0.f;  // m_ref is -inf until a score is not
    for (int j = 0; j < nt; ++j) {
      const int sb = j & 1, pb = j & 1;
      const int live = p.len - (t0 + j) * kBN - half * 64;  // scores of this thread's half that belong to the prefix
      mbar_wait(&s_full[sb], (j >> 1) & 1, p.status, kFaultMmaBarrier);
      tc_fence_after();
      uint32_t r[2][32];
#pragma unroll
      for (int q = 0; q < 2; ++q) tmem_ld_32x32(tmem_base + lane_field + kColS + sb * kBN + half * 64 + q * 32, r[q]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[sb]);
      float mx = -INFINITY;
      if (live >= 64) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float v = __uint_as_float(r[q][i]) * p.scale_log2;
            r[q][i] = __float_as_uint(v);
            mx = fmaxf(mx, v);
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float v = q * 32 + i < live ? __uint_as_float(r[q][i]) * p.scale_log2 : -INFINITY;
            r[q][i] = __float_as_uint(v);
            mx = fmaxf(mx, v);
          }
        }
      }
      mx_exch[(sb * 2 + half) * kBM + row] = mx;
      named_bar_sync(pair_bar, 64);
      mx = fmaxf(mx, mx_exch[(sb * 2 + (half ^ 1)) * kBM + row]);
      float alpha = 1.f;
      bool rescale = false;
      if (mx > m_ref + kRescaleThreshold) {
        alpha = fast_exp2(m_ref - mx);
        m_ref = mx;
        rescale = j > 0;  // the first tile's product overwrites O
      }
      mbar_wait(&p_empty[pb], ((j >> 1) & 1) ^ 1, p.status, kFaultMmaBarrier);
      if (__any_sync(0xffffffffu, rescale)) {  // rare: the maximum grew by more than 2^8
        mbar_wait(&p_empty[pb ^ 1], ((j - 1) >> 1) & 1, p.status, kFaultMmaBarrier);
        tc_fence_after();
#pragma unroll 1
        for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 32) {
          uint32_t o[32];
          tmem_ld_32x32(tmem_base + lane_field + kColO + c0, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = alpha == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32(tmem_base + lane_field + kColO + c0, o);
        }
        tmem_st_wait();
      }
      tc_fence_after();
      float psum = 0.f;
      const float shift = m_ref == -INFINITY ? 0.f : m_ref - kHeadroom;
      {
        uint32_t pk[32];  // P in the storage type, as the operand of a 16-bit product must be; its sum is that of the fp32 values
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int c = 2 * i;
          const float p0 = fast_exp2(__uint_as_float(r[c >> 5][c & 31]) - shift);
          const float p1 = fast_exp2(__uint_as_float(r[(c + 1) >> 5][(c + 1) & 31]) - shift);
          psum += p0 + p1;
          pk[i] = pack2<T>(p0, p1);
        }
        tmem_st_32x32(tmem_base + lane_field + kColP + pb * 64 + half * 32, pk);
      }
      l_run = l_run * alpha + psum;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[pb]);
    }
    // ---- the item's partial: O as it stands, the reference maximum and the row sum of both halves
    if (half) l_exch[row] = l_run;
    named_bar_sync(pair_bar, 64);
    mbar_wait(o_done, 0, p.status, kFaultMmaBarrier);
    tc_fence_after();
    const int bi = row / p.group;
    const bool live_row = bi < p.per_block && blk * p.per_block + bi < p.batch;
    const size_t part = (static_cast<size_t>(h) * p.blocks + blk) * p.splits + split;
    float* dst = p.o + (part * kBM + row) * D;
#pragma unroll 1
    for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 32) {
      uint32_t o[32];
      tmem_ld_32x32(tmem_base + lane_field + kColO + c0, o);
      tmem_ld_wait();
      if (live_row) {
#pragma unroll
        for (int i = 0; i < 32; i += 8)  // whole sectors: neighbouring lanes write rows that are far apart
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + c0 + i), "r"(o[i]), "r"(o[i + 1]), "r"(o[i + 2]),
                       "r"(o[i + 3]), "r"(o[i + 4]), "r"(o[i + 5]), "r"(o[i + 6]), "r"(o[i + 7]) : "memory");
      }
    }
    if (!half && live_row) {
      p.ml[part * 256 + row] = m_ref - kHeadroom;
      p.ml[part * 256 + kBM + row] = l_run + l_exch[row];
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------------- host side
struct Plan {
  int group, per_block, blocks, splits, n_tiles;
  size_t o_bytes, ml_bytes;
};

int plan_prefix(const cb200_attn_decode_args* a, int prefix_len, Plan* pl) {
  pl->group = a->num_qo_heads / a->num_kv_heads;
  if (pl->group > kBM) return CB200_ERR_UNSUPPORTED;
  pl->per_block = std::min(kBM / pl->group, a->batch);
  pl->blocks = ceil_div(a->batch, pl->per_block);
  pl->n_tiles = static_cast<int>((static_cast<long long>(prefix_len) + kBN - 1) / kBN);
  const long long base = static_cast<long long>(a->num_kv_heads) * pl->blocks;
  int sms = sm_count();
  if (sms <= 0) return CB200_ERR_CUDA;
  if (bounded(a)) sms = a->max_ctas;
  // Parts per (kv head, row block): the fewest rounds of tiles over the SMs, in units of a tile (about 1.2 us). A CTA
  // costs about three tiles beside its tiles (launch, first loads, the partial); every part adds one fp32 copy of
  // the rows that is written and read again, and every eight parts a round trip to L2 for each (request, kv head) of the
  // second kernel, of which a CTA has its share one after the other.
  const double merge = 2.0 * a->batch * a->num_qo_heads * a->head_dim * 4 / 6e6 / 1.2;
  const double trip = 0.95 * a->batch * a->num_kv_heads / sms;
  double best = 0;
  pl->splits = 1;
  for (int s = 1; s <= pl->n_tiles && s <= 256; ++s) {
    const double cost = static_cast<double>((base * s + sms - 1) / sms) * (ceil_div(pl->n_tiles, s) + 3) + merge * s + trip * ceil_div(s, 8);
    if (s == 1 || cost < best) {
      best = cost;
      pl->splits = s;
    }
  }
  if (base * pl->splits >= (1LL << 31)) return CB200_ERR_UNSUPPORTED;
  const size_t parts = static_cast<size_t>(base) * pl->splits;
  pl->o_bytes = parts * kBM * a->head_dim * sizeof(float);
  pl->ml_bytes = parts * 2 * kBM * sizeof(float);
  return CB200_OK;
}

template <typename T, int D, bool GATHER>
int launch_prefix(const cb200_attn_decode_args* a, Params p, cudaStream_t stream) {
  const CUtensorMapDataType dt = a->dtype == CB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  CUtensorMap tm_q, tm_k, tm_v;
  memset(&tm_k, 0, sizeof(tm_k));
  memset(&tm_v, 0, sizeof(tm_v));
  const uint64_t row = static_cast<uint64_t>(D) * 2;
  {
    const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a->num_qo_heads), static_cast<uint64_t>(a->batch)};
    const uint64_t strides[2] = {row, row * a->num_qo_heads};
    const uint32_t box[3] = {64u, static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.per_block)};
    if (!encode_tensor_map(&tm_q, dt, 3, const_cast<void*>(a->q), dims, strides, box, sw)) return CB200_ERR_CUDA;
  }
  if (!GATHER) {
    const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.hkv), static_cast<uint64_t>(p.page_size),
                              static_cast<uint64_t>(p.num_pages)};
    const uint64_t strides[3] = {row, row * p.hkv, row * p.hkv * p.page_size};
    const uint32_t box[4] = {64u, 1u, 64u, 1u};
    if (!encode_tensor_map(&tm_k, dt, 4, const_cast<void*>(a->k_cache), dims, strides, box, sw) ||
        !encode_tensor_map(&tm_v, dt, 4, const_cast<void*>(a->v_cache), dims, strides, box, sw))
      return CB200_ERR_CUDA;
  }
  auto kern = prefix_attn_kernel<T, D, GATHER>;
  CB200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmemBytes));
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(GATHER ? kThreadsGather : kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg<D>::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // One launch, or as many as keep each of them to the caller's bound; those behind the first wait for the one before
  const int items = p.hkv * p.blocks * p.splits, most = bounded(a) ? std::min(items, a->max_ctas) : items;
  for (p.item0 = 0; p.item0 < items; p.item0 += most) {
    cfg.gridDim = dim3(static_cast<unsigned>(std::min(most, items - p.item0)), 1, 1);
    CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm_q, tm_k, tm_v, p));
    cfg.numAttrs = 0;
  }
  CB200_CUDA_TRY(cudaGetLastError());
  return CB200_OK;
}

template <typename T, int D>
int launch_prefix_any(const cb200_attn_decode_args* a, const Params& p, bool gather, cudaStream_t st) {
  return gather ? launch_prefix<T, D, true>(a, p, st) : launch_prefix<T, D, false>(a, p, st);
}

}  // namespace pre
}  // namespace cb200

extern "C" size_t cb200_attn_decode_shared_prefix_scratch_bytes(const cb200_attn_decode_args* a, int prefix_len) {
  using namespace cb200;
  DecodeSetup s;
  pre::Plan pl;
  if (prefix_len <= 0 || plan_decode(a, &s, false) != CB200_OK || pre::plan_prefix(a, prefix_len, &pl) != CB200_OK) return 0;
  return pl.o_bytes + pl.ml_bytes;
}

extern "C" int cb200_attn_decode_shared_prefix(const cb200_attn_decode_args* a, const int32_t* prefix_indices, int num_prefix_indices,
                                               int prefix_len, void* scratch, size_t scratch_bytes, void* stream) {
  using namespace cb200;
  if (!a || !a->kv_indptr || prefix_len < 0 || num_prefix_indices < 0) return CB200_ERR_BAD_ARG;
  if (a->q_rows > 1) return CB200_ERR_UNSUPPORTED;
  DecodeSetup s;
  const int rc = plan_decode(a, &s, true, true);
  if (rc != CB200_OK) return rc;
  if (static_cast<long long>(num_prefix_indices) * a->page_size < prefix_len) return CB200_ERR_BAD_ARG;
  if (prefix_len > (1 << 30)) return CB200_ERR_UNSUPPORTED;  // token indices are rounded up to tiles in 32 bits
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  s.p.pre_splits = 0;
  s.p.pre_blocks = s.p.pre_batch = 1;
  if (prefix_len > 0) {
    if (!prefix_indices) return CB200_ERR_BAD_ARG;
    pre::Plan pl;
    const int prc = pre::plan_prefix(a, prefix_len, &pl);
    if (prc != CB200_OK) return prc;
    if (!scratch || scratch_bytes < pl.o_bytes + pl.ml_bytes) return CB200_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(scratch) & 31) return CB200_ERR_ALIGNMENT;
    pre::Params p{};
    p.indices = prefix_indices;
    p.k = a->k_cache;
    p.v = a->v_cache;
    p.o = static_cast<float*>(scratch);
    p.ml = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + pl.o_bytes);
    p.status = s.p.status;
    p.len = prefix_len;
    p.page_size = a->page_size;
    p.num_pages = a->num_pages;
    p.batch = a->batch;
    p.hkv = a->num_kv_heads;
    p.group = pl.group;
    p.per_block = pl.per_block;
    p.blocks = pl.blocks;
    p.splits = pl.splits;
    p.n_tiles = pl.n_tiles;
    p.scale_log2 = s.p.scale_log2;
    const bool f16 = a->dtype == CB200_F16;
    const int done = a->head_dim == 64 ? (f16 ? pre::launch_prefix_any<__half, 64>(a, p, s.gather, st) : pre::launch_prefix_any<__nv_bfloat16, 64>(a, p, s.gather, st))
                                       : (f16 ? pre::launch_prefix_any<__half, 128>(a, p, s.gather, st) : pre::launch_prefix_any<__nv_bfloat16, 128>(a, p, s.gather, st));
    if (done != CB200_OK) return done;
    s.p.pre_o = p.o;
    s.p.pre_ml = p.ml;
    s.p.pre_splits = pl.splits;
    s.p.pre_blocks = pl.blocks;
    s.p.pre_batch = pl.per_block;
    s.overlap = !bounded(a);
  }
  return launch_decode_mode<kSuffix>(s, a, st);
}
