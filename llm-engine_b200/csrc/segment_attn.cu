// Attention without a causal mask over paged K/V (include/pkv.h, "attention to an encoder's states" and "shared
// prefix"): the tile kernel on the 5th-generation tensor cores, the merge kernel, and the entry points.  How a step is
// cut into work for them and for the decode kernels is in segment_plan.hpp.
//
//   out[t][h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp(scale q[t][h] . K[j] - m),   m = the row's maximum
//
// A tile item is up to 256 rows (token, query head of one kv head's group) that all see the same keys, walked in tiles of
// 128.  The rows are two groups of 128, each with its own scores S (128 columns of tensor memory) and output O (head_dim
// columns); a K or V tile is fetched once for both.  While one group's scores are turned into probabilities, the tensor
// cores work on the other group: a 128 x 128 x 128 product takes 512 cycles, the 16,384 exponentials of a group's tile 1,024.
//
//   warps 0-7, 8-15 softmax of group 0, 1: a row is two threads, of 64 keys each, which exchange their maxima through shared
//                   memory.  (One thread a row, eight warps in all, left the exponential unit half idle: 3,850 cycles for a
//                   tile of both groups at head_dim 128, 3,300 at 64.)  P goes back to tensor memory as 16-bit pairs, the A
//                   operand of the second product.  O stays there and is rescaled only when a row's maximum has grown by
//                   more than 2^8.
//   warps 16, 19    TMA: K, V tiles through the block table into one ring (boxes of up to 128 slots x 128 bytes).  Two, because a warp
//                   sends a 16-slot box every 170 cycles, half as fast as two heads of 64 dims eat them.
//   warp 17         issues the products, one thread: S = Q K^T and O += P V of both groups in turns.
//   warp 18         TMA: the next item's rows of Q, a box for each token's heads, or for several consecutive tokens'.
//
// head_dim 64: P has 64 columns of its own.  The next scores of a group are issued as soon as its threads hold the present ones
// in registers, so the softmax warps never wait for a product: the exponentials decide.
// head_dim 128: S and O fill the group's half of tensor memory, P lies over the first half of S, and the next scores follow
// the second product.
//
// An item of at most 128 rows brings those of two kv heads, one for each group, whose K and V tiles alternate in the ring.
// P is rounded to 16 bits for the second product (the sums are of the unrounded ones), as the operands of the
// tensor cores are; scores, sums and accumulators are fp32.
//
// Measured on B200: a key tile of both groups takes about 3,500 cycles at head_dim 128 (products 2,048, exponentials 2,048, the rest a
// group's chain of load, maximum, exponentials, store that one other group does not cover) and 3,200 at 64 (products 1,024; the issuing
// warp's waits); an item's start and end 5,000.  4 sequences of 1,000 - 2,048 tokens and 4,000 - 6,500 keys, 32/8 heads of 128 dims: 593 us,
// 1,155 TFLOP/s, in a burst (688, 995, over seconds, under the power cap).  24 of 3 - 448 tokens and 100 - 1,500 keys, 16/16 heads of 64: 50 us.
//
// Blocks are persistent, one on an SM, each with a list of items of its own.  Every wait is bounded: one that runs
// out sets bit 32 of the error word and the block winds down.
#include <algorithm>
#include <cstdlib>
#include <new>
#include <type_traits>
#include <vector>

#include "common.cuh"
#include "decode_list.hpp"
#include "launch_util.hpp"
#include "segment_plan.hpp"
#include "status.hpp"
#include "tcgen05.cuh"
#include "tma_util.hpp"

namespace pkv {

__device__ unsigned int g_pkv_tile_error = 0;
constexpr unsigned kErrTileWait = 32u, kErrOtherPlan = 64u;   // kErrOtherPlan: as in decode_attn.cuh

unsigned int* error_mirror(bool create);                 // error_mirror.cu
int check_error_mirror(const char* fn, unsigned int bits = ~0u);

namespace {

constexpr int kTileThreads = 640;
// Registers a thread of the softmax warps and of the others; launched with 96 each (4 x 104 + 64 <= 5 x 96).
constexpr int kSoftmaxRegs = 104, kOtherRegs = 64;
constexpr int kProducer = 16, kIssuer = 17, kRowsLoader = 18, kProducerV = 19;
constexpr int kBlockBytes = 128 * 128;                   // 128 rows x 64 16-bit elements: one operand block
constexpr uint32_t kGroupCols = 256, kColO = 128;        // tensor memory of a group: S, then O ...
constexpr float kRescale = 8.f;                          // in log2 units: P stays below 2^8
// A blocking poll takes 2 us.  Waits for a tile: 0.27 s; waits that may span whole items, or a block's list of them (kMostListCycles): 2.1 s.
constexpr uint32_t kItemPolls = 1u << 20;
constexpr int kBoxRows = 64;                             // rows of Q, at most, that a box of several tokens brings
constexpr int kMinTileTokens = 2, kManyTileTokens = 32;  // sequences with fewer tokens always go to the decode kernels, with as many never

template <int D> struct TileSmem {
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * kBlockBytes;    // a K or V tile, or one group's Q
  static constexpr int kStages = D == 64 ? 8 : 4;
  static constexpr uint32_t kColP = D == 64 ? 192 : 0;   // ... and P behind O, or over S
  static constexpr int kLead = D == 64 ? 2 : 1;          // key tiles a group's scores are issued ahead of its values
  // Q: half (64 dims) by half, 256 rows each; the next item's beside the present one's where there is room
  static constexpr int kQ = 2 * kTile, kQBufs = D == 64 ? 2 : 1, kQHalf = 2 * kBlockBytes;
  static constexpr int kRing = kQBufs * kQ;
  static constexpr int kBytes = kRing + kStages * kTile + 1024;
};

struct TileArgs {
  const int *block_tables, *table_offset, *token_seq;
  const int *row_token, *list_first;
  const TileItem* tiles;
  const PlanHeader* header;          // shows `stamp`, or this launch is not for the plan that the workspace holds
  int stamp;
  void* out;
  float *part_ml, *part_acc;         // by partial row
  int q_heads, group;
  int block_size, bs_log2, box_log2; // a TMA box is 1 << box_log2 slots
  int box_tokens;                    // tokens of a box of the second Q map (the first: one)
  float scale;
  float ml_scale;                    // what partial maxima are multiplied with: scale, or scale log2 e
  unsigned int* host_err;
};

__device__ __forceinline__ void report(unsigned int* host_err, unsigned int bit) {
  atomicOr(&g_pkv_tile_error, bit);
  if (host_err) {
    *reinterpret_cast<volatile unsigned int*>(host_err) = bit;
    __threadfence_system();
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 ra, rb, rc, rd;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %5};\n mov.b64 rc, {%6, %7};\n"
      " fma.rn.f32x2 rd, ra, rb, rc;\n mov.b64 {%0, %1}, rd;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 ra, rb, rd;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %5};\n add.rn.f32x2 rd, ra, rb;\n mov.b64 {%0, %1}, rd;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// N 16-byte pieces a lane: piece i of lane j of every N lanes becomes piece j of lane i.
template <int N>
__device__ __forceinline__ void transpose(uint32_t (&x)[4 * N], int lane) {
#pragma unroll
  for (int s = 1; s < N; s <<= 1) {
    const bool upper = (lane & s) != 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i & s) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t& a = x[4 * i + k];
        uint32_t& b = x[4 * (i | s) + k];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? a : b, s);
        a = upper ? got : a;
        b = upper ? b : got;
      }
    }
  }
}

__device__ __forceinline__ TileItem load_tile(const TileItem* p) {
  const int4 a = __ldg(reinterpret_cast<const int4*>(p)), b = __ldg(reinterpret_cast<const int4*>(p) + 1);
  return TileItem{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    tile_attn_kernel(const TileArgs a, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap qmap_many,
                     const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using S = TileSmem<D>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kInstrQK = tc::instruction(kBf16, kTileKeys, false), kInstrPV = tc::instruction(kBf16, D, true);
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int NS = S::kStages;

  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long bars[2 * NS + 12];
  __shared__ float sm_max[2][2][2][128], sm_sum[2][2][128];   // [tile parity][group][half][row]; [group][half][row]
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t ring = base + S::kRing, bar0 = smem_u32(&bars[0]);
  enum { KV_FULL = 0, KV_EMPTY = NS, Q_FULL = 2 * NS, Q_EMPTY = Q_FULL + 2, S_FULL = Q_EMPTY + 2, S_READ = S_FULL + 2, P_FULL = S_READ + 2, O_FULL = P_FULL + 2 };
  auto BAR = [&](int i) { return bar0 + 8u * i; };

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(BAR(KV_FULL + i), 1);
      mbar_init(BAR(KV_EMPTY + i), 1);  // commit after the last product that reads the stage
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(BAR(Q_FULL + g), 1);    // (of a buffer, not of a group)
      mbar_init(BAR(Q_EMPTY + g), 1);   // commit after the item's last Q K^T
      mbar_init(BAR(S_FULL + g), 1);    // commit after the group's Q K^T
      mbar_init(BAR(S_READ + g), 256);  // kLead 2: the group's softmax threads (32 at a time) hold S in registers
      mbar_init(BAR(P_FULL + g), 256);  // they have written P
      mbar_init(BAR(O_FULL + g), 1);    // commit after the group's P V: kLead 2 each, kLead 1 the item's last
    }
    mbar_fence_init();
  }
  if (warp == kIssuer) tc::alloc<512>(smem_u32(&tmem_slot));
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_slot;

  // The plan and the index arrays were complete before the launch ahead of this one began, so the look-ups that lead to the
  // first loads run while it is finishing; what it may have written (K, V, q, the partials' space) is touched only behind the wait.
  // The launch behind this one may be the decode kernel of the same call, which does not wait for this one before
  // it reads (decode_list.hpp): it may start once everything before this launch is complete.
  auto after_previous = [] {
    pdl_wait();
    pdl_launch_dependents();
  };

  const TileItem* tiles = a.tiles + __ldg(a.list_first + blockIdx.x);
  // (no list is empty: 0 stands for another plan's image)
  const int n_items = __ldg(&a.header->stamp) == a.stamp ? __ldg(a.list_first + blockIdx.x + 1) - __ldg(a.list_first + blockIdx.x) : 0;

  bool dead = false;
  auto WAIT = [&](uint32_t bar, uint32_t parity, uint32_t polls = 1u << 17) {
    if (!dead) dead = !mbar_wait(bar, parity, polls);
  };
  // Without the first look, for waits that are waits nearly always: it only takes the others' cycles and power.
  auto BLOCK = [&](uint32_t bar, uint32_t parity, uint32_t polls = 1u << 17) {
    if (dead) return;
    bool there = false;
    for (uint32_t i = 0; i < polls && !there; ++i) there = mbar_try_wait(bar, parity);
    dead = !there;
  };

  if (warp >= kProducer) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
    if (warp == kProducer || warp == kProducerV) {
      // The entries of the ring for an item of n key tiles, in the order the products use them: K of the first `lead` tiles,
      // then V0 K(lead) V1 K(lead + 1) ..., and the last V.
      const bool for_v = warp == kProducerV;
      const CUtensorMap* map = for_v ? &vmap : &kmap;
      uint32_t e = 0, mine = 0, parity = 0;                        // ring entries; stages this warp filled last, and in which phase
      bool first = true;
      if (lane == 0) asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
      const int box_rows = 1 << a.box_log2, boxes = kTileKeys >> a.box_log2, per_batch_log2 = 5 - (7 - a.box_log2);   // key tiles of a batch
      for (int r = 0; r < n_items && !dead; ++r) {
        const TileItem it = load_tile(tiles + r);
        const int pair = it.flags & kPair ? 1 : 0, n = (it.kv_len + kTileKeys - 1) / kTileKeys << pair, end = it.kv_begin + it.kv_len;
        const int* tbl = a.block_tables + __ldg(a.table_offset + (it.source < 0 ? ~it.source : __ldg(a.token_seq + it.source)));
        const int lead = min(n, S::kLead << pair), turns = 2 * (n - lead);
        auto is_v = [&](int i) { return i >= lead && !(i - lead < turns && ((i - lead) & 1)); };
        auto tile_of = [&](int i) { return i < lead ? i : i - lead >= turns ? i - n : ((i - lead) & 1) ? lead + ((i - lead) >> 1) : (i - lead) >> 1; };
        // Pool rows of the item's boxes, a batch of 32 at a time, a lane each: the look-up through the block table takes longer
        // than a tile, and its batches are asked for one ahead.
        auto batch = [&](int b) {
          const int pos = it.kv_begin + ((b * 32 + lane) << a.box_log2);
          if (pos >= end) return 0;
          return (__ldg(tbl + (pos >> a.bs_log2)) << a.bs_log2) + (pos & (a.block_size - 1));
        };
        int at = 0, here = batch(0), ahead = batch(1);
        auto row_of = [&](int kt) {          // pool row of this lane's box of a key tile
          const int b = kt >> per_batch_log2;
          if (b > at) {
            here = ahead;
            ahead = batch(++at + 1);
          }
          return __shfl_sync(0xffffffffu, here, ((kt << (5 - per_batch_log2)) + (lane & (boxes - 1))) & 31);
        };
        if (first) after_previous();
        first = false;
        for (int i = 0; i < 2 * n; ++i, ++e) {
          const int st = static_cast<int>(e % NS);
          if (is_v(i) != for_v) {
            mine &= ~(1u << st);
            continue;
          }
          const int t = tile_of(i), y = row_of(t >> pair), left = it.kv_len - (t >> pair) * kTileKeys;
          const int x = (it.kvh + (t & pair)) * D;
          const int valid = min(boxes, (left + box_rows - 1) >> a.box_log2);
          if (lane == 0) {
            WAIT(BAR(KV_EMPTY + st), ((e / NS) & 1) ^ 1);
            if (!dead) mbar_arrive_expect_tx(BAR(KV_FULL + st), static_cast<uint32_t>(valid * box_rows) * 128u * S::kHalves);
          }
          dead = __shfl_sync(0xffffffffu, dead ? 1 : 0, 0) != 0;
          if (dead) break;
          mine |= 1u << st;
          parity = (parity & ~(1u << st)) | ((e / NS) & 1) << st;
          if (lane < valid) {
            const uint32_t dst = ring + st * S::kTile + (lane << a.box_log2) * 128;
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h) tma_load_2d(dst + h * kBlockBytes, map, x + h * 64, y, BAR(KV_FULL + st));
          }
          __syncwarp();
        }
      }
      // whatever this warp has sent for has arrived before the block leaves
      if (lane == 0) {
        for (int st = 0; st < NS; ++st)
          if (mine >> st & 1) mbar_wait(BAR(KV_FULL + st), parity >> st & 1);
      }
      __syncwarp();
    } else if (warp == kRowsLoader) {
      int r = 0;
      if (lane == 0) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&qmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&qmap_many) : "memory");
      }
      for (; r < n_items && !dead; ++r) {
        const TileItem it = load_tile(tiles + r);
        const int heads = it.flags & kPair ? 2 : 1, qb = r % S::kQBufs;
        const uint32_t bar = BAR(Q_FULL + qb), dst = base + qb * S::kQ;
        // A lane a box: boxes of several tokens where the tokens are consecutive, the last one with rows past the item's that
        // nobody looks at if there is room for them, else boxes of one.
        const int up = (it.n_tok + a.box_tokens - 1) / a.box_tokens;
        const int many = !(it.flags & kConsecutive) ? 0 : up * a.box_tokens * a.group <= 256 / heads ? up : it.n_tok / a.box_tokens;
        const int boxes = many + max(it.n_tok - many * a.box_tokens, 0);
        int token = 0;
        auto first_of = [&](int b) { return b < many ? b * a.box_tokens : b + many * (a.box_tokens - 1); };   // first token of a box
        if (lane < boxes) token = __ldg(a.row_token + it.tok0 + first_of(lane));
        if (r == 0) after_previous();
        if (lane == 0) {
          WAIT(BAR(Q_EMPTY + qb), ((r / S::kQBufs) & 1) ^ 1, kItemPolls);
          if (!dead) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(heads * (many * a.box_tokens + boxes - many) * a.group) * 128u * S::kHalves);
        }
        dead = __shfl_sync(0xffffffffu, dead ? 1 : 0, 0) != 0;
        if (dead) break;
        for (int b = lane; b < boxes; b += 32) {
          if (b >= 32) token = __ldg(a.row_token + it.tok0 + first_of(b));
          const uint32_t to = dst + first_of(b) * a.group * 128;
          for (int i = 0; i < heads; ++i)
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
              tma_load_3d(to + i * kBlockBytes + h * S::kQHalf, b < many ? &qmap_many : &qmap, h * 64, (it.kvh + i) * a.group, token, bar);
        }
        __syncwarp();
      }
      if (lane == 0) {
        for (int i = max(r - S::kQBufs, 0); i < r; ++i) mbar_wait(BAR(Q_FULL + i % S::kQBufs), (i / S::kQBufs) & 1);
      }
      __syncwarp();
    } else if (warp == kIssuer) {
      after_previous();
      const uint32_t one = lane == 0 ? 1u : 0u;
      uint32_t e = 0, done = 0, read = 0;                        // ring entries; bit g: parity of group g's P and S taken
      for (int r = 0; r < n_items && !dead; ++r) {
        const TileItem it = load_tile(tiles + r);
        const int pair = it.flags & kPair ? 1 : 0, n = (it.kv_len + kTileKeys - 1) / kTileKeys << pair;
        const int last = it.n_tok * a.group > 128 ? 1 : 0, qb = r % S::kQBufs;   // last group, if both take every tile; buffer of Q
        // waits for the ring entry and returns where it lies
        auto full = [&](uint32_t entry) {
          WAIT(BAR(KV_FULL + entry % NS), (entry / NS) & 1);
          tc::fence_after();
          return ring + (entry % NS) * S::kTile;
        };
        // Descriptors differ in their low word only.  It is made opaque at every call: the compiler would otherwise keep two
        // dozen of them per group at hand, spilled, and a product waited 200 cycles for its own.
        auto scores = [&](int g, uint32_t k_addr, bool read_first) {
          if (S::kLead > 1) {
            if (read_first) {
              WAIT(BAR(S_READ + g), (read >> g) & 1);
              tc::fence_after();
            }
            // counted by tiles: the phase of an item's last tile, which nobody waits for, is over when its P is there
            if (read_first) read ^= 1u << g;
          }
          uint32_t q_lo = (base + qb * S::kQ + g * kBlockBytes) >> 4, k_lo = k_addr >> 4;
          const uint32_t d = tmem + g * kGroupCols;
          asm volatile("" : "+r"(q_lo), "+r"(k_lo));
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            tc::mma_ss(d, tc::operand_at(q_lo + (ks >> 2) * (S::kQHalf >> 4) + (ks & 3) * 2),
                       tc::operand_at(k_lo + (ks >> 2) * (kBlockBytes >> 4) + (ks & 3) * 2), kInstrQK, ks > 0, one);
          }
          tc::commit(BAR(S_FULL + g), one);
        };
        // Products of one thread run in order: where P lies over S, the group's next scores overwrite it behind these.
        auto values = [&](int g, uint32_t v_addr, bool first, bool final) {
          // (a look first: 242 us against 247 for full tiles at 64 dims; at 128, the largest case over seconds, 691 against 688, and
          // 695 where the softmax threads look first too)
          if constexpr (D == 64) WAIT(BAR(P_FULL + g), (done >> g) & 1);
          else BLOCK(BAR(P_FULL + g), (done >> g) & 1);
          tc::fence_after();
          uint32_t v_lo = v_addr >> 4, t = tmem + g * kGroupCols;
          asm volatile("" : "+r"(v_lo), "+r"(t));
#pragma unroll
          for (int kk = 0; kk < kTileKeys / 16; ++kk)
            tc::mma_ts(t + kColO, t + S::kColP + kk * 8, tc::operand_at(v_lo + kk * (2048 >> 4), kBlockBytes), kInstrPV, !(first && kk == 0), one);
          done ^= 1u << g;
          if (final && S::kLead > 1) read ^= 1u << g;              // see scores()
          if (final || S::kLead > 1) tc::commit(BAR(O_FULL + g), one);
        };
        auto free_entry = [&](uint32_t entry) { tc::commit(BAR(KV_EMPTY + entry % NS), one); };
        WAIT(BAR(Q_FULL + qb), (r / S::kQBufs) & 1);
        tc::fence_after();
        const int lead = min(n, S::kLead << pair);
        for (int t = 0; t < lead; ++t, ++e) {
          const uint32_t k_addr = full(e);
          if (pair) {
            scores(t & 1, k_addr, t >= 2);
          } else {
            for (int g = 0; g <= last; ++g) scores(g, k_addr, t >= 1);
          }
          free_entry(e);
          if (t == n - 1) tc::commit(BAR(Q_EMPTY + qb), one);
        }
        for (int t = 0; t < n && !dead; ++t) {
          const int kt = t + lead;
          const bool more = kt < n;
          const uint32_t v_addr = full(e);
          uint32_t k_addr = 0;
          const int g0 = pair ? t & 1 : 0, g1 = pair ? t & 1 : last;
          for (int g = g0; g <= g1; ++g) {
            values(g, v_addr, t <= pair, t + 1 + pair >= n);
            if (g == g1) free_entry(e);
            if (!more) continue;
            if (g == g0) k_addr = full(e + 1);
            scores(g, k_addr, true);
            if (g == g1) {
              free_entry(e + 1);
              if (kt == n - 1) tc::commit(BAR(Q_EMPTY + qb), one);
            }
          }
          e += more ? 2 : 1;
        }
      }
      __syncwarp();
    }
  } else {
    after_previous();
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
    // ---- softmax: thread = 64 keys (half) of a row of its group = lane of tensor memory ----
    const int g = warp >> 3, half = (warp >> 2) & 1, r_in = (warp & 3) * 32 + lane;
    const uint32_t t_g = tmem + g * kGroupCols + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = t_g + half * 64, t_p = t_g + S::kColP + half * 32, t_o = t_g + kColO + half * (D / 2);   // its share of each
    const float sl2 = a.scale * kLog2e;
    // the two warps of a row's threads
    auto meet = [&] { asm volatile("bar.sync %0, 64;\n" ::"r"(1 + g * 4 + (warp & 3)) : "memory"); };
    uint32_t e0 = 0, done = 0, items = 0;                        // ring entries before this item; the group's key tiles and items
    // (A thread whose wait has run out goes on to the end without waiting: its partner meets it at every tile.)
    for (int r = 0; r < n_items; ++r) {
      int pair, n, kv_len;
      bool working;                                              // some row of this warp is the item's
      {
        const TileItem it = load_tile(tiles + r);
        pair = it.flags & kPair ? 1 : 0;
        n = (it.kv_len + kTileKeys - 1) / kTileKeys << pair;
        kv_len = it.kv_len;
        const int rows = it.n_tok * a.group;
        e0 += 2 * n;
        if (g == 1 && !pair && rows <= 128) continue;
        working = (pair ? 0 : g * 128) + (warp & 3) * 32 < rows;
      }
      const int step = 1 + pair;
      float m_used = -INFINITY;
      float2 l = both(0.f);
      for (int t = pair & g; t < n; t += step, ++done) {
        BLOCK(BAR(S_FULL + g), done & 1, kItemPolls);            // (the second group lets items of one group pass)
        tc::fence_after();
        const int valid = kv_len - (t >> pair) * kTileKeys;   // keys of this tile, if fewer than kTileKeys
        const bool opening = t < step;
        float sc[64];
        if (working) {
          tc::ld32(t_s, reinterpret_cast<uint32_t*>(sc));
          tc::ld32(t_s + 32, reinterpret_cast<uint32_t*>(sc) + 32);
          tc::wait_ld();
          tc::fence_before();
        }
        if constexpr (S::kLead > 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive_warp(BAR(S_READ + g));
        }
        if (working) {
          if (valid < kTileKeys) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (half * 64 + i >= valid) sc[i] = -INFINITY;
          }
          float mx4[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) mx4[u] = fmaxf(sc[u], sc[4 + u]);
#pragma unroll
          for (int i = 8; i < 64; i += 8)
#pragma unroll
            for (int u = 0; u < 4; ++u) mx4[u] = max3(mx4[u], sc[i + u], sc[i + 4 + u]);
          float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          sm_max[done & 1][g][half][r_in] = mx;
          meet();
          // Where P lies over S, one warp's stores go over scores that the other has loaded: its loads (wait_ld, fence_before) come first.
          if constexpr (S::kLead == 1) tc::fence_after();
          mx = fmaxf(mx, sm_max[done & 1][g][half ^ 1][r_in]);
          // O is free of the group's product before this one where that is awaited here, or where the next scores, which have
          // arrived, were issued behind it; so is P's place.
          if constexpr (S::kLead > 1) {
            if (!opening) {
              BLOCK(BAR(O_FULL + g), (done & 1) ^ 1);
              tc::fence_after();
            }
          }
          if (opening) {
            m_used = mx;
          } else if (__any_sync(0xffffffffu, (mx - m_used) * sl2 > kRescale)) {
            const float m_new = (mx - m_used) * sl2 > kRescale ? mx : m_used;
            // (one row's growth rescales the warp's 32: the others keep theirs, which may still be -inf, by a factor of exactly one)
            const float f = m_new == m_used ? 1.f : ex2((m_used - m_new) * sl2);
            m_used = m_new;
            l.x *= f;
            l.y *= f;
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
              uint32_t v[16];
              tc::ld16(t_o + c, v);
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
              tc::st16(t_o + c, v);
            }
          }
          // (no finite score yet: the weights are zero, not inf - inf)
          const float2 neg = both(m_used == -INFINITY ? 0.f : -m_used * sl2), by = both(sl2);
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2 x = fma2(make_float2(sc[c + 2 * i], sc[c + 2 * i + 1]), by, neg);
              x = make_float2(ex2(x.x), ex2(x.y));
              l = add2(l, x);
              pk[i] = pack2<T>(x.x, x.y);
            }
            tc::st16(t_p + c / 2, pk);
          }
        } else if constexpr (S::kLead > 1) {
          // no row of this warp is the item's: it keeps step only
          if (!opening) BLOCK(BAR(O_FULL + g), (done & 1) ^ 1);
        }
        if (t + step >= n && valid < kTileKeys && (g == 0 || pair)) {
          // Keys past the end: their P is zero, but the V rows behind them are whatever the pool or the ring held.  Cleared
          // before the group's threads report the tile's P, so that 0 * x stays 0.
          const uint32_t last_v = e0 - 1 - pair + (pair & g);  // ring entry of the group's last V tile
          BLOCK(BAR(KV_FULL + last_v % NS), (last_v / NS) & 1);
          if (r_in >= valid && half < S::kHalves) {
            unsigned char* v = base_ptr + S::kRing + (last_v % NS) * S::kTile + half * kBlockBytes + r_in * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(v + c * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        }
        if (working) tc::wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_warp(BAR(P_FULL + g));
      }
      // ---- epilogue: the next item's first product cannot touch O before this thread has arrived with its P ----
      float sum = l.x + l.y;
      if (working) {
        sm_sum[g][half][r_in] = sum;
        meet();
        sum += sm_sum[g][half ^ 1][r_in];
      }
      // A thread holds (half) a row; stored as it is, every instruction would touch 32 rows, 16 bytes each (an item's output then
      // took 20,000 cycles).  Lanes exchange their pieces instead and store whole sectors.
      const TileItem* again = tiles + r;                         // (not held in registers through the tiles)
      asm volatile("" : "+l"(again));
      const TileItem it = load_tile(again);
      const bool partial = it.part >= 0;
      const int rows = it.n_tok * a.group, row = pair ? r_in : g * 128 + r_in;
      unsigned long long to = 0;
      if (row < rows) {
        if (partial) {
          const size_t p = static_cast<size_t>(it.part + (pair & g) * rows + row);
          to = reinterpret_cast<unsigned long long>(a.part_acc + p * D + half * (D / 2));
          if (half == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * p) = make_float2(m_used * a.ml_scale, sum);
        } else {
          const int t = row / a.group, token = __ldg(a.row_token + it.tok0 + t), head = (it.kvh + (pair & g)) * a.group + (row - t * a.group);
          to = reinterpret_cast<unsigned long long>(static_cast<T*>(a.out) + (static_cast<size_t>(token) * a.q_heads + head) * D + half * (D / 2));
        }
      }
      BLOCK(BAR(O_FULL + g), S::kLead > 1 ? (done & 1) ^ 1 : items & 1);
      ++items;
      tc::fence_after();
      if (!working) continue;
      const float inv = 1.f / sum;
      if (partial) {
#pragma unroll 1
        for (int c = 0; c < D / 2; c += 16) {
          uint32_t v[16];
          tc::ld16(t_o + c, v);
          tc::wait_ld();
          transpose<4>(v, lane);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned long long row_to = __shfl_sync(0xffffffffu, to, (lane & 28) + i);
            if (row_to) *reinterpret_cast<uint4*>(row_to + c * 4 + (lane & 3) * 16) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < D / 2; c += 16) {
          uint32_t v[16], x[8];
          tc::ld16(t_o + c, v);
          tc::wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = pack2<T>(__uint_as_float(v[2 * i]) * inv, __uint_as_float(v[2 * i + 1]) * inv);
          transpose<2>(x, lane);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned long long row_to = __shfl_sync(0xffffffffu, to, (lane & 30) + i);
            if (row_to) *reinterpret_cast<uint4*>(row_to + c * 2 + (lane & 1) * 16) = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          }
        }
      }
      tc::fence_before();
    }
  }
  if (dead) report(a.host_err, kErrTileWait);
  if (n_items == 0 && blockIdx.x == 0 && threadIdx.x == 0) report(a.host_err, kErrOtherPlan);
  tc::fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    tc::fence_after();
    tc::dealloc<512>(tmem);
  }
}

// Folds the partials of each listed (token, kv head): thread = (record, head of the group, VEC dims).  Partials sit in L2; a
// batch of loads is in flight before the first is used.
constexpr int kMergeThreads = 256, kMergeBatch = 8;
struct MergeArgs {
  const MergeRow* rows;
  int n_rows, q_heads, group, head_dim;
  const float *tile_ml, *tile_acc, *own_ml, *own_acc;
  void* out;
  const PlanHeader* header;
  int stamp;
  unsigned int* host_err;
};
template <typename T, bool LOG2, int VEC>
__global__ void __launch_bounds__(kMergeThreads) segment_merge_kernel(const MergeArgs a) {
  pdl_launch_dependents();
  const int per_head = a.head_dim / VEC, per_row = a.group * per_head;
  const long long i = blockIdx.x * static_cast<long long>(kMergeThreads) + threadIdx.x, row = i / per_row;
  const bool other = __ldg(&a.header->stamp) != a.stamp, live = row < a.n_rows && !other;
  MergeRow m{};
  if (live) {                                            // part of the plan, complete before the kernels that wrote the partials began
    const int4 x = __ldg(reinterpret_cast<const int4*>(a.rows + row)), y = __ldg(reinterpret_cast<const int4*>(a.rows + row) + 1);
    m = MergeRow{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  }
  pdl_wait();
  if (other && i == 0) report(a.host_err, kErrOtherPlan);
  if (!live) return;
  const int at = static_cast<int>(i - row * per_row), h = at / per_head, d = (at - h * per_head) * VEC, head = m.kvh * a.group + h;
  const int n = m.n_tile + m.n_own;
  float run = -INFINITY, sum = 0.f, acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
  for (int p0 = 0; p0 < n; p0 += kMergeBatch) {
    float2 ml[kMergeBatch];
    float x[kMergeBatch][VEC];
#pragma unroll
    for (int u = 0; u < kMergeBatch; ++u) {
      ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[u][v] = 0.f;
      const int p = p0 + u;
      if (p < n) {
        const bool tile = p < m.n_tile;
        const size_t r = tile ? static_cast<size_t>(m.tile_row) + h + static_cast<size_t>(p) * m.tile_stride
                              : static_cast<size_t>(m.own_part + p - m.n_tile) * a.q_heads + head;
        ml[u] = __ldcg(reinterpret_cast<const float2*>(tile ? a.tile_ml : a.own_ml) + r);
        const float* src = (tile ? a.tile_acc : a.own_acc) + r * a.head_dim + d;
        if constexpr (VEC == 4) {
          const float4 f = __ldcg(reinterpret_cast<const float4*>(src));
          x[u][0] = f.x; x[u][1] = f.y; x[u][2] = f.z; x[u][3] = f.w;
        } else {
          x[u][0] = __ldcg(src);
        }
      }
    }
    float top = run;
#pragma unroll
    for (int u = 0; u < kMergeBatch; ++u) top = fmaxf(top, ml[u].x);
    auto weight = [&](float m0) { return m0 == -INFINITY ? 0.f : LOG2 ? exp2f(m0 - top) : expf(m0 - top); };
    const float keep = weight(run);
    sum *= keep;
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] *= keep;
#pragma unroll
    for (int u = 0; u < kMergeBatch; ++u) {
      const float f = weight(ml[u].x);
      sum += f * ml[u].y;
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] += f * x[u][v];
    }
    run = top;
  }
  const float inv = n > 0 ? 1.f / sum : 0.f;
  T* o = static_cast<T*>(a.out) + (static_cast<size_t>(m.token) * a.q_heads + head) * a.head_dim + d;
  if constexpr (VEC == 4 && sizeof(T) == 2) {
    *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<float4*>(o) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
  } else {
    o[0] = Elem<T>::from_f32(acc[0] * inv);
  }
}

// ---------------------------------------------------------------- launches ----
// Rows of q as [tokens][heads][head_dim], fetched in boxes of 64 dims x heads x tokens.
int make_q_map(CUtensorMap* map, const void* q, PoolElem elem, int head_dim, int heads, int n_tokens, int box_heads, int box_tokens) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(n_tokens)};
  const cuuint64_t strides[2] = {dims[0] * 2, dims[0] * dims[1] * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)}, step[3] = {1, 1, 1};
  const CUresult r = tensor_map_encoder()(map, elem == PoolElem::kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                                          const_cast<void*>(q), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? PKV_OK : fail(PKV_E_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
}

template <typename T, int D>
int launch_tiles(const TileArgs& a, int blocks, int kv_heads, const void* q, int n_tokens, const void* k_cache, const void* v_cache, uint64_t pool_rows, cudaStream_t stream) {
  using S = TileSmem<D>;
  auto kern = tile_attn_kernel<T, D>;
  static thread_local int configured_device = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured_device != dev) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    if (e != cudaSuccess) return fail(PKV_E_CUDA, "tile_attn_kernel: cannot reserve %d bytes of shared memory: %s", S::kBytes, cudaGetErrorString(e));
    configured_device = dev;
  }
  constexpr PoolElem elem = std::is_same<T, __half>::value ? PoolElem::kF16 : PoolElem::kBF16;
  alignas(64) CUtensorMap qmap, qmap_many, kmap, vmap;
  int st = make_q_map(&qmap, q, elem, D, a.q_heads, n_tokens, a.group, 1);
  if (st == PKV_OK) st = make_q_map(&qmap_many, q, elem, D, a.q_heads, n_tokens, a.group, a.box_tokens);
  if (st == PKV_OK) st = make_pool_tensor_map(&kmap, k_cache, elem, kv_heads * D, 1u << a.box_log2, pool_rows);
  if (st == PKV_OK) st = make_pool_tensor_map(&vmap, v_cache, elem, kv_heads * D, 1u << a.box_log2, pool_rows);
  if (st != PKV_OK) return st;
  launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(kTileThreads), S::kBytes, stream, a, qmap, qmap_many, kmap, vmap);
  return check_launch("tile_attn_kernel");
}

int log2_floor(int x) {
  int l = 0;
  while ((2 << l) <= x) ++l;
  return l;
}

struct SegmentOffsets { size_t seq, pos, rows, items, lists, tiles, merge, image, tile_ml, tile_acc, ml, acc, total; };
struct SegmentCounts { size_t rows, items, shares, lists, tiles, merge, tile_rows, parts; };   // shares, lists: with the end
SegmentOffsets segment_offsets(const SegmentGeometry& g, const SegmentCounts& c) {
  SegmentOffsets o;
  size_t at = align256(sizeof(PlanHeader));
  auto region = [&](size_t bytes) {
    const size_t here = at;
    at = align256(at + bytes);
    return here;
  };
  o.seq = region(sizeof(int) * g.n_tokens);
  o.pos = region(sizeof(int) * g.n_tokens);
  o.rows = region(sizeof(int) * c.rows);
  o.items = region(sizeof(WorkItem) * c.items + sizeof(int) * c.shares);
  o.lists = region(sizeof(int) * c.lists);
  o.tiles = region(sizeof(TileItem) * c.tiles);
  o.merge = region(sizeof(MergeRow) * c.merge);
  o.image = at;
  o.tile_ml = region(sizeof(float) * 2 * c.tile_rows);
  o.tile_acc = region(sizeof(float) * c.tile_rows * g.head_dim);
  o.ml = region(sizeof(float) * 2 * c.parts * g.q_heads);
  o.acc = region(sizeof(float) * c.parts * g.q_heads * g.head_dim);
  o.total = at;
  return o;
}
// For any step of these sizes: a tile has a token at least, and every block cuts one at most.
SegmentOffsets segment_bounds(const SegmentGeometry& g, bool prefix) {
  const size_t n = static_cast<size_t>(g.n_tokens), sms = static_cast<size_t>(decode_sms());
  const size_t items = n + own_extra(g) + 2;
  return segment_offsets(g, SegmentCounts{n, items, items + 1, sms + 1, n * g.kv_heads + 2 * sms, n * g.kv_heads,
                                          static_cast<size_t>(most_tile_rows(g, decode_sms(), prefix)), static_cast<size_t>(most_parts(g, prefix))});
}

int check_geometry(const char* fn, const SegmentGeometry& g) {
  if (g.q_heads <= 0 || g.kv_heads <= 0 || g.head_dim <= 0 || g.block_size <= 0)
    return fail(PKV_E_ARG, "%s: q_heads %d, kv_heads %d, head_dim %d, block_size %d must all be > 0", fn, g.q_heads, g.kv_heads, g.head_dim, g.block_size);
  if (g.elem_bytes != 2 && g.elem_bytes != 4) return fail(PKV_E_ARG, "%s: elements of %d bytes; 2 (f16, bf16) or 4 (f32)", fn, g.elem_bytes);
  if (g.q_heads % g.kv_heads) return fail(PKV_E_UNSUPPORTED, "%s: q_heads %d is not a multiple of kv_heads %d", fn, g.q_heads, g.kv_heads);
  if (g.head_dim > 256) return fail(PKV_E_UNSUPPORTED, "%s: head_dim %d exceeds 256", fn, g.head_dim);
  if (static_cast<long long>(g.n_tokens) * g.q_heads > 0x7fffffffll) return fail(PKV_E_UNSUPPORTED, "%s: %d tokens of %d heads; at most 2^31 - 1 rows", fn, g.n_tokens, g.q_heads);
  return PKV_OK;
}

enum Kind { kCross = 1, kPrefix = 2 };
constexpr int kMostKeys = 1 << 30;       // of a token: lengths rounded up to tiles stay below 2^31

// PKV_SEGMENT_TILES=1: whatever the tile kernel can take goes to it, =0: nothing does; else what is reckoned to take least.
// Read at every planning call (a measurement and testing aid).
int tiles_asked() {
  const char* e = std::getenv("PKV_SEGMENT_TILES");
  return e && (*e == '0' || *e == '1') ? *e - '0' : -1;
}

// Names what a step's launches are made for: everything in the plan but the caller's num_blocks.  Never 0.
int stamp_of(const pkv_segment_plan& plan) {
  pkv_segment_plan p = plan;
  p.num_blocks = 0;
  static_assert(sizeof(p) % 8 == 0, "whole words, no padding");
  unsigned long long word, h = 0x9e3779b97f4a7c15ull;
  for (size_t i = 0; i < sizeof(p); i += 8) {
    std::memcpy(&word, reinterpret_cast<const char*>(&p) + i, 8);
    h = (h ^ word) * 0xd1342543de82ef95ull;
    h ^= h >> 32;
  }
  return static_cast<int>(h) | 1;
}
// What the cluster form, which reads the tokens' positions and sequences only, needs: a step of the same sizes.
int cluster_stamp_of(const pkv_segment_plan& plan) {
  pkv_segment_plan p{};
  p.kind = plan.kind;
  p.n_tokens = plan.n_tokens; p.q_heads = plan.q_heads; p.kv_heads = plan.kv_heads; p.head_dim = plan.head_dim;
  p.block_size = plan.block_size; p.elem_bytes = plan.elem_bytes;
  return stamp_of(p);
}

// every: every row has keys.
int write_image(const char* fn, Kind kind, const SegmentGeometry& g, const SegmentLists& l, const std::vector<int>& seq, const std::vector<int>& pos,
                bool every, bool cluster, void* h_staging, size_t staging_bytes, size_t workspace_bytes, pkv_segment_plan* plan) {
  const SegmentOffsets o = segment_offsets(g, SegmentCounts{l.row_token.size(), l.items.size(), l.first.size(), l.list_first.size(), l.tiles.size(),
                                                            l.merge.size(), static_cast<size_t>(l.n_tile_rows), static_cast<size_t>(l.n_parts)});
  if (o.total > workspace_bytes) return fail(PKV_E_WORKSPACE, "%s: workspace of %zu bytes; this step takes %zu", fn, workspace_bytes, o.total);
  if (o.image > staging_bytes) return fail(PKV_E_WORKSPACE, "%s: staging buffer of %zu bytes; this step's plan takes %zu", fn, staging_bytes, o.image);
  if (l.list_cycles > kMostListCycles)
    return fail(PKV_E_UNSUPPORTED, "%s: more than a second's work (%.3g cycles) for one call; split the step", fn, static_cast<double>(l.list_cycles));
  if (l.n_tile_rows > 0x7fffffffll || static_cast<long long>(l.items.size()) * g.kv_heads > 0x7fffffffll)
    return fail(PKV_E_UNSUPPORTED, "%s: more than 2^31 - 1 work items or partial rows", fn);
  char* img = static_cast<char*>(h_staging);
  std::memset(img, 0, o.seq);
  PlanHeader* hd = reinterpret_cast<PlanHeader*>(img);
  hd->magic = kPlanMagic;
  hd->n_items = static_cast<int>(l.items.size());
  hd->chunk = l.chunk;
  hd->n_tokens = g.n_tokens;
  hd->n_parts = l.n_parts;
  hd->kv_heads = g.kv_heads;
  hd->n_shares = l.first.empty() ? 0 : static_cast<int>(l.first.size()) - 1;
  auto put = [&](size_t at, const void* p, size_t bytes) { if (bytes) std::memcpy(img + at, p, bytes); };
  put(o.seq, seq.data(), seq.size() * sizeof(int));
  put(o.pos, pos.data(), pos.size() * sizeof(int));
  put(o.rows, l.row_token.data(), l.row_token.size() * sizeof(int));
  put(o.items, l.items.data(), l.items.size() * sizeof(WorkItem));
  put(o.items + l.items.size() * sizeof(WorkItem), l.first.data(), l.first.size() * sizeof(int));
  put(o.lists, l.list_first.data(), l.list_first.size() * sizeof(int));
  put(o.tiles, l.tiles.data(), l.tiles.size() * sizeof(TileItem));
  put(o.merge, l.merge.data(), l.merge.size() * sizeof(MergeRow));
  std::memset(plan, 0, sizeof(*plan));
  plan->kind = kind;
  plan->n_tokens = g.n_tokens; plan->q_heads = g.q_heads; plan->kv_heads = g.kv_heads; plan->head_dim = g.head_dim;
  plan->block_size = g.block_size; plan->elem_bytes = g.elem_bytes;
  plan->n_tiles = static_cast<int>(l.tiles.size());
  plan->n_items = static_cast<int>(l.items.size());
  plan->n_merged = static_cast<int>(l.merge.size());
  plan->n_parts = l.n_parts;
  plan->n_lists = l.list_first.empty() ? 0 : static_cast<int>(l.list_first.size()) - 1;
  plan->n_tile_rows = static_cast<int>(l.n_tile_rows);
  plan->image_bytes = o.image;
  plan->workspace_bytes = o.total;
  plan->off_seq = o.seq; plan->off_pos = o.pos; plan->off_rows = o.rows; plan->off_items = o.items;
  plan->off_lists = o.lists; plan->off_tiles = o.tiles; plan->off_merge = o.merge;
  plan->off_tile_ml = o.tile_ml; plan->off_tile_acc = o.tile_acc; plan->off_ml = o.ml; plan->off_acc = o.acc;
  if (every && cluster && l.n_parts > 0) plan->cluster = decode_cluster_size(g.n_tokens, l.longest, g.q_heads, g.kv_heads, g.head_dim, &plan->cluster_least);
  hd->stamp = stamp_of(*plan);
  hd->cluster_stamp = every ? cluster_stamp_of(*plan) : 0;
  return PKV_OK;
}

int plan_cross(const char* fn, const int* q_start, const int* q_len, const int* kv_len, int n_seqs, const SegmentGeometry& g, void* h_staging,
               size_t staging_bytes, size_t workspace_bytes, pkv_segment_plan* plan) {
  if (!plan) return fail(PKV_E_ARG, "%s: null plan", fn);
  std::memset(plan, 0, sizeof(*plan));                           // (kind 0: a refused plan is refused again where it is used)
  if (g.n_tokens <= 0 || n_seqs <= 0) {
    plan->kind = kCross;
    return PKV_OK;
  }
  if (!q_len || !kv_len || !h_staging) return fail(PKV_E_ARG, "%s: null pointer", fn);
  int st = check_geometry(fn, g);
  if (st != PKV_OK) return st;
  std::vector<int> seq(g.n_tokens, -1), pos(g.n_tokens, -1), empty, start(n_seqs);
  long long next = 0;
  int listed = 0;
  for (int s = 0; s < n_seqs; ++s) {
    const long long at = q_start ? q_start[s] : next;
    if (kv_len[s] > kMostKeys) return fail(PKV_E_UNSUPPORTED, "%s: sequence %d has %d keys; at most 2^30", fn, s, kv_len[s]);
    if (q_len[s] < 0 || kv_len[s] < 0 || at < 0 || at + q_len[s] > g.n_tokens)
      return fail(PKV_E_ARG, "%s: sequence %d has rows %lld .. + %d of %d and %d keys", fn, s, at, q_len[s], g.n_tokens, kv_len[s]);
    next = at + q_len[s];
    start[s] = static_cast<int>(at);
    listed += q_len[s];
    for (int t = start[s]; t < next; ++t) {
      if (seq[t] >= 0) return fail(PKV_E_ARG, "%s: row %d belongs to sequences %d and %d", fn, t, seq[t], s);
      seq[t] = s;
      pos[t] = kv_len[s] - 1;
      if (kv_len[s] == 0) empty.push_back(t);
    }
  }
  // Sequences of at least `fewest` tokens go to the tile kernel, the others to the decode kernels, which fetch the keys anew for
  // every token.  The number for which the step is reckoned to take least.
  std::vector<Segment> segs;
  std::vector<OwnRange> own;
  SegmentLists l;
  auto split = [&](int fewest) {
    segs.clear();
    own.clear();
    l.row_token.clear();
    for (int s = 0; s < n_seqs; ++s) {
      if (q_len[s] == 0 || kv_len[s] == 0) continue;
      const bool tiled = g.tiles() && q_len[s] >= fewest && kv_len[s] <= kMostTileKeys;
      if (tiled) segs.push_back(Segment{static_cast<int>(l.row_token.size()), q_len[s], kv_len[s], ~s});
      for (int t = start[s]; t < start[s] + q_len[s]; ++t) {
        if (tiled) l.row_token.push_back(t);
        else own.push_back(OwnRange{t, 0, kv_len[s]});
      }
    }
  };
  const int asked = tiles_asked();
  int fewest = asked == 1 ? 1 : asked == 0 ? 0x7fffffff : kMinTileTokens;
  if (g.tiles() && asked < 0) {
    long long least = -1;
    size_t tiled = 0;
    for (int f = kMinTileTokens; f <= kManyTileTokens; f = f < 4 ? f + 1 : f * 2) {
      split(f);
      if (least >= 0 && segs.size() == tiled) continue;          // the same sequences as before
      tiled = segs.size();
      const long long c = step_cycles(segs, own, l.row_token, g, decode_sms(), false);
      if (least < 0 || c < least) { least = c; fewest = f; }
      if (segs.empty()) break;
    }
  }
  split(fewest);
  list_segments(segs, own, empty, g, decode_sms(), false, l);
  return write_image(fn, kCross, g, l, seq, pos, empty.empty() && listed == g.n_tokens, segs.empty(), h_staging, staging_bytes, workspace_bytes, plan);
}

int plan_prefix(const char* fn, const int* token_pos, int prefix_len, const SegmentGeometry& g, void* h_staging, size_t staging_bytes,
                size_t workspace_bytes, pkv_segment_plan* plan) {
  if (!plan) return fail(PKV_E_ARG, "%s: null plan", fn);
  std::memset(plan, 0, sizeof(*plan));
  if (g.n_tokens <= 0) {
    plan->kind = kPrefix;
    return PKV_OK;
  }
  if (!token_pos || !h_staging) return fail(PKV_E_ARG, "%s: null pointer", fn);
  if (prefix_len < 0) return fail(PKV_E_ARG, "%s: prefix_len %d must not be negative", fn, prefix_len);
  int st = check_geometry(fn, g);
  if (st != PKV_OK) return st;
  // the decode kernels fetch boxes of 16 slots: a token's own keys begin on a multiple of 16
  const int shared = g.tiles() && prefix_len <= kMostTileKeys ? prefix_len & ~15 : 0;
  std::vector<int> none, pos(token_pos, token_pos + g.n_tokens), empty;
  std::vector<Segment> segs;
  std::vector<OwnRange> own;
  SegmentLists l;
  for (int t = 0; t < g.n_tokens; ++t) {
    if (token_pos[t] < 0) return fail(PKV_E_ARG, "%s: token %d has negative position %d", fn, t, token_pos[t]);
    if (token_pos[t] >= kMostKeys) return fail(PKV_E_UNSUPPORTED, "%s: token %d has position %d; below 2^30", fn, t, token_pos[t]);
    if (shared > 0 && token_pos[t] >= shared - 1) l.row_token.push_back(t);
  }
  // worth while where every token's own way through the prefix, on the decode kernels, is reckoned to take longer
  auto ranges = [&](bool together) {
    own.clear();
    for (int t = 0; t < g.n_tokens; ++t) {
      const int begin = together && token_pos[t] >= shared - 1 ? shared : 0, len = token_pos[t] + 1 - begin;
      if (len > 0) own.push_back(OwnRange{t, begin, len});
    }
  };
  const int asked = tiles_asked();
  if (asked == 1 && !l.row_token.empty()) {
    segs.push_back(Segment{0, static_cast<int>(l.row_token.size()), shared, l.row_token[0]});
  } else if (asked < 0 && l.row_token.size() >= 2) {
    ranges(false);
    const long long apart = step_cycles(segs, own, l.row_token, g, decode_sms(), true);
    ranges(true);
    segs.push_back(Segment{0, static_cast<int>(l.row_token.size()), shared, l.row_token[0]});
    if (step_cycles(segs, own, l.row_token, g, decode_sms(), true) >= apart) segs.clear();
  }
  if (segs.empty()) l.row_token.clear();
  ranges(!segs.empty());
  list_segments(segs, own, empty, g, decode_sms(), true, l);
  return write_image(fn, kPrefix, g, l, none, pos, true, segs.empty(), h_staging, staging_bytes, workspace_bytes, plan);
}

int upload(const char* fn, pkv_segment_plan* plan, const void* h_staging, void* workspace, pkv_stream stream) {
  if (plan->n_tokens <= 0) return PKV_OK;
  const cudaError_t e = cudaMemcpyAsync(workspace, h_staging, plan->image_bytes, cudaMemcpyHostToDevice, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(PKV_E_CUDA, "%s: plan upload failed: %s", fn, cudaGetErrorString(e));
  return PKV_OK;
}

template <typename T>
int segment_attn(Kind kind, const pkv_segment_plan* plan, const void* q, const void* k_cache, const void* v_cache, const int* block_tables,
                 const int* table_offset, const int* token_seq, void* out, float scale, void* workspace, size_t workspace_bytes, pkv_stream stream) {
  const char* fn = kind == kCross ? "pkv_cross_attn" : "pkv_prefix_attn";
  if (!plan) return fail(PKV_E_ARG, "%s: null plan", fn);
  if (plan->kind != kind) return fail(PKV_E_ARG, "%s: a plan of the other kind, or one that was never made", fn);
  if (plan->n_tokens <= 0 || (plan->n_tiles == 0 && plan->n_items == 0 && plan->n_merged == 0)) return PKV_OK;
  int st = check_error_mirror(fn);
  if (st != PKV_OK) return st;
  if (plan->elem_bytes != static_cast<int>(sizeof(T))) return fail(PKV_E_ARG, "%s: the plan is for elements of %d bytes", fn, plan->elem_bytes);
  const bool keys = plan->n_tiles > 0 || plan->n_items > 0;      // else every row's output is zero
  if (!out || (keys && (!q || !k_cache || !v_cache || !block_tables || !table_offset || (kind == kPrefix && !token_seq))))
    return fail(PKV_E_ARG, "%s: null device pointer", fn);
  if (!(scale > 0.f)) return fail(PKV_E_ARG, "%s: scale must be positive", fn);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255)) return fail(PKV_E_ARG, "%s: workspace null or not 256-byte aligned", fn);
  if (workspace_bytes < plan->workspace_bytes) return fail(PKV_E_WORKSPACE, "%s: workspace of %zu bytes; the plan takes %zu", fn, workspace_bytes, plan->workspace_bytes);
  const int D = plan->head_dim, group = plan->q_heads / plan->kv_heads;
  if (static_cast<size_t>(D) * sizeof(T) % 16 == 0 && (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)))
    return fail(PKV_E_ARG, "%s: q, out and the K/V pools must be 16-byte aligned", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const uint64_t pool_rows = plan->num_blocks > 0 ? static_cast<uint64_t>(plan->num_blocks) * plan->block_size : 0;
  const bool log2_domain = decode_log2_domain<T>(plan->q_heads, plan->kv_heads, D, plan->block_size, scale);
  const int* seq = kind == kCross ? reinterpret_cast<const int*>(ws + plan->off_seq) : token_seq;
  float *ml = reinterpret_cast<float*>(ws + plan->off_ml), *acc = reinterpret_cast<float*>(ws + plan->off_acc);
  float *tile_ml = reinterpret_cast<float*>(ws + plan->off_tile_ml), *tile_acc = reinterpret_cast<float*>(ws + plan->off_tile_acc);
  unsigned int* host_err = error_mirror(true);
  const PlanHeader* header = reinterpret_cast<const PlanHeader*>(ws);
  const int stamp = stamp_of(*plan);
  if (plan->n_tiles > 0) {
    if constexpr (sizeof(T) == 2) {
      if (!tensor_map_encoder()) return fail(PKV_E_CUDA, "%s: cuTensorMapEncodeTiled is not available from this driver", fn);
      TileArgs a;
      a.block_tables = block_tables; a.table_offset = table_offset; a.token_seq = seq;
      a.row_token = reinterpret_cast<const int*>(ws + plan->off_rows);
      a.list_first = reinterpret_cast<const int*>(ws + plan->off_lists);
      a.tiles = reinterpret_cast<const TileItem*>(ws + plan->off_tiles);
      a.header = header; a.stamp = stamp;
      a.out = out; a.part_ml = tile_ml; a.part_acc = tile_acc;
      a.q_heads = plan->q_heads; a.group = group;
      a.block_size = plan->block_size; a.bs_log2 = log2_floor(plan->block_size); a.box_log2 = std::min(a.bs_log2, 7);
      a.box_tokens = std::max(1, kBoxRows / group);
      a.scale = scale;
      a.ml_scale = log2_domain ? scale * 1.4426950408889634f : scale;
      a.host_err = host_err;
      const uint64_t rows = pool_rows ? pool_rows : 1ull << 30;
      st = D == 64 ? launch_tiles<T, 64>(a, plan->n_lists, plan->kv_heads, q, plan->n_tokens, k_cache, v_cache, rows, s) : launch_tiles<T, 128>(a, plan->n_lists, plan->kv_heads, q, plan->n_tokens, k_cache, v_cache, rows, s);
      if (st != PKV_OK) return st;
    }
  }
  if (plan->n_items > 0) {
    DecodeList l;
    l.q = q; l.k_cache = k_cache; l.v_cache = v_cache; l.block_tables = block_tables; l.table_offset = table_offset; l.token_seq = seq;
    l.token_pos = reinterpret_cast<const int*>(ws + plan->off_pos);
    l.out = out;
    l.n_tokens = plan->n_tokens; l.q_heads = plan->q_heads; l.kv_heads = plan->kv_heads; l.head_dim = D; l.block_size = plan->block_size;
    l.scale = scale;
    l.header = header;
    l.stamp = stamp; l.cluster_stamp = plan->cluster > 0 ? cluster_stamp_of(*plan) : 0;
    l.items = reinterpret_cast<const WorkItem*>(ws + plan->off_items);
    l.n_items = plan->n_items;
    l.part_ml = ml; l.part_acc = acc;
    l.pool_rows = pool_rows;
    l.host_err = host_err;
    l.behind_tiles = plan->n_tiles > 0;
    l.cluster = plan->cluster; l.cluster_least = plan->cluster_least;
    bool merged = false;
    st = decode_listed<T>(l, s, &merged);
    if (st != PKV_OK || merged) return st;
  }
  if (plan->n_merged > 0) {
    MergeArgs m{reinterpret_cast<const MergeRow*>(ws + plan->off_merge), plan->n_merged, plan->q_heads, group, D, tile_ml, tile_acc, ml, acc, out, header, stamp, host_err};
    // four values in one store where every row of out begins on a multiple of them (rows of other than 16-byte multiples may begin anywhere)
    const int vec = D % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0 ? 4 : 1;
    const long long blocks = (static_cast<long long>(plan->n_merged) * group * (D / vec) + kMergeThreads - 1) / kMergeThreads;
    if (blocks > 0x7fffffffll) return fail(PKV_E_UNSUPPORTED, "%s: %lld blocks to merge", fn, blocks);
    auto kern = vec == 4 ? (log2_domain ? segment_merge_kernel<T, true, 4> : segment_merge_kernel<T, false, 4>)
                         : (log2_domain ? segment_merge_kernel<T, true, 1> : segment_merge_kernel<T, false, 1>);
    launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(kMergeThreads), 0, s, m);
    return check_launch("segment_merge_kernel");
  }
  return PKV_OK;
}

// No exception leaves the C entry points.
template <typename F> int guarded(const char* fn, F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(PKV_E_NOMEM, "%s: out of host memory", fn);
  } catch (...) {
    return fail(PKV_E_STATE, "%s: internal error", fn);
  }
}

}  // namespace

int tile_read_flags(unsigned int* flags) {
  unsigned int v = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_pkv_tile_error, sizeof(v));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_pkv_tile_error, &zero, sizeof(zero));
  if (e != cudaSuccess) return fail(PKV_E_CUDA, "pkv_debug_device_flags: %s", cudaGetErrorString(e));
  *flags = v;
  return PKV_OK;
}

}  // namespace pkv

using namespace pkv;

extern "C" {

static size_t segment_workspace(int n_tokens, int q_heads, int kv_heads, int head_dim, bool prefix) {
  if (n_tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || q_heads % kv_heads) return 0;
  return segment_bounds(SegmentGeometry{n_tokens, q_heads, kv_heads, head_dim, 16, 2}, prefix).total;
}
size_t pkv_cross_workspace_bytes(int n_tokens, int q_heads, int kv_heads, int head_dim) { return segment_workspace(n_tokens, q_heads, kv_heads, head_dim, false); }
size_t pkv_prefix_workspace_bytes(int n_tokens, int q_heads, int kv_heads, int head_dim) { return segment_workspace(n_tokens, q_heads, kv_heads, head_dim, true); }
size_t pkv_segment_staging_bytes(int n_tokens, int q_heads, int kv_heads) {
  if (n_tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return 0;
  return segment_bounds(SegmentGeometry{n_tokens, q_heads, kv_heads, 64, 16, 2}, true).image;
}

int pkv_cross_plan_host_image(const int* h_q_start, const int* h_q_len, const int* h_kv_len, int n_seqs, int n_tokens, int q_heads, int kv_heads,
                              int head_dim, int block_size, int elem_bytes, void* h_staging, size_t staging_bytes, size_t workspace_bytes,
                              pkv_segment_plan* plan) {
  const char* fn = "pkv_cross_plan_host_image";
  return guarded(fn, [&] {
    return plan_cross(fn, h_q_start, h_q_len, h_kv_len, n_seqs, SegmentGeometry{n_tokens, q_heads, kv_heads, head_dim, block_size, elem_bytes}, h_staging,
                      staging_bytes, workspace_bytes, plan);
  });
}
int pkv_cross_plan_host(const int* h_q_start, const int* h_q_len, const int* h_kv_len, int n_seqs, int n_tokens, int q_heads, int kv_heads,
                        int head_dim, int block_size, int elem_bytes, void* h_staging, size_t staging_bytes, void* workspace, size_t workspace_bytes,
                        pkv_stream stream, pkv_segment_plan* plan) {
  const char* fn = "pkv_cross_plan_host";
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255)) return fail(PKV_E_ARG, "%s: workspace null or not 256-byte aligned", fn);
  const int st = pkv_cross_plan_host_image(h_q_start, h_q_len, h_kv_len, n_seqs, n_tokens, q_heads, kv_heads, head_dim, block_size, elem_bytes,
                                           h_staging, staging_bytes, workspace_bytes, plan);
  return st != PKV_OK ? st : upload(fn, plan, h_staging, workspace, stream);
}
int pkv_prefix_plan_host_image(const int* h_token_pos, int n_tokens, int prefix_len, int q_heads, int kv_heads, int head_dim, int block_size,
                               int elem_bytes, void* h_staging, size_t staging_bytes, size_t workspace_bytes, pkv_segment_plan* plan) {
  const char* fn = "pkv_prefix_plan_host_image";
  return guarded(fn, [&] {
    return plan_prefix(fn, h_token_pos, prefix_len, SegmentGeometry{n_tokens, q_heads, kv_heads, head_dim, block_size, elem_bytes}, h_staging,
                       staging_bytes, workspace_bytes, plan);
  });
}
int pkv_prefix_plan_host(const int* h_token_pos, int n_tokens, int prefix_len, int q_heads, int kv_heads, int head_dim, int block_size,
                         int elem_bytes, void* h_staging, size_t staging_bytes, void* workspace, size_t workspace_bytes, pkv_stream stream,
                         pkv_segment_plan* plan) {
  const char* fn = "pkv_prefix_plan_host";
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255)) return fail(PKV_E_ARG, "%s: workspace null or not 256-byte aligned", fn);
  const int st = pkv_prefix_plan_host_image(h_token_pos, n_tokens, prefix_len, q_heads, kv_heads, head_dim, block_size, elem_bytes, h_staging,
                                            staging_bytes, workspace_bytes, plan);
  return st != PKV_OK ? st : upload(fn, plan, h_staging, workspace, stream);
}

#define PKV_SEGMENT_ATTN(SUFFIX, TYPE)                                                                                                            \
  int pkv_cross_attn_##SUFFIX(const pkv_segment_plan* plan, const void* q, const void* k_cache, const void* v_cache, const int* block_tables,      \
                              const int* table_offset, void* out, float scale, void* workspace, size_t workspace_bytes, pkv_stream stream) {       \
    return segment_attn<TYPE>(kCross, plan, q, k_cache, v_cache, block_tables, table_offset, nullptr, out, scale, workspace, workspace_bytes,      \
                              stream);                                                                                                            \
  }                                                                                                                                               \
  int pkv_prefix_attn_##SUFFIX(const pkv_segment_plan* plan, const void* q, const void* k_cache, const void* v_cache, const int* block_tables,     \
                               const int* table_offset, const int* token_seq, void* out, float scale, void* workspace, size_t workspace_bytes,     \
                               pkv_stream stream) {                                                                                               \
    return segment_attn<TYPE>(kPrefix, plan, q, k_cache, v_cache, block_tables, table_offset, token_seq, out, scale, workspace, workspace_bytes,   \
                              stream);                                                                                                            \
  }
PKV_SEGMENT_ATTN(f16, __half)
PKV_SEGMENT_ATTN(bf16, __nv_bfloat16)
PKV_SEGMENT_ATTN(f32, float)
}
