// Attention over packed sequences with a sliding window and a few first tokens that stay visible, optionally with a bias
// by distance (head size 64, fp16 in and out, heads that may share keys and values).
//
// Query i of a sequence of Lq queries over Lk keys stands at position p = i + Lk - Lq.  It sees key j < Lk if
//   j <= p + right   and   (j >= p - left  or  j < sinks),
//   out_i = sum_j softmax_j(scale * q_i . k_j + bias[h, j - p]) v_j     over the keys it sees, 0 where it sees none.
//
// window_mha_kernel: 128 query rows of a head at a time.  The keys that any of them sees are a run of the first keys
// and a run around the tile; the two are laid end to end ("virtual" keys: the first run, in steps of 32, then the second) and
// walked in tiles of 64, so a handful of first tokens does not cost a tile of its own and the window starts wherever
// the first row's does.  The tile that holds the seam is fetched in boxes of 32 keys.
//   What bounds it is the chain of a softmax (scores from tensor memory, maximum, exponentials, weights back), not the tensor
//   core: a warp by itself leaves the special-function unit idle more than half of the time.  So two groups of four warps
//   share the 128 rows, one takes the even tiles, the other the odd ones, each with scores, weights, reference, sum and O of
//   its own; the two results are put together when the item ends (the groups take turns in that).  With two CTAs to an SM
//   four warps take turns on each scheduler.
//   Measured on B200: one sequence of 8192, 2047 keys back, 16 heads over 4: 100.4 us, 600 TFLOP/s of the visible pairs (one group
//   with 128-key tiles: 116); 8 ragged sequences of up to 4096, 256 keys to either side, bias, 12 heads: 79 us.  A group's tile of 64
//   keys takes 2546 clocks with four groups to an SM: 700 until S is there, 540 for scores and maximum, 1060 for the weights (the
//   special-function unit works 448 of them), 240 to hand them over.
//   S = Q K^T (128 x 64 x 64) lands in 64 columns of tensor memory; the weights go back over them as fp16 pairs, from where
//   O += P V takes them; the next S of a group is issued right behind that product.  One thread issues a group's MMAs and
//   they execute in order, so no barrier stands between P V and the S that overwrites P.
// window_few_kernel: calls of few queries (single tokens), see there.
#include <float.h>
#include <math.h>

#include <mutex>

#include "common.cuh"
#include "kernels.h"
#include "../../include/bt_b200.h"

namespace bt {

namespace {

constexpr int kRows = 128;  // query rows of a block
constexpr int kKeys = 64;   // keys of a tile
constexpr int kHeadDim = 64;
constexpr int kQTile = kRows * kHeadDim * 2;   // 16 KiB
constexpr int kKvTile = kKeys * kHeadDim * 2;  // 8 KiB
constexpr int kThreads = 384;  // two groups of four softmax warps; loads, MMAs of either group; a warp that only makes the four whole
constexpr int kSlots = 4;  // items between the loader and the other roles
constexpr int kSeam = 32;  // keys of a box of the tile with the seam
constexpr float kOneBias = 1048576.0f;  // a bias that is one for many keys is kept out of their scores below this (log2 units)

struct WindowArgs {
  const __half *q, *k, *v;
  long long q_stride, k_stride, v_stride;
  __half* out;
  long long out_stride;
  const int *q_offsets, *k_offsets, *k_lens;
  int batch, heads, group;  // group: heads that share a key/value head
  int q_rows, k_rows, max_q, max_k;
  int left, right, sinks;  // left, right < 0: no bound
  float scale_log2e;
  const float* bias;  // [heads, bias_n]: distances -bias_left ..., the outermost values beyond
  int bias_n, bias_left;
  int* status;
  int take_over;  // the grid has more blocks than are resident
  int by_rows;    // the grid has blocks for as many items as offsets that rise can hold, which others may exceed
};

struct Item {
  int q_row, rows;     // first row of the tile in q and out, rows that exist; 0 rows: no more items
  int p0;              // position of the first
  int head;
  int k_row, k_len;    // the sequence's keys
  int number;          // see find_item
};

// The virtual keys of an item.
struct Keys {
  int ns;     // keys of the first run, a multiple of kSeam, or 0: the second run starts at key 0 or there are none
  int ws;     // first key of the second run
  int total;  // virtual keys
  int tiles;  // >= 1: an item that sees nothing walks one tile of masked keys
};
__device__ __forceinline__ Keys keys_of(const WindowArgs& a, const Item& it) {
  Keys k;
  const int last = it.p0 + it.rows - 1;
  const int hi = a.right < 0 ? it.k_len : min(it.k_len, last + a.right + 1);
  const int lo = a.left < 0 ? 0 : max(0, it.p0 - a.left);
  const int first = (max(min(a.sinks, hi), 0) + kSeam - 1) & ~(kSeam - 1);
  const bool apart = lo > first;
  k.ns = apart ? first : 0;
  k.ws = apart ? lo : 0;
  k.total = max(k.ns + hi - k.ws, 0);
  k.tiles = max(1, (k.total + kKeys - 1) / kKeys);
  return k;
}

// Item n = (sequence, query tile, head), heads fastest, a sequence's last tiles (which see most keys where nothing behind them is
// seen) first; called by whole warps, 32 sequences at a time.  A sequence whose
// offsets do not describe rows of the buffers is left out and reported.
__device__ __forceinline__ bool find_item(const WindowArgs& a, int n, int& cur_b, int& cur_first, Item& it) {
  const int lane = static_cast<int>(threadIdx.x & 31u);
  if (n < cur_first) cur_b = cur_first = 0;
  while (cur_b < a.batch) {
    const int b = cur_b + lane;
    int start = 0, len = 0, k_row = 0, k_len = 0;
    if (b < a.batch) {
      start = __ldg(a.q_offsets + b);
      len = __ldg(a.q_offsets + b + 1) - start;
      k_row = __ldg(a.k_offsets + b);
      const int room = __ldg(a.k_offsets + b + 1) - k_row;
      k_len = a.k_lens != nullptr ? __ldg(a.k_lens + b) : room;
      if (start < 0 || len < 0 || len > a.max_q || start > a.q_rows - len || k_row < 0 || k_len < 0 || k_len > a.max_k ||
          k_len > room || k_row > a.k_rows - room) {
        if (a.status != nullptr) atomicCAS(a.status, 0, kStatusBadOffsets);
        len = 0;
      }
    }
    const int items = ((len + kRows - 1) / kRows) * a.heads;
    int incl = items;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += up;
    }
    const unsigned found = __ballot_sync(0xffffffffu, b < a.batch && n < cur_first + incl);
    if (found != 0u) {
      const int src = __ffs(found) - 1;
      start = __shfl_sync(0xffffffffu, start, src);
      len = __shfl_sync(0xffffffffu, len, src);
      it.k_row = uniform_int(__shfl_sync(0xffffffffu, k_row, src));
      it.k_len = uniform_int(__shfl_sync(0xffffffffu, k_len, src));
      cur_first += __shfl_sync(0xffffffffu, incl - items, src);
      cur_b += src;
      const int r = n - cur_first;
      const int from_end = r / a.heads, qt = (len - 1) / kRows - from_end;
      if (from_end < 0 || qt < 0) break;  // (offsets so wrong that the count of items passed 32 bits)
      it.head = uniform_int(r - from_end * a.heads);
      it.q_row = uniform_int(start + qt * kRows);
      it.rows = uniform_int(min(kRows, len - qt * kRows));
      it.p0 = uniform_int(qt * kRows + it.k_len - len);
      return true;
    }
    cur_first += __shfl_sync(0xffffffffu, incl, 31);
    cur_b += 32;
  }
  it.rows = 0;
  return false;
}

// Wait of the roles that one warp walks: between polls it sleeps, the softmax warps need the issue slots.
__device__ __forceinline__ bool wait_role(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const long long t0 = clock64();
  uint32_t polls = 0;
  while (true) {
    __nanosleep(40);
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((++polls & 63u) == 0u) {
      if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
      if (__any_sync(0xffffffffu, clock64() - t0 > (1ll << 31))) {
        *abort_flag = 1;
        if (status != nullptr) atomicCAS(status, 0, code);
        return false;
      }
    }
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A bias in log2 units.  The type's lowest value stays a number (a row that sees only such keys weighs them alike, as the
// formula says), an infinity one (a key at such a distance is not seen).
__device__ __forceinline__ float bias_log2(float b) {
  const float x = b * 1.4426950408889634f;
  return fabsf(b) < INFINITY ? fminf(fmaxf(x, -FLT_MAX), FLT_MAX) : x;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// S = Q K^T of a 128 x 64 tile and the commit to `bar`; called by a whole warp.
__device__ __forceinline__ void mma_scores(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint64_t* bar) {
  asm volatile(
      "{\n\t"
      ".reg .pred q, f, t;\n\t"
      ".reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "add.u64 a1, %1, 2;\n\t"
      "add.u64 a2, %1, 4;\n\t"
      "add.u64 a3, %1, 6;\n\t"
      "add.u64 b1, %2, 2;\n\t"
      "add.u64 b2, %2, 4;\n\t"
      "add.u64 b3, %2, 6;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.u32 f, 0, 0;\n\t"
      "setp.eq.u32 t, 0, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, f;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(smem_u32(bar))
      : "memory");
}
// O (+)= P V over the first `steps` <= 4 groups of 16 keys, P from tensor memory; called by a whole warp.
__device__ __forceinline__ void mma_values(uint32_t d_tmem, uint32_t p_tmem, uint64_t vdesc, uint32_t idesc, uint32_t accumulate,
                                           uint32_t steps) {
  asm volatile(
      "{\n\t"
      ".reg .pred q, p, t;\n\t"
      ".reg .b64 b;\n\t"
      ".reg .b32 a;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.u32 p, %4, 0;\n\t"
      "setp.eq.u32 t, 0, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
#define BT_STEP(I, A, B)                        \
  "add.u32 a, %1, " A ";\n\t"                   \
  "add.u64 b, %2, " B ";\n\t"                   \
  "setp.gt.and.u32 p, %5, " I ", q;\n\t"        \
  "@p tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
      BT_STEP("1", "8", "128") BT_STEP("2", "16", "256") BT_STEP("3", "24", "384")
#undef BT_STEP
      "}\n" ::"r"(d_tmem),
      "r"(p_tmem), "l"(vdesc), "r"(idesc), "r"(accumulate), "r"(steps)
      : "memory");
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int N>
struct Int {
  static constexpr int value = N;
};

// `t` grows to the largest magnitude of the halves of w, NaN above all.
__device__ __forceinline__ void watch(__half2& t, uint32_t w) {
  t = __hmax2_nan(__habs2(*reinterpret_cast<const __half2*>(&w)), t);
}
__device__ __forceinline__ void watch_row(__half2& t, const __half* row) {
#pragma unroll 4
  for (int x = 0; x < kHeadDim; x += 8) {
    const uint4 w = *reinterpret_cast<const uint4*>(row + x);
    watch(t, w.x);
    watch(t, w.y);
    watch(t, w.z);
    watch(t, w.w);
  }
}
__device__ __forceinline__ bool not_finite(__half2 t) { return !(__low2float(t) < INFINITY) || !(__high2float(t) < INFINITY); }
// Where values of keys that a row does not see are infinities or NaN, a product with their weights of zero leaves NaN in the row.
// And where scores are so large (from 2^24 on) that a reference in single precision is off by whole steps of the exponent, weights may pass fp16's
// range.  A row that came out so is looked at again, by a whole warp: if any key or value that it does not see, of those that its item
// multiplied, holds such a number, or nothing that it does see, the row is done anew over the keys that it sees alone.  Slow (32 keys at a time, without
// matrix instructions: 190 us for a row of 2,047 keys, 560 before eight loads went at a time), but nothing with finite inputs and scores below
// 10^7 comes here.
template <bool BIAS>
__device__ __forceinline__ void redo_row(const WindowArgs& a, const Keys& keys, const Item& it, int i, int head) {
  const int lane = static_cast<int>(threadIdx.x & 31u);
  const int p = it.p0 + i, kv = head / a.group;
  const int hi = a.right < 0 ? it.k_len : min(it.k_len, p + a.right + 1);
  const int a_hi = a.left < 0 ? 0 : min(a.sinks, hi), lo = a.left < 0 ? 0 : p - a.left;
  const float* table = BIAS ? a.bias + static_cast<long long>(head) * a.bias_n : nullptr;
  auto key_of = [&](int u) { return u < keys.ns ? u : keys.ws + u - keys.ns; };
  auto bias_of = [&](int u) {
    return BIAS ? bias_log2(__ldg(table + min(max(key_of(u) - p + a.bias_left, 0), a.bias_n - 1))) : 0.f;
  };
  auto seen = [&](int u) {
    const int key = key_of(u);
    return u < keys.total && key < hi && (key >= lo || key < a_hi) && bias_of(u) != -INFINITY;
  };
  auto row_of = [&](const __half* base, long long stride, int u) {
    return base + (static_cast<long long>(it.k_row) + key_of(u)) * stride + kv * kHeadDim;
  };
  const __half* q = a.q + static_cast<long long>(it.q_row + i) * a.q_stride + head * kHeadDim;
  auto not_finite_among = [&](bool what_it_sees) {
    bool found = false;
#pragma unroll 1
    for (int u = lane; u - lane < keys.total && !found; u += 32) {
      __half2 t = __half2half2(__ushort_as_half(0));
      if (u < keys.total && seen(u) == what_it_sees) {
        watch_row(t, row_of(a.k, a.k_stride, u));
        watch_row(t, row_of(a.v, a.v_stride, u));
      }
      found = __any_sync(0xffffffffu, not_finite(t));
    }
    return found;
  };
  if (!not_finite_among(false)) {
    __half2 t = __half2half2(__ushort_as_half(0));
    watch_row(t, q);
    if (__any_sync(0xffffffffu, not_finite(t)) || not_finite_among(true)) return;
  }
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;  // dimensions 2 lane, 2 lane + 1
#pragma unroll 1
  for (int u0 = 0; u0 < keys.total; u0 += 32) {
    const int u = u0 + lane;
    const bool mine = seen(u);
    unsigned left = __ballot_sync(0xffffffffu, mine);
    if (left == 0u) continue;
    float s = -INFINITY;
    if (mine) {
      const __half* k = row_of(a.k, a.k_stride, u);
      float dot = 0.f;
#pragma unroll 4
      for (int x = 0; x < kHeadDim; x += 8) {
        const uint4 qw = *reinterpret_cast<const uint4*>(q + x), kw = *reinterpret_cast<const uint4*>(k + x);
        const uint32_t qs[4] = {qw.x, qw.y, qw.z, qw.w}, ks[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float2 qf = __half22float2(*reinterpret_cast<const __half2*>(&qs[y]));
          const float2 kf = __half22float2(*reinterpret_cast<const __half2*>(&ks[y]));
          dot = fmaf(qf.x, kf.x, fmaf(qf.y, kf.y, dot));
        }
      }
      s = fmaf(dot, a.scale_log2e, bias_of(u));
    }
    float top = s;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float m_new = fmaxf(m, top);
    const float f = m_new == m ? 1.0f : ex2(m - m_new);
    m = m_new;
    const float w = mine ? ex2(s - (m == -INFINITY ? 0.f : m)) : 0.f;
    l = fmaf(l, f, w);
    o0 *= f;
    o1 *= f;
#pragma unroll 1
    for (int t0 = 0; t0 < 32; t0 += 8, left >>= 8) {  // (eight loads under way at a time)
      if ((left & 0xffu) == 0u) continue;
      uint32_t v[8];
#pragma unroll
      for (int t = 0; t < 8; ++t)
        v[t] = (left >> t) & 1u ? *reinterpret_cast<const uint32_t*>(row_of(a.v, a.v_stride, u0 + t0 + t) + 2 * lane) : 0u;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float wt = __shfl_sync(0xffffffffu, w, t0 + t);  // (0 where the key is not seen)
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[t]));
        o0 = fmaf(wt, f.x, o0);
        o1 = fmaf(wt, f.y, o1);
      }
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  __syncwarp();  // behind what the warp has written there
  *reinterpret_cast<uint32_t*>(a.out + static_cast<long long>(it.q_row + i) * a.out_stride + head * kHeadDim + 2 * lane) =
      pack_half2(o0 * inv, o1 * inv);
}
// Bits lo .. hi - 1 of a word.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  const uint32_t below_hi = hi >= 32 ? 0xffffffffu : (hi > 0 ? (1u << hi) - 1u : 0u);
  const uint32_t below_lo = lo >= 32 ? 0xffffffffu : (lo > 0 ? (1u << lo) - 1u : 0u);
  return below_hi & ~below_lo;
}

// The bias of a tile for a warp's rows: value of (column c of half h, lane l) at 64 h + c - l + 31, in log2 units.  Two copies, one an
// element further on, so that a lane reads its row's values two at a time wherever they start; the pitch keeps the copies
// that neighbouring lanes read in different banks.
struct BiasSlice {
  float copy[2][144];
};

// Items in which a softmax warp has found rows that are not finite, looked at again when the block has no more items (in the
// loop they would cost it the registers).  A warp with kMany of them asks the loader to take over no more blocks, which
// then start as others end: it meets four more at most, but for items that only offsets that fall bring (their rows
// beyond the list's end stay as they are).
struct Again {
  static constexpr int kMany = 5, kSize = 10;
  int current, count, item[kSize];
};

struct Layout {
  static constexpr int kStages = 2;  // Q tiles; K and V tiles for each group
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kStages * kQTile;
  static constexpr int kV = kK + 2 * kStages * kKvTile;
  // For each of the eight warps: the bias of the tile that it is at, then its reference and sums for the other group; or
  // 32 output rows of 64 bytes
  static constexpr int kOwn = kV + 2 * kStages * kKvTile;
  static constexpr int kOwnBytes = 32 * 64;
  static constexpr int kOwnSums = sizeof(BiasSlice);
  static constexpr int kBar = kOwn + 8 * kOwnBytes;
  static constexpr int kBytes = kBar + 1024;
  static_assert(kOwnSums % 8 == 0 && kOwnSums + 32 * 8 <= kOwnBytes, "a warp's own bytes");
};

template <bool BIAS>
__global__ void __launch_bounds__(kThreads, 2)
window_mha_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_k_seam,
                  const __grid_constant__ CUtensorMap tm_v_seam, const WindowArgs args) {
  using L = Layout;
  constexpr int kStages = L::kStages, kQStages = L::kStages;
  constexpr int kLoadTimeout = kStatusMhaLoadTimeout, kMmaTimeout = kStatusMhaMmaTimeout, kSoftmaxTimeout = kStatusMhaSoftmaxTimeout;
  extern __shared__ __align__(1024) uint8_t smem[];

  pdl_launch_dependents();
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* q_full = bars;                    // [2] by item
  uint64_t* q_empty = bars + 2;               // [2] both groups' last products with Q
  uint64_t* k_full = bars + 4;                // [group][kStages] by the group's tiles
  uint64_t* k_empty = bars + 8;
  uint64_t* v_full = bars + 12;
  uint64_t* v_empty = bars + 16;
  uint64_t* s_full = bars + 20;               // [group] S is there, and the P V before it has retired
  uint64_t* p_full = bars + 22;               // [group] P is there, V rows blanked
  uint64_t* o_done = bars + 24;               // [group] the item's last P V has retired
  uint64_t* merge_full = bars + 26;           // [group][warp] this group's O, reference and sum may be read by the other group
  uint64_t* merge_empty = bars + 34;          // [group][warp] they have been
  uint64_t* item_full = bars + 42;            // [kSlots]
  uint64_t* item_empty = bars + 46;           // [kSlots]
  uint64_t* taken_full = bars + 50;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 51);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* enough = abort_flag + 1;  // no more blocks are to be taken over
  uint8_t* taken = smem + L::kBar + 480;       // 16 bytes
  Item* items = reinterpret_cast<Item*>(smem + L::kBar + 496);
  Again* again_all = reinterpret_cast<Again*>(smem + L::kBar + 496 + kSlots * sizeof(Item));
  static_assert(496 + kSlots * sizeof(Item) + 8 * sizeof(Again) <= 1024, "barriers, items and what is looked at again");

  const int warp = uniform_int(static_cast<int>(threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  const bool smem_ok = (smem_u32(smem) & 1023u) == 0u;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 2);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&o_done[s], 1);
    }
    for (int s = 0; s < 2 * kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 8; ++s) {
      mbar_init(&merge_full[s], 1);
      mbar_init(&merge_empty[s], 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], 10);
    }
    mbar_init(taken_full, 1);
    *abort_flag = smem_ok ? 0 : 1;
    *enough = 0;
    for (int s = 0; s < 8; ++s) {
      again_all[s].current = static_cast<int>(blockIdx.x);
      again_all[s].count = 0;
    }
    fence_mbar_init();
    if (!smem_ok && args.status != nullptr) atomicCAS(args.status, 0, kLoadTimeout + 0x10);
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = uniform_u32(*tmem_slot);
  pdl_wait();
  // tensor memory of group g: S (and P over it) at 64 g, O at 128 + 64 g

  // Each role finds the block's own item by itself; the n-th taken over comes through slot n % kSlots.
  Item it;
  auto own_item = [&]() {
    int b = 0, f = 0;
    return find_item(args, static_cast<int>(blockIdx.x), b, f, it);
  };
  auto parity = [](uint32_t n) { return (n / kSlots) & 1u; };
  auto read_item = [&](uint32_t n) {  // (once item_full has completed)
    const Item* s = &items[n % kSlots];
    it.q_row = uniform_int(s->q_row);
    it.rows = uniform_int(s->rows);
    it.p0 = uniform_int(s->p0);
    it.head = uniform_int(s->head);
    it.k_row = uniform_int(s->k_row);
    it.k_len = uniform_int(s->k_len);
    __syncwarp();
    if (lane == 0) {
      if (warp < 8) again_all[warp].current = s->number;
      mbar_arrive(&item_empty[n % kSlots]);
    }
  };
  // Tile j of item n belongs to group (j + n) & 1, so the group that had one tile more has one less next time.

  if (warp >= 8) {
    regs_dec<32>();
    if (!smem_ok) {
      // straight to the teardown
    } else if (warp == 8) {
      // ------------------------------------------------------------------ loads
      int cur_b = 0, cur_first = 0;
      bool have = find_item(args, static_cast<int>(blockIdx.x), cur_b, cur_first, it);
      uint32_t asked = 0;
      int cur_number = 0;
      int beyond = args.by_rows && blockIdx.x == 0 ? static_cast<int>(gridDim.x) : -1;
      // The next block that has not started, or, behind the last one, items that the grid's bound did not foresee: offsets
      // that fall can hold more than it does, so the first block's CTA looks there once (which reports such offsets too).
      auto take_next = [&]() {
        have = false;
        if (args.take_over && asked != 0xffffffffu) {
          while (__any_sync(0xffffffffu, *enough == 0)) {
            if (elect_one()) launch_control_ask(taken, taken_full);
            if (!wait_role(taken_full, asked & 1u, abort_flag, args.status, kLoadTimeout)) return;
            ++asked;
            const int block = uniform_int(launch_control_answer(taken));
            if (block < 0) break;
            have = find_item(args, cur_number = block, cur_b, cur_first, it);
            if (have) return;
          }
          asked = 0xffffffffu;
        }
        if (beyond >= 0) have = find_item(args, cur_number = beyond++, cur_b, cur_first, it);
        if (!have) beyond = -1;
      };
      uint32_t count[2] = {0, 0};  // tiles of the groups so far
      bool ok = true;
      for (uint32_t n = 0; have; ++n) {
        const Keys keys = keys_of(args, it);
        const int qb = static_cast<int>(n % kQStages);
        const int kv_col = it.head / args.group * kHeadDim;
        ok = wait_role(&q_empty[qb], ((n / kQStages) & 1u) ^ 1u, abort_flag, args.status, kLoadTimeout);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&q_full[qb], kQTile);
          tma_load_2d(smem + L::kQ + qb * kQTile, &tm_q, &q_full[qb], it.head * kHeadDim, it.q_row);
        }
        for (int j = 0; j < keys.tiles; ++j) {
          const int g = (j + static_cast<int>(n)) & 1;
          const uint32_t cnt = g ? count[1]++ : count[0]++;
          const int slot = g * kStages + static_cast<int>(cnt % kStages);
          const uint32_t phase = (cnt / kStages) & 1u;
          const int u0 = j * kKeys;
          const bool seam = u0 < keys.ns && u0 + kKeys > keys.ns;
          const int row = it.k_row + (u0 < keys.ns ? u0 : keys.ws + u0 - keys.ns);
          auto fetch = [&](uint8_t* dst, const CUtensorMap* whole, const CUtensorMap* box, uint64_t* bar) {
            mbar_arrive_expect_tx(bar, kKvTile);
            if (!seam) {
              tma_load_2d(dst, whole, bar, kv_col, row);
            } else {
              for (int s = 0; s < kKeys; s += kSeam) {
                const int u = u0 + s;
                tma_load_2d(dst + s * 128, box, bar, kv_col, it.k_row + (u < keys.ns ? u : keys.ws + u - keys.ns));
              }
            }
          };
          ok = wait_role(&k_empty[slot], phase ^ 1u, abort_flag, args.status, kLoadTimeout);
          if (!ok) break;
          if (elect_one()) fetch(smem + L::kK + slot * kKvTile, &tm_k, &tm_k_seam, &k_full[slot]);
          __syncwarp();
          ok = wait_role(&v_empty[slot], phase ^ 1u, abort_flag, args.status, kLoadTimeout);
          if (!ok) break;
          if (elect_one()) fetch(smem + L::kV + slot * kKvTile, &tm_v, &tm_v_seam, &v_full[slot]);
          __syncwarp();
        }
        if (!ok) break;
        take_next();
        const uint32_t slot = n % kSlots;
        if (!wait_role(&item_empty[slot], parity(n) ^ 1u, abort_flag, args.status, kLoadTimeout)) break;
        if (lane == 0) {
          Item w = it;
          if (!have) w.rows = 0;
          w.number = cur_number;
          items[slot] = w;
          mbar_arrive(&item_full[slot]);
        }
        __syncwarp();
      }
    } else if (warp <= 10) {
      // -------------------------------------------------------------- MMA issue, warp 9 + g for group g
      constexpr uint64_t kDescK = make_smem_desc_hi(16, 1024);
      constexpr uint64_t kDescV = make_smem_desc_hi(kKvTile, 1024);
      constexpr uint32_t kIdescS = make_idesc_f16(128, kKeys, 0, 0);
      constexpr uint32_t kIdescO = make_idesc_f16(128, kHeadDim, 0, 1);
      const int g = warp - 9;
      const uint32_t t_s = tmem_base + 64u * g, t_o = tmem_base + 128u + 64u * g;
      const uint32_t s_q = smem_u32(smem + L::kQ);
      const uint32_t s_k = smem_u32(smem + L::kK + g * kStages * kKvTile), s_v = smem_u32(smem + L::kV + g * kStages * kKvTile);
      uint64_t *kf = k_full + g * kStages, *ke = k_empty + g * kStages, *vf = v_full + g * kStages, *ve = v_empty + g * kStages;
      uint32_t cnt = 0;  // the group's tiles so far
      bool have = own_item();
      for (uint32_t n = 0; have; ++n) {
        const Keys keys = keys_of(args, it);
        const int first = (g + static_cast<int>(n)) & 1;  // the group's first tile
        if (!wait_role(&q_full[n % kQStages], (n / kQStages) & 1u, abort_flag, args.status, kMmaTimeout)) break;
        bool ok = true;
        // (an item's last product with Q lets go of it)
        auto issue_s = [&](uint32_t c, bool last) {
          if (!wait_role(&kf[c % kStages], (c / kStages) & 1u, abort_flag, args.status, kMmaTimeout)) return false;
          tc_fence_after();
          mma_scores(t_s, smem_desc(kDescK, s_q + (n % kQStages) * kQTile), smem_desc(kDescK, s_k + (c % kStages) * kKvTile), kIdescS,
                     &s_full[g]);
          if (elect_one()) umma_commit(&ke[c % kStages]);
          if (last && elect_one()) umma_commit(&q_empty[n % kQStages]);
          return true;
        };
        if (first < keys.tiles)
          ok = issue_s(cnt, first + 2 >= keys.tiles);
        else if (elect_one())
          umma_commit(&q_empty[n % kQStages]);
        for (int j = first; ok && j < keys.tiles; j += 2, ++cnt) {
          ok = mbar_wait_warp(&p_full[g], cnt & 1u, abort_flag, args.status, kMmaTimeout) &&
               wait_role(&vf[cnt % kStages], (cnt / kStages) & 1u, abort_flag, args.status, kMmaTimeout);
          if (!ok) break;
          tc_fence_after();
          const int valid = max(1, min(kKeys, keys.total - j * kKeys));
          mma_values(t_o, t_s, smem_desc(kDescV, s_v + (cnt % kStages) * kKvTile), kIdescO, j > first ? 1u : 0u,
                     static_cast<uint32_t>((valid + 15) >> 4));
          if (elect_one()) umma_commit(&ve[cnt % kStages]);
          if (j + 2 < keys.tiles)
            ok = issue_s(cnt + 1, j + 4 >= keys.tiles);
          else if (elect_one())
            umma_commit(&o_done[g]);
        }
        if (!ok) break;
        if (!wait_role(&item_full[n % kSlots], parity(n), abort_flag, args.status, kMmaTimeout)) break;
        read_item(n);
        have = it.rows > 0;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax (warps 0..3 and 4..7)
    regs_inc<104>();
    const int g = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // query row inside the tile == tensor-memory lane
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_s = t_lane + 64u * g, t_o = t_lane + 128u + 64u * g;
    const float c = args.scale_log2e;
    uint32_t cnt = 0;      // the group's tiles so far
    uint8_t* own = smem + L::kOwn + warp * L::kOwnBytes;
    uint32_t o_items[2] = {0, 0};            // items in which this group, the other one had tiles
    uint32_t handed = 0, received = 0;
    bool lent = false;                       // the other group may still be reading this one's O, reference and sum
    bool ok = true;
    auto take_back = [&]() {
      if (lent && !mbar_wait_warp(&merge_empty[g * 4 + quarter], (handed - 1u) & 1u, abort_flag, args.status, kSoftmaxTimeout)) ok = false;
      lent = false;
    };
    // The end of an item.  The group of the odd tiles says what its reference and sum are and goes on (its next product waits
    // until its O has been read, see take_back).
    auto hand_over = [&](float m, float l) {
      reinterpret_cast<float2*>(own + L::kOwnSums)[lane] = make_float2(m, l);
      __syncwarp();
      if (lane == 0) mbar_arrive(&merge_full[g * 4 + quarter]);
      lent = true;
      ++handed;
    };
    auto merge = [&](float m, float l, bool both, __half2& bad) {
      // the group of the even ones puts the two together: O / row sum -> fp16 -> this warp's staging rows, half a row at a time
      // -> global memory, four threads to a half row
      const int other = (g ^ 1) * 4 + quarter;
      float2 theirs = make_float2(-INFINITY, 0.f);
      ok = mbar_wait_warp(&o_done[g], o_items[0] & 1u, abort_flag, args.status, kSoftmaxTimeout) && ok;
      if (both) {
        ok = mbar_wait_warp(&merge_full[other], received++ & 1u, abort_flag, args.status, kSoftmaxTimeout) && ok;
        ok = mbar_wait_warp(&o_done[g ^ 1], o_items[1] & 1u, abort_flag, args.status, kSoftmaxTimeout) && ok;
      }
      tc_fence_after();
      if (both) {
        theirs = reinterpret_cast<const float2*>(smem + L::kOwn + other * L::kOwnBytes + L::kOwnSums)[lane];
      }
      const float top = fmaxf(theirs.x, m);
      float f0 = m == -INFINITY ? 0.f : ex2(m - top);
      float f1 = theirs.x == -INFINITY ? 0.f : ex2(theirs.x - top);
      const float sum = fmaf(theirs.y, f1, l * f0);
      // A row that sees no key: zeros.  Any other has a key whose weight is 1 or more, but for references beyond 2^24 or so: their
      // rounding is in all of the row's weights alike, and where these leave fp16's range the sum says so, or the products are not
      // finite.  Such a row is done anew.
      const float inv = sum >= 0.5f ? 1.0f / sum : (top == -INFINITY && sum == 0.f ? 0.f : NAN);
      f0 *= inv;
      f1 *= inv;
      __half* out = args.out + static_cast<long long>(it.q_row + quarter * 32) * args.out_stride + it.head * kHeadDim + (lane & 3) * 8;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        // (O is finite where a row has seen nothing: its weights were zeros)
        uint32_t a[32];
        tmem_ld_32x32(t_o + 32 * h, a);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) a[i] = __float_as_uint(__uint_as_float(a[i]) * f0);
        if (both) {
          uint32_t b[32];
          tmem_ld_32x32(t_lane + 128u + 64u * (g ^ 1) + 32 * h, b);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) a[i] = __float_as_uint(fmaf(__uint_as_float(b[i]), f1, __uint_as_float(a[i])));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint4 w;
          w.x = pack_half2(__uint_as_float(a[u * 8]), __uint_as_float(a[u * 8 + 1]));
          w.y = pack_half2(__uint_as_float(a[u * 8 + 2]), __uint_as_float(a[u * 8 + 3]));
          w.z = pack_half2(__uint_as_float(a[u * 8 + 4]), __uint_as_float(a[u * 8 + 5]));
          w.w = pack_half2(__uint_as_float(a[u * 8 + 6]), __uint_as_float(a[u * 8 + 7]));
          watch(bad, w.x);
          watch(bad, w.y);
          watch(bad, w.z);
          watch(bad, w.w);
          *reinterpret_cast<uint4*>(own + lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4)) = w;
        }
        if (h == 1) tc_fence_before();
        __syncwarp();
        if (h == 1 && both && lane == 0) mbar_arrive(&merge_empty[other]);  // all of the other group's part has been read
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = 8 * k + (lane >> 2);
          const uint4 w = *reinterpret_cast<const uint4*>(own + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4));
          if (quarter * 32 + row < it.rows) *reinterpret_cast<uint4*>(out + row * args.out_stride + 32 * h) = w;
        }
        __syncwarp();
      }
    };
    bool have = smem_ok && own_item();
    for (uint32_t n = 0; have; ++n) {
      const Keys keys = keys_of(args, it);
      const int first = (g + static_cast<int>(n)) & 1;
      const bool exists = r < it.rows;
      const bool idle = quarter * 32 >= it.rows;  // no row of this warp exists
      // virtual keys that this row sees: [0, a_hi) and [b_lo, b_hi)
      const int p = it.p0 + r;
      const int hi = args.right < 0 ? it.k_len : min(it.k_len, p + args.right + 1);
      const int a_hi = args.left < 0 ? 0 : min(args.sinks, hi);
      const int b_lo = keys.ns + max((args.left < 0 ? 0 : p - args.left) - keys.ws, 0);
      const int b_hi = keys.ns + hi - keys.ws;
      // The exponent reference of a row may lag its maximum by 2^kLag (fp16 holds the weights up to there); beyond, the warp's
      // rows move theirs to their maxima and rescale O.  Rows that do not exist have no say, so results are a function of
      // the inputs alone.
      constexpr float kLag = 12.0f;
      float m_ref = -INFINITY, l_run = 0.f;
      for (int j = first; j < keys.tiles; j += 2, ++cnt) {
        const int u0 = j * kKeys;
        const int slot = g * kStages + static_cast<int>(cnt % kStages);
        // The bias, laid out while S is on its way: of a half, 63 values from that of (column 0, lane 31) on, at index `at`
        float one[2] = {0.f, 0.f};        // a half's bias where it is one for all its keys and rows
        bool several[2] = {false, false};
        if (BIAS && !idle) {
          const float* table = args.bias + static_cast<long long>(it.head) * args.bias_n;
          BiasSlice* slice = reinterpret_cast<BiasSlice*>(own);
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int u = u0 + 32 * h;
            const int at = (u < keys.ns ? u : keys.ws + u - keys.ns) - (it.p0 + quarter * 32 + 31) + args.bias_left;
            const float v0 = bias_log2(__ldg(table + min(max(at + lane, 0), args.bias_n - 1)));
            const float v1 = bias_log2(__ldg(table + min(max(at + 32 + lane, 0), args.bias_n - 1)));
            one[h] = v0;
            // One value for all need not be added to each score: it goes into the exponent's offset, less the reference.  That needs a
            // reference that is no coarser than the weights' range allows (below 2^20 it is rounded to 2^-4 at worst); beyond,
            // it would lose the scores (at 1e9 its steps are 128) and leave their weights without bound.  There the value is
            // added to each score, as where there are several, and the sum swallows the score for all alike.
            several[h] = !((at >= args.bias_n - 1 || at + 62 <= 0) && (fabsf(v0) < kOneBias || v0 == -INFINITY));
            slice->copy[0][64 * h + lane] = v0;
            slice->copy[0][64 * h + 32 + lane] = v1;
            if (lane > 0) slice->copy[1][64 * h + lane - 1] = v0;
            slice->copy[1][64 * h + 31 + lane] = v1;
          }
          __syncwarp();
        }
        mbar_wait_anyway_lane(&s_full[g], cnt & 1u, abort_flag, args.status, kSoftmaxTimeout);
        tc_fence_after();
        if (!idle) {
          const bool whole = __all_sync(0xffffffffu, !exists || (b_lo <= u0 && b_hi >= u0 + kKeys));
          uint32_t s[64];
          tmem_ld_32x32_at<0>(t_s, s);
          tmem_ld_32x32_at<32>(t_s + 32, s);
          tmem_ld_wait();
          float top = -INFINITY;              // largest score of the row, in log2 units
          float scale[2] = {c, c}, shift[2] = {0.f, 0.f};  // of what `s` holds of either half, to log2 units
          unsigned some = 3u;  // halves of the tile of which any row of the warp sees a key
          // scores of half CH: the bias added, masked keys out; the row's maximum
          auto fix = [&](auto half) {
            constexpr int B = decltype(half)::value * 32;
            if (BIAS) {
              constexpr int H = decltype(half)::value;
              if (several[H]) {
                scale[H] = 1.0f;
                const unsigned long long c2 = pack_f32x2(c, c);
                const float* from = &reinterpret_cast<const BiasSlice*>(own)->copy[(31 - lane) & 1][64 * H + ((31 - lane) & ~1)];
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  const float2 b = *reinterpret_cast<const float2*>(from + i);
                  float x0, x1;
                  unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[B + i]), __uint_as_float(s[B + i + 1])), c2, pack_f32x2(b.x, b.y)), x0, x1);
                  s[B + i] = __float_as_uint(x0);
                  s[B + i + 1] = __float_as_uint(x1);
                }
              } else {
                shift[H] = one[H];
              }
            }
            if (!whole) {
              const uint32_t w = bits_between(0, a_hi - u0 - B) | bits_between(b_lo - u0 - B, b_hi - u0 - B);
              if (!__any_sync(0xffffffffu, exists && w != 0u)) {
                some &= ~(1u << (B / 32));
                return;
              }
#pragma unroll
              for (int i = 0; i < 32; ++i) s[B + i] = ((w >> i) & 1u) ? s[B + i] : 0xff800000u;
            }
            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
            for (int i = B; i < B + 32; i += 4) {
              mx0 = max3(mx0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
              mx1 = max3(mx1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
            }
            top = fmaxf(top, BIAS ? fmaf(scale[B / 32], fmaxf(mx0, mx1), shift[B / 32]) : c * fmaxf(mx0, mx1));
          };
          fix(Int<0>());
          fix(Int<1>());
          const float m_new = fmaxf(m_ref, top);
          if (j == first) {
            m_ref = m_new;
          } else if (__any_sync(0xffffffffu, exists && m_new - m_ref > kLag)) {
            const float f = m_new == m_ref ? 1.0f : ex2(m_ref - m_new);
#pragma unroll 1
            for (int cb = 0; cb < kHeadDim; cb += 16) {
              uint32_t v[16];
              tmem_ld_32x16(t_o + cb, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
              tmem_st_32x16(t_o + cb, v);
            }
            l_run *= f;
            m_ref = m_new;
          }
          const float minus = m_ref == -INFINITY ? 0.f : -m_ref;  // (a row that has seen nothing yet keeps its masked scores at 2^-inf)
          unsigned long long l0 = 0ull, l1 = 0ull;  // pairs of zeros
          // weights of half CH: fp16 pairs over the scores, fp32 sums
          auto weigh = [&](auto half) {
            constexpr int B = decltype(half)::value * 32;
            uint32_t pk[16];
            if (some & (1u << (B / 32))) {
              const float mul = BIAS ? scale[B / 32] : c, add = BIAS ? shift[B / 32] + minus : minus;
              const unsigned long long sc2 = pack_f32x2(mul, mul), mi2 = pack_f32x2(add, add);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float t0, t1;
                unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[B + 2 * i]), __uint_as_float(s[B + 2 * i + 1])), sc2, mi2), t0, t1);
                t0 = ex2(t0);
                t1 = ex2(t1);
                if (i & 1) l1 = add_f32x2(l1, pack_f32x2(t0, t1)); else l0 = add_f32x2(l0, pack_f32x2(t0, t1));
                pk[i] = pack_half2(t0, t1);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = 0u;
            }
            tmem_st_32x16(t_s + B / 2, pk);
          };
          weigh(Int<0>());
          weigh(Int<1>());
          float la, lb;
          unpack_f32x2(add_f32x2(l0, l1), la, lb);
          l_run += la + lb;
        }
        const int valid = min(kKeys, keys.total - u0);
        if (valid < kKeys) {
          // blank the V rows behind the last key (as far as they are multiplied): they may be anybody's
          mbar_wait_anyway_lane(&v_full[slot], (cnt / kStages) & 1u, abort_flag, args.status, kSoftmaxTimeout);
          if (r >= valid && r < max(16, (valid + 15) & ~15)) {
            uint4* vr = reinterpret_cast<uint4*>(smem + L::kV + slot * kKvTile + r * 128);
#pragma unroll
            for (int i = 0; i < 8; ++i) vr[i] = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        tmem_st_wait();
        if (j == first) take_back();  // the product of an item's first tile overwrites O
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
      }
      const bool both = keys.tiles > 1;
      if (first == 0) {
        __half2 bad = __half2half2(__ushort_as_half(0));
        merge(m_ref, l_run, both, bad);
        if (__any_sync(0xffffffffu, exists && not_finite(bad)) && lane == 0) {
          Again& mine = again_all[warp];
          if (mine.count < Again::kSize) mine.item[mine.count++] = mine.current;
          if (mine.count >= Again::kMany) *enough = 1;
        }
      } else if (both)
        hand_over(m_ref, l_run);
      o_items[0] += first < keys.tiles ? 1u : 0u;
      o_items[1] += 1 - first < keys.tiles ? 1u : 0u;
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (!mbar_wait_warp(&item_full[n % kSlots], parity(n), abort_flag, args.status, kSoftmaxTimeout)) break;
      read_item(n);
      have = it.rows > 0;
    }
    tc_fence_before();
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < again_all[warp].count; ++i) {
      int b = 0, f = 0;
      find_item(args, again_all[warp].item[i], b, f, it);
      const Keys keys = keys_of(args, it);
      __half2 bad = __half2half2(__ushort_as_half(0));
      if (r < it.rows) watch_row(bad, args.out + static_cast<long long>(it.q_row + r) * args.out_stride + it.head * kHeadDim);
      unsigned rows = __ballot_sync(0xffffffffu, not_finite(bad));
      for (; rows != 0u; rows &= rows - 1u) redo_row<BIAS>(args, keys, it, quarter * 32 + __ffs(rows) - 1, it.head);
    }
  }

  __syncthreads();
  if (*abort_flag != 0) {  // copies in flight land before the block's memory goes to another
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

template <bool BIAS>
cudaError_t launch_window(const CUtensorMap (&tm)[5], WindowArgs a, int sms, cudaStream_t stream) {
  auto kern = window_mha_kernel<BIAS>;
  // A block per item, by an upper bound: tiles of sequences of max_q queries, or of sequences that share q_rows rows
  long long tiles = static_cast<long long>(a.batch) * ((a.max_q + kRows - 1) / kRows);
  const long long by_rows = (a.q_rows + static_cast<long long>(a.batch) * (kRows - 1)) / kRows;
  a.by_rows = tiles > by_rows ? 1 : 0;
  if (a.by_rows) tiles = by_rows;
  const long long grid = tiles * a.heads;
  if (grid > 0x7fffffffLL - 0x10000) return cudaErrorInvalidValue;
  a.take_over = grid > 2LL * sms ? 1 : 0;
  return launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(kThreads), Layout::kBytes, stream, tm[0], tm[1], tm[2], tm[3],
                    tm[4], a);
}

// -------------------------------------------------------------------------------------------- few queries
// The queries of a sequence times the heads that share a key/value head are at most 16 rows: what a step of generation
// asks for.  The keys are read once and that is the time it takes, so a CTA belongs to a (sequence, key/value head, range of
// its virtual keys) and all rows that need them; each of its four warps walks every fourth 32 keys with a softmax of its
// own, on mma.sync (16 x 8 x 16: a tcgen05 tile would be one eighth full at best).  A warp has a ring of its own of 32 keys and
// values, fetched by TMA a step ahead; no warp waits for another before the range ends.  Bound by HBM: 32 sequences of 8192 keys, 32 heads
// over 8, 81.7 us (6.6 TB/s); 64 of 4100 keys, 16 heads over 4, 44.2 us (with loads straight into the operands' registers 98 and 55;
// 45.0 with the look at rows that are not finite, with the bias 64.4).
// Rings of 2 stages and three CTAs to an SM, 3 and two, 4 and one, of the latter 44.2 / 46.2 / 68.2 us.
constexpr int kFewRows = 16;
constexpr int kFewWarps = 4;
constexpr int kFewKeys = 32;  // of a step
constexpr int kFewCluster = 8;  // ranges that a cluster holds
constexpr int kFewStages = 2;   // of a warp's ring
constexpr int kFewCtas = 3;     // to an SM
constexpr int kFewTile = kFewKeys * kHeadDim * 2;  // 4 KiB of K, and of V
constexpr int kFewRing = kFewStages * 2 * kFewTile;
constexpr int kFewSmemBytes = kFewWarps * kFewRing;
static_assert(kFewKeys == kSeam, "a step's keys are neighbours, also at the seam");

struct FewArgs {
  WindowArgs w;
  int splits;
  int cluster;  // the ranges of an item are a cluster, which puts them together itself; else they are left in `partial_*`
  float* partial_o;  // [batch, kv_heads, splits, 16, 64]
  float2* partial_ml;  // [batch, kv_heads, splits, 16]: reference and sum
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four 8 x 8 matrices of 16-byte rows, lane l giving the address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Every thread of every CTA of the cluster: what was written to shared memory before is visible to all after.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 16 (8) bytes at the place of `p` in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ float4 load_of(const float* p, int rank) {
  float4 v;
  asm volatile(
      "{\n\t"
      ".reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t"
      "}\n"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(smem_u32(p)), "r"(rank)
      : "memory");
  return v;
}
__device__ __forceinline__ float2 load_of(const float2* p, int rank) {
  float2 v;
  asm volatile(
      "{\n\t"
      ".reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %2, %3;\n\t"
      "ld.shared::cluster.v2.f32 {%0, %1}, [a];\n\t"
      "}\n"
      : "=f"(v.x), "=f"(v.y)
      : "r"(smem_u32(p)), "r"(rank)
      : "memory");
  return v;
}

// A range (reference, sum) of whose keys the row sees none.  Scores that are NaN leave the reference alone, and a sum that is not 0.
__device__ __forceinline__ bool saw_nothing(float2 ml) { return ml.x == -INFINITY && ml.y == 0.f; }

// The sequence of a CTA: rows of its queries, position of the first, its keys.  false: nothing to do.
__device__ __forceinline__ bool few_item(const WindowArgs& a, int b, Item& it) {
  const int start = a.q_offsets[b], len = a.q_offsets[b + 1] - start;
  const int k_row = a.k_offsets[b], room = a.k_offsets[b + 1] - k_row;
  const int k_len = a.k_lens != nullptr ? a.k_lens[b] : room;
  if (start < 0 || len < 0 || len > a.max_q || start > a.q_rows - len || k_row < 0 || k_len < 0 || k_len > a.max_k || k_len > room ||
      k_row > a.k_rows - room) {
    if (threadIdx.x == 0 && a.status != nullptr) atomicCAS(a.status, 0, kStatusBadOffsets);
    return false;
  }
  it.q_row = start;
  it.rows = len;
  it.p0 = k_len - len;
  it.k_row = k_row;
  it.k_len = k_len;
  return len > 0;
}

template <bool BIAS>
__global__ void __launch_bounds__(kFewWarps * 32, kFewCtas)
window_few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ FewArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t bars[kFewWarps][kFewStages];
  __shared__ float2 ml_all[kFewWarps][kFewRows], ml_cta[kFewRows];
  __shared__ int abort_word;
  // the warps' results, where their rings were
  auto& o_all = *reinterpret_cast<float(*)[kFewWarps][kFewRows][kHeadDim + 4]>(smem);
  static_assert(sizeof(o_all) <= kFewWarps * kFewRing, "the results fit");
  pdl_launch_dependents();
  const WindowArgs& w = a.w;
  const int warp = uniform_int(static_cast<int>(threadIdx.x >> 5)), lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, kv = blockIdx.y, b = blockIdx.z;
  const bool smem_ok = (smem_u32(smem) & 1023u) == 0u;
  volatile int* abort_flag = &abort_word;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kFewWarps * kFewStages; ++i) mbar_init(&bars[0][0] + i, 1);
    abort_word = smem_ok ? 0 : 1;
    fence_mbar_init();
    if (!smem_ok && w.status != nullptr) atomicCAS(w.status, 0, kStatusMhaLoadTimeout + 0x10);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  __syncthreads();
  pdl_wait();
  Item it;
  if (!few_item(w, b, it)) return;
  const Keys keys = keys_of(w, it);
  const int rows = it.rows * w.group;
  // virtual keys between the first tokens and the window that none of the rows sees: of one step
  const int hole_lo = min(w.sinks, keys.total), hole_hi = w.left < 0 ? 0 : keys.ns > 0 ? keys.ns : max(0, it.p0 - w.left) - keys.ws;
  // this CTA's virtual keys, in whole steps
  const int steps = (keys.total + kFewKeys - 1) / kFewKeys;
  const int first = static_cast<int>(static_cast<long long>(steps) * split / a.splits);
  const int last = static_cast<int>(static_cast<long long>(steps) * (split + 1) / a.splits);

  uint8_t* ring = smem + warp * kFewRing;
  auto fetch = [&](int step, int stage) {
    const int u0 = step * kFewKeys;
    const int row = it.k_row + (u0 < keys.ns ? u0 : keys.ws + u0 - keys.ns);
    if (elect_one()) {
      uint8_t* dst = ring + stage * 2 * kFewTile;
      mbar_arrive_expect_tx(&bars[warp][stage], 2 * kFewTile);
      tma_load_2d(dst, &tm_k, &bars[warp][stage], kv * kHeadDim, row);
      tma_load_2d(dst + kFewTile, &tm_v, &bars[warp][stage], kv * kHeadDim, row);
    }
    __syncwarp();
  };
  if (smem_ok) {
#pragma unroll
    for (int i = 0; i < kFewStages; ++i)
      if (first + warp + i * kFewWarps < last) fetch(first + warp + i * kFewWarps, i);
  }
  // Queries: row r is query r / group, head r % group
  uint32_t qa[4][4];  // [16 dimensions][register]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    const __half* p = w.q + static_cast<long long>(it.q_row + r / w.group) * w.q_stride + (kv * w.group + r % w.group) * kHeadDim + 2 * c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qa[i][h] = r < rows ? *reinterpret_cast<const uint32_t*>(p + 16 * i) : 0u;
      qa[i][2 + h] = r < rows ? *reinterpret_cast<const uint32_t*>(p + 16 * i + 8) : 0u;
    }
  }
  // virtual keys that the thread's two rows see: [0, a_hi) and [b_lo, b_hi); their bias rows
  int a_hi[2], b_lo[2], b_hi[2], pos[2];
  const float* bias[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = min(g + 8 * h, rows - 1);
    pos[h] = it.p0 + r / w.group;
    const int hi = w.right < 0 ? it.k_len : min(it.k_len, pos[h] + w.right + 1);
    a_hi[h] = w.left < 0 ? 0 : min(w.sinks, hi);
    b_lo[h] = keys.ns + max((w.left < 0 ? 0 : pos[h] - w.left) - keys.ws, 0);
    b_hi[h] = keys.ns + hi - keys.ws;
    bias[h] = BIAS ? w.bias + static_cast<long long>(kv * w.group + r % w.group) * w.bias_n : nullptr;
  }
  auto key_of = [&](int u) { return u < keys.ns ? u : keys.ws + u - keys.ns; };
  float o[8][4];
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[t][i] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int stage = 0;
  uint32_t phase = 0;
  bool ok = smem_ok;
#pragma unroll 1
  for (int step = first + warp; ok && step < last; step += kFewWarps) {
    const int u0 = step * kFewKeys;
    ok = mbar_wait_warp(&bars[warp][stage], phase, abort_flag, w.status, kStatusMhaLoadTimeout);
    if (!ok) break;
    uint8_t* tile = ring + stage * 2 * kFewTile;
    const uint32_t k_tile = smem_u32(tile), v_tile = k_tile + kFewTile;
    float s[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // keys 8 n .. (row lane % 8), 16-byte units 4 i + lane / 8 of their 128 swizzled bytes
        uint32_t k[4];
        load_matrices(k, k_tile + (8 * n + (lane & 7)) * 128 + (((4 * i + (lane >> 3)) ^ (lane & 7)) << 4));
        mma_16816(s[n], qa[2 * i][0], qa[2 * i][1], qa[2 * i][2], qa[2 * i][3], k[0], k[1]);
        mma_16816(s[n], qa[2 * i + 1][0], qa[2 * i + 1][1], qa[2 * i + 1][2], qa[2 * i + 1][3], k[2], k[3]);
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // row g + 8 (i / 2), key 8 n + 2 c + i % 2
        const int h = i >> 1, u = u0 + 8 * n + 2 * c + (i & 1);
        const bool seen = u < a_hi[h] || (u >= b_lo[h] && u < b_hi[h]);
        float x = s[n][i] * w.scale_log2e;
        if (BIAS) x += bias_log2(__ldg(bias[h] + min(max(key_of(u) - pos[h] + w.bias_left, 0), w.bias_n - 1)));
        s[n][i] = seen ? x : -INFINITY;
        top[h] = fmaxf(top[h], s[n][i]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      const float m_new = fmaxf(m[h], top[h]);
      const float f = m_new == m[h] ? 1.0f : ex2(m[h] - m_new);
      m[h] = m_new;
      l[h] *= f;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        o[t][2 * h] *= f;
        o[t][2 * h + 1] *= f;
      }
    }
    uint32_t p[4][2];  // [n][row half]
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float ref = m[h] == -INFINITY ? 0.f : m[h];
        const float p0 = ex2(s[n][2 * h] - ref), p1 = ex2(s[n][2 * h + 1] - ref);
        l[h] += p0 + p1;
        p[n][h] = pack_half2(p0, p1);
      }
    if (u0 + kFewKeys > keys.total || (u0 < hole_hi && hole_lo < hole_hi)) {
      // the values that no row sees: none (those behind the last key may be anybody's)
      const int u = u0 + lane;
      if (u >= keys.total || (u >= hole_lo && u < hole_hi)) {
        uint4* row = reinterpret_cast<uint4*>(tile + kFewTile + lane * 128);
#pragma unroll
        for (int i = 0; i < 8; ++i) row[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();  // ahead of the copy that fills this stage again
      __syncwarp();
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
#pragma unroll
      for (int t = 0; t < 8; t += 2) {  // keys 16 st .. and 16 st + 8 .. of the dimensions 8 t .., then 8 t + 8 ..
        const int key = 16 * st + (lane & 15);
        uint32_t v[4];
        load_matrices_transposed(v, v_tile + key * 128 + (((t + (lane >> 4)) ^ (key & 7)) << 4));
        mma_16816(o[t], p[2 * st][0], p[2 * st][1], p[2 * st + 1][0], p[2 * st + 1][1], v[0], v[1]);
        mma_16816(o[t + 1], p[2 * st][0], p[2 * st][1], p[2 * st + 1][0], p[2 * st + 1][1], v[2], v[3]);
      }
    }
    __syncwarp();  // the warp has read the tiles
    if (step + kFewStages * kFewWarps < last) fetch(step + kFewStages * kFewWarps, stage);
    if (++stage == kFewStages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  __syncthreads();  // all rings are read
  if (*abort_flag != 0) {  // copies in flight land before the block's memory goes to another
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  // The warps' results: O, reference and sum of each row
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (c == 0) ml_all[warp][g + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
    for (int t = 0; t < 8; ++t)
      *reinterpret_cast<float2*>(&o_all[warp][g + 8 * h][8 * t + 2 * c]) = make_float2(o[t][2 * h], o[t][2 * h + 1]);
  }
  __syncthreads();
  // eight columns of a row to a thread
  const int r = threadIdx.x >> 3, col = (threadIdx.x & 7) * 8;
  float top = -INFINITY, sum = 0.f, acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  if (r < rows) {
#pragma unroll
    for (int i = 0; i < kFewWarps; ++i) top = fmaxf(top, ml_all[i][r].x);
#pragma unroll
    for (int i = 0; i < kFewWarps; ++i) {
      const float2 ml = ml_all[i][r];
      if (saw_nothing(ml)) continue;
      const float f = ex2(ml.x - top);
      sum = fmaf(ml.y, f, sum);
#pragma unroll
      for (int x = 0; x < 8; ++x) acc[x] = fmaf(o_all[i][r][col + x], f, acc[x]);
    }
  }
  bool write = r < rows;
  if (a.cluster) {
    // each CTA's result in its shared memory; the rows go round the CTAs, a row's reads all of them
    float* mine = &o_all[0][r][col];  // (read by this thread alone)
#pragma unroll
    for (int x = 0; x < 8; ++x) mine[x] = acc[x];
    if (col == 0) ml_cta[r] = make_float2(top, sum);
    __syncwarp();
    cluster_sync();
    write = write && r % a.splits == split;
    if (write) {
      top = -INFINITY;
      for (int i = 0; i < a.splits; ++i) top = fmaxf(top, load_of(&ml_cta[r], i).x);
      sum = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x) acc[x] = 0.f;
      for (int i = 0; i < a.splits; ++i) {
        const float2 ml = load_of(&ml_cta[r], i);
        const float4 o0 = load_of(mine, i), o1 = load_of(mine + 4, i);
        if (saw_nothing(ml)) continue;
        const float f = ex2(ml.x - top);
        sum = fmaf(ml.y, f, sum);
        const float o[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] = fmaf(o[x], f, acc[x]);
      }
    }
    __syncwarp();
    cluster_sync();  // nobody's shared memory goes away while another reads it
  }
  if (a.splits == 1 || a.cluster) {
    __half2 bad = __half2half2(__ushort_as_half(0));
    if (write) {
      const float inv = sum != 0.f ? 1.0f / sum : 0.f;
      const uint4 out = make_uint4(pack_half2(acc[0] * inv, acc[1] * inv), pack_half2(acc[2] * inv, acc[3] * inv),
                                   pack_half2(acc[4] * inv, acc[5] * inv), pack_half2(acc[6] * inv, acc[7] * inv));
      *reinterpret_cast<uint4*>(w.out + static_cast<long long>(it.q_row + r / w.group) * w.out_stride +
                                (kv * w.group + r % w.group) * kHeadDim + col) = out;
      watch(bad, out.x);
      watch(bad, out.y);
      watch(bad, out.z);
      watch(bad, out.w);
    }
    const unsigned again = __ballot_sync(0xffffffffu, not_finite(bad));
    for (int i = 0; again != 0u && i < 4; ++i)
      if ((again >> (8 * i)) & 0xffu) redo_row<BIAS>(w, keys, it, (4 * warp + i) / w.group, kv * w.group + (4 * warp + i) % w.group);
  } else if (write) {
    const long long at = ((static_cast<long long>(b) * gridDim.y + kv) * a.splits + split) * kFewRows + r;
    if (col == 0) a.partial_ml[at] = make_float2(top, sum);
    float4* dst = reinterpret_cast<float4*>(a.partial_o + at * kHeadDim + col);
    dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  }
}

// The ranges of a row put together: sixteen threads by four columns, each of sixteen groups takes every sixteenth range.
template <bool BIAS>
__global__ void __launch_bounds__(256) window_few_join_kernel(const __grid_constant__ FewArgs a) {
  __shared__ float4 o_all[16][16];
  __shared__ float2 ml_all[16];
  pdl_launch_dependents();
  const WindowArgs& w = a.w;
  const int r = blockIdx.x, kv = blockIdx.y, b = blockIdx.z, part = threadIdx.x >> 4, x = threadIdx.x & 15;
  pdl_wait();
  Item it;
  if (!few_item(w, b, it) || r >= it.rows * w.group) return;
  const long long at = (static_cast<long long>(b) * gridDim.y + kv) * a.splits * kFewRows + r;
  float top = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto take = [&](float2 ml, float4 o) {
    if (saw_nothing(ml)) return;
    const float next = fmaxf(top, ml.x), f0 = ex2(top - next), f1 = ex2(ml.x - next);
    top = next;
    sum = fmaf(ml.y, f1, sum * f0);
    acc.x = fmaf(o.x, f1, acc.x * f0);
    acc.y = fmaf(o.y, f1, acc.y * f0);
    acc.z = fmaf(o.z, f1, acc.z * f0);
    acc.w = fmaf(o.w, f1, acc.w * f0);
  };
#pragma unroll 4
  for (int s = part; s < a.splits; s += 16) {
    const long long i = at + static_cast<long long>(s) * kFewRows;
    take(a.partial_ml[i], *reinterpret_cast<const float4*>(a.partial_o + i * kHeadDim + 4 * x));
  }
  o_all[part][x] = acc;
  if (x == 0) ml_all[part] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x >= 32) return;
  __half2 bad = __half2half2(__ushort_as_half(0));
  if (part == 0) {
    for (int i = 1; i < min(16, a.splits); ++i) take(ml_all[i], o_all[i][x]);
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    const uint2 out = make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
    *reinterpret_cast<uint2*>(w.out + static_cast<long long>(it.q_row + r / w.group) * w.out_stride +
                              (kv * w.group + r % w.group) * kHeadDim + 4 * x) = out;
    watch(bad, out.x);
    watch(bad, out.y);
  }
  if (__any_sync(0xffffffffu, not_finite(bad))) redo_row<BIAS>(w, keys_of(w, it), it, r / w.group, kv * w.group + r % w.group);
}

// How a call of few queries is cut: ranges of a sequence's keys (0: the call is not one of few queries), and whether the ranges of
// an item are a cluster of CTAs, which put their results together through each other's shared memory, or leave them to a second
// kernel.
struct FewSplit {
  int ranges = 0;
  bool cluster = false;
};
// A CTA's time goes with its keys and something like 200 more (its first loads wait for one another, its results are put
// together), so of the numbers of ranges that leave a range 128 keys the one with the shortest sum over the waves is taken.
// Three CTAs are resident to an SM, but two of them already keep the memory busy: waves are counted by two.  us per call with
// waves of 296 / 370 / 444 / 592: 64 sequences of 4100 keys, 16 heads over 4, 44.2 / 51.3 / 50.3 / 56.8; 32 of 8192, 32 over 8, 81.7 / 91.1 /
// 88.6 / 105; 40 of 3000, 8 heads, 45.4 / 41.4 / 45.2 / 47.4; 8 of 4096, 12 heads, 21.5 / 21.5 / 21.0 / 25.2.
// Clusters save the second kernel, but their CTAs come and go together, so only calls whose CTAs are all resident at once take them.
// us with clusters (second kernel): 16 sequences of 1027 keys, one key/value head, 128 CTAs 6.4 (6.7); 4 of 700, 2 heads, 40 CTAs 5.4
// (6.3); 60 of 1000, 240 CTAs 7.6 (8.4); 110 of 1000, 220 CTAs 8.6 (10.7); 8 of 4096, 12 heads, 288 CTAs 21.9 (22.8); 74 of 2000, 296
// CTAs 11.9 (11.6).  Beyond the limit: 150 of 2000, 450 CTAs 23.5 (21.9); 48 of 1024, 4 heads, 576 CTAs 18.8 (17.6); 40 of 3000,
// 8 heads, 1280 CTAs 49.9 (48.1); 444 of 2000, 888 CTAs 43.5 (45.9).
// 148 SMs, a B200's: the workspace is asked for without a device, and the call has to come to the same split.
FewSplit few_split(int batch, int kv_heads, int group, int max_q, int max_k, int left, int sinks) {
  FewSplit f;
  if (static_cast<long long>(max_q) * group > kFewRows || batch > 65535 || kv_heads > 65535) return f;
  constexpr long long kWave = 2 * 148, kOverhead = 200, kTogether = 400;
  long long keys = max_k;
  if (left >= 0) keys = static_cast<long long>(left) + max_q + sinks + kSeam < keys ? static_cast<long long>(left) + max_q + sinks + kSeam : keys;
  const long long items = static_cast<long long>(batch) * kv_heads;
  long long best = 0x7fffffffffffffffLL;
  for (int s = 1; s <= 148 && (s == 1 || s * 128LL <= keys); ++s) {
    const long long cost = (items * s + kWave - 1) / kWave * (keys / s + kOverhead);
    if (cost < best) {
      f.ranges = s;
      best = cost;
    }
  }
  f.cluster = f.ranges > 1 && f.ranges <= kFewCluster && items * f.ranges <= kTogether;
  return f;
}
size_t few_workspace(long long items, FewSplit f) {
  return f.ranges <= 1 || f.cluster ? 0 : static_cast<size_t>(items) * f.ranges * kFewRows * (kHeadDim * 4 + 8);
}

template <bool BIAS>
cudaError_t launch_few(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const FewArgs& a, int kv_heads, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits, kv_heads, a.w.batch);
  cfg.blockDim = dim3(kFewWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (pdl_take_attr()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (a.cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.splits;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cfg.dynamicSmemBytes = kFewSmemBytes;
  cudaError_t e = cudaLaunchKernelEx(&cfg, window_few_kernel<BIAS>, tm_k, tm_v, a);
  if (e == cudaSuccess && a.splits > 1 && !a.cluster) e = launch_pdl(window_few_join_kernel<BIAS>, dim3(a.w.max_q * a.w.group, kv_heads, a.w.batch), dim3(256), 0, stream, a);
  return e;
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

struct DeviceFacts {
  int sms = 0, major = 0;
  int* status = nullptr;
};
// What a call needs to know of the current device, and what the device needs to know of the kernels; once (outside a
// capture, see bt_b200.h).
cudaError_t device_facts(DeviceFacts* f) {
  static std::mutex mu;
  static DeviceFacts known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (known[dev].status == nullptr) {
    DeviceFacts n;
    e = cudaDeviceGetAttribute(&n.sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n.major, cudaDevAttrComputeCapabilityMajor, dev);
    if (e != cudaSuccess) return e;
    n.status = device_status_word();
    if (n.status == nullptr) return cudaErrorUnknown;
    e = cudaFuncSetAttribute(window_mha_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout::kBytes);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(window_mha_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout::kBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(window_few_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmemBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(window_few_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmemBytes);
    if (e != cudaSuccess) return e;
    known[dev] = n;
  }
  *f = known[dev];
  return cudaSuccess;
}

// Lengths, windows and positions stay below this, so that none of their sums passes 32 bits.
constexpr int kMaxLength = (1 << 30) - 1;

}  // namespace

}  // namespace bt

using namespace bt;

extern "C" int bt_window_attention_workspace(int batch, int head_num, int kv_head_num, int max_q_len, int max_k_len, int left, int sinks,
                                             size_t* bytes) {
  if (!bytes || batch <= 0 || head_num <= 0 || head_num > 1024 || kv_head_num <= 0 || head_num % kv_head_num != 0 || max_q_len <= 0 ||
      max_q_len > kMaxLength || max_k_len < 0 || max_k_len > kMaxLength || sinks < 0)
    return BT_ERR_INVALID_ARG;
  *bytes = few_workspace(static_cast<long long>(batch) * kv_head_num,
                         few_split(batch, kv_head_num, head_num / kv_head_num, max_q_len, max_k_len, left, sinks));
  return BT_OK;
}

extern "C" int bt_window_attention(const bt_window_attention_args* a, void* stream_v) {
  if (a == nullptr || !a->q || !a->out || !a->q_offsets || !a->k_offsets) return BT_ERR_INVALID_ARG;
  if (a->k_rows > 0 && (!a->k || !a->v)) return BT_ERR_INVALID_ARG;
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->out, 16)) return BT_ERR_INVALID_ARG;
  if (!aligned(a->q_offsets, 4) || !aligned(a->k_offsets, 4) || !aligned(a->k_lens, 4) || !aligned(a->distance_bias, 4)) return BT_ERR_INVALID_ARG;
  if (a->head_num <= 0 || a->head_num > 1024 || a->kv_head_num <= 0 || a->head_num % a->kv_head_num != 0) return BT_ERR_INVALID_ARG;
  if (a->batch <= 0 || a->q_rows <= 0 || a->k_rows < 0 || a->max_q_len <= 0 || a->max_q_len > kMaxLength || a->max_k_len < 0 ||
      a->max_k_len > kMaxLength || a->sinks < 0 || !(a->scale > 0.f) || !(a->scale < INFINITY))
    return BT_ERR_INVALID_ARG;
  const long long q_cols = 64LL * a->head_num, kv_cols = 64LL * a->kv_head_num, max_stride = 1LL << 32;
  const long long strides[4] = {a->q_row_stride, a->k_row_stride, a->v_row_stride, a->out_row_stride};
  for (int i = 0; i < 4; ++i)
    if (strides[i] % 8 != 0 || strides[i] < (i == 0 || i == 3 ? q_cols : kv_cols) || strides[i] > max_stride) return BT_ERR_INVALID_ARG;
  if (a->distance_bias != nullptr && (a->bias_len <= 0 || a->bias_len > kMaxLength / 2 || a->bias_left < 0 || a->bias_left >= a->bias_len))
    return BT_ERR_INVALID_ARG;
  DeviceFacts dev;
  if (device_facts(&dev) != cudaSuccess) return BT_ERR_CUDA;
  if (dev.major != 10) return BT_ERR_UNSUPPORTED;
  WindowArgs w;
  w.q = static_cast<const __half*>(a->q);
  w.k = static_cast<const __half*>(a->k);
  w.v = static_cast<const __half*>(a->v);
  w.q_stride = a->q_row_stride;
  w.k_stride = a->k_row_stride;
  w.v_stride = a->v_row_stride;
  w.out = static_cast<__half*>(a->out);
  w.out_stride = a->out_row_stride;
  w.q_offsets = a->q_offsets;
  w.k_offsets = a->k_offsets;
  w.k_lens = a->k_lens;
  w.batch = a->batch;
  w.heads = a->head_num;
  w.group = a->head_num / a->kv_head_num;
  w.q_rows = a->q_rows;
  w.k_rows = a->k_rows;
  w.max_q = a->max_q_len;
  w.max_k = a->max_k_len;
  // a bound that no distance reaches is none
  w.left = a->left >= a->max_k_len ? -1 : a->left;
  w.right = a->right >= kMaxLength ? -1 : a->right;
  w.sinks = a->sinks < a->max_k_len ? a->sinks : a->max_k_len;
  w.scale_log2e = a->scale * 1.4426950408889634f;
  w.bias = a->distance_bias;
  w.bias_n = a->bias_len;
  w.bias_left = a->bias_left;
  w.status = dev.status;
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
  cudaError_t e;
  // Without any key rows the loads of the one masked tile that an item walks need some rows: those of q do.
  const bool none = a->k_rows == 0;
  const void *k = none ? a->q : a->k, *v = none ? a->q : a->v;
  const uint64_t k_rows = none ? a->q_rows : a->k_rows;
  const long long k_ld = none ? a->q_row_stride : a->k_row_stride, v_ld = none ? a->q_row_stride : a->v_row_stride;
  const FewSplit split = few_split(a->batch, a->kv_head_num, w.group, a->max_q_len, a->max_k_len, a->left, a->sinks);
  if (split.ranges > 0) {
    const int splits = split.ranges;
    const long long items = static_cast<long long>(a->batch) * a->kv_head_num;
    const size_t need = few_workspace(items, split);
    if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return BT_ERR_WORKSPACE;
    if (!aligned(a->workspace, 16)) return BT_ERR_INVALID_ARG;
    CUtensorMap tm_k, tm_v;
    if (!make_tmap_2d(&tm_k, k, k_rows, kv_cols, k_ld, 64, kFewKeys) || !make_tmap_2d(&tm_v, v, k_rows, kv_cols, v_ld, 64, kFewKeys))
      return BT_ERR_CUDA;
    FewArgs f{w, splits, split.cluster ? 1 : 0,
              static_cast<float*>(a->workspace), nullptr};
    f.partial_ml = reinterpret_cast<float2*>(f.partial_o + items * splits * kFewRows * kHeadDim);
    e = w.bias != nullptr ? launch_few<true>(tm_k, tm_v, f, a->kv_head_num, stream) : launch_few<false>(tm_k, tm_v, f, a->kv_head_num, stream);
    return e == cudaSuccess ? BT_OK : BT_ERR_CUDA;
  }
  CUtensorMap tm[5];
  const bool ok = make_tmap_2d(&tm[0], a->q, a->q_rows, q_cols, a->q_row_stride, 64, 128) &&
                  make_tmap_2d(&tm[1], k, k_rows, kv_cols, k_ld, 64, kKeys) && make_tmap_2d(&tm[2], v, k_rows, kv_cols, v_ld, 64, kKeys);
  if (!ok) return BT_ERR_CUDA;
  if (w.sinks > 0 && w.left >= 0) {  // a tile may hold the seam
    if (!make_tmap_2d(&tm[3], k, k_rows, kv_cols, k_ld, 64, kSeam) || !make_tmap_2d(&tm[4], v, k_rows, kv_cols, v_ld, 64, kSeam)) return BT_ERR_CUDA;
  } else {
    tm[3] = tm[1];
    tm[4] = tm[2];
  }
  e = w.bias != nullptr ? launch_window<true>(tm, w, dev.sms, stream) : launch_window<false>(tm, w, dev.sms, stream);
  if (e == cudaErrorInvalidValue) return BT_ERR_INVALID_ARG;
  return e == cudaSuccess ? BT_OK : BT_ERR_CUDA;
}
