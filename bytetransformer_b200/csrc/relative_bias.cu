// Learned relative position bias by buckets of distance, and its gradient.
//
//   bias[h, q, k] = table[bucket(k - (q + q_start)), h]
//   grad_table[b, h] = sum of grad[i, h, q, k] over i, q, k with bucket(k - (q + q_start)) = b
//
// bucket(d), N buckets, largest distance told apart D: one-sided, the N buckets belong to n = max(-d, 0);
// bidirectional, half of them to n = |d| at d <= 0 and half to n = d at d > 0.  Of a side's m buckets the first
// e = m / 2 hold one distance each, the others grow with its logarithm:
//   n < e: n,   else min(m - 1, e + floor((m - e) * log(n / e) / log(D / e))).
// The borders are whole numbers, found on the host without rounding (see bucket_borders), so a distance on a border
// falls on the same side for every caller and every device.
//
// What both kernels live on: a bias is constant along diagonals.  Both are bound by memory: the forward writes
// heads * q_len * k_len elements and reads nothing to speak of, the gradient reads as many and writes a table.
// Measured on B200: 16 heads, 1024 x 1024 fp16 7.3 us (4.6 TB/s of stores into L2; filling the same with a constant takes 9.1), fp32 13.0; the
// gradient of 16 sequences of that 94 us (5.7 TB/s, 0.88 of a plain copy; fp32 160 us, 6.7 TB/s), of 8 x 12 heads x 509 x 509 16.4 us.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "../../include/bt_b200.h"

namespace bt {

namespace {

constexpr int kMaxBuckets = 256;
constexpr int kMaxDistance = 1 << 20;

// Smallest distance of each bucket of a side, rising: bucket(n) = the last i with first[i] <= n.
struct Borders {
  int first[kMaxBuckets];
  int count;      // buckets of a side
  int sides;      // 1 or 2
  int exact;      // buckets of one distance each
  float log_scale;  // (count - exact) / log2(D / exact): where to look first
};

// n^m * e^j against D^j * e^m in whole numbers of at most 4096 bits (20 bits * 128 + 7 bits * 128 at the limits above).
struct Whole {
  uint32_t limb[128];
  int n = 1;
  Whole() { limb[0] = 1; }
  void times(uint32_t f, int power) {
    while (power-- > 0) {
      uint64_t carry = 0;
      for (int i = 0; i < n; ++i) {
        carry += static_cast<uint64_t>(limb[i]) * f;
        limb[i] = static_cast<uint32_t>(carry);
        carry >>= 32;
      }
      if (carry != 0 && n < 128) limb[n++] = static_cast<uint32_t>(carry);
    }
  }
  bool less(const Whole& o) const {
    if (n != o.n) return n < o.n;
    for (int i = n - 1; i >= 0; --i)
      if (limb[i] != o.limb[i]) return limb[i] < o.limb[i];
    return false;
  }
};

void bucket_borders(Borders* b, int num_buckets, int max_distance, int bidirectional) {
  b->sides = bidirectional ? 2 : 1;
  b->count = num_buckets / b->sides;
  b->exact = b->count / 2;
  const int e = b->exact, m = b->count - e;
  b->log_scale = static_cast<float>(m / log2(static_cast<double>(max_distance) / e));
  for (int i = 0; i <= e; ++i) b->first[i] = i;
  const double ratio = pow(static_cast<double>(max_distance) / e, 1.0 / m);
  double x = e;
  for (int j = 1; j < m; ++j) {
    // Step j starts at the first whole n >= e * (D / e)^(j / m).  Double precision finds it (128 products are off by 1e-13 at
    // most) unless that is a whole number itself, or so near one that rounding could tell them apart wrongly.
    x *= ratio;
    const double near = nearbyint(x);
    int n = static_cast<int>(ceil(x));
    if (fabs(x - near) < 1e-9 * x) {
      n = static_cast<int>(near);
      Whole have, need;
      have.times(static_cast<uint32_t>(n), m);
      have.times(static_cast<uint32_t>(e), j);
      need.times(static_cast<uint32_t>(max_distance), j);
      need.times(static_cast<uint32_t>(e), m);
      if (have.less(need)) ++n;
    }
    b->first[e + j] = n;
  }
}

// Bucket of distance d by the borders in shared memory: the logarithm to a few bits, then the borders decide.
__device__ __forceinline__ int bucket_of(int d, const Borders& b, const int* first) {
  int n = d < 0 ? -d : (b.sides == 2 ? d : 0);
  int i = n;
  if (n >= b.exact) {
    i = b.exact + static_cast<int>(__log2f(__fdividef(static_cast<float>(n), static_cast<float>(b.exact))) * b.log_scale);
    i = min(i, b.count - 1);
    while (i + 1 < b.count && first[i + 1] <= n) ++i;
    while (first[i] > n) --i;
  }
  return (b.sides == 2 && d > 0) ? i + b.count : i;
}

// ------------------------------------------------------------------------------------------------ forward
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

struct BiasArgs {
  const void* table;  // [buckets, heads]
  void* out;          // [heads, q_len, k_len]
  int heads, q_len, k_len, q_start;
  int rows, cols;     // of a CTA's tile (the last one of a row: up to V columns more)
  Borders borders;
};

constexpr int kBiasThreads = 256;

// A CTA writes `rows` x `cols` of one head.  The tile holds rows + cols - 1 different values, one per diagonal; row r is
// the slice of them that starts at rows - 1 - r.  So the CTA lays the values of its diagonals out in shared memory once,
// 16 / sizeof(T) times, each copy an element further on: a slice then starts on a 16-byte boundary in one of the copies,
// whichever boundary its place in global memory asks for, and leaves by one bulk copy.
template <typename T, typename TableT>
__global__ void __launch_bounds__(kBiasThreads) relative_bias_kernel(const __grid_constant__ BiasArgs a) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ T column[kMaxBuckets];
  __shared__ int first[kMaxBuckets];
  pdl_launch_dependents();
  const int head = blockIdx.z;
  const int q0 = blockIdx.y * a.rows;
  const int k0 = blockIdx.x * a.cols;
  const int rows = min(a.rows, a.q_len - q0);
  // A row's share of the tile starts and ends on 16-byte boundaries of its own (up to V - 1 columns on), except at the row's ends.
  // (The last tile has more than V columns, so these boundaries lie inside it, or is the only one.)
  const bool first_cols = blockIdx.x == 0, last_cols = blockIdx.x + 1 == gridDim.x;
  const int cols = last_cols ? a.k_len - k0 : a.cols;
  const int diagonals = rows + cols + (last_cols ? 0 : V - 1) - 1;
  const int pitch = (a.rows + a.cols + 4 * V - 1) / V * V;  // elements of a copy, a multiple of 16 bytes
  T* copies = reinterpret_cast<T*>(smem);
  for (int i = threadIdx.x; i < a.borders.count; i += kBiasThreads) first[i] = a.borders.first[i];
  pdl_wait();
  for (int i = threadIdx.x; i < a.borders.count * a.borders.sides; i += kBiasThreads)
    column[i] = static_cast<T>(static_cast<float>(reinterpret_cast<const TableT*>(a.table)[static_cast<size_t>(i) * a.heads + head]));
  __syncthreads();
  // diagonal x of the tile: distance of its last row's first element, plus x
  const int d0 = k0 - (q0 + rows - 1) - a.q_start;
  for (int x = threadIdx.x; x < diagonals; x += kBiasThreads) copies[x] = column[bucket_of(d0 + x, a.borders, first)];
  __syncthreads();
  for (int y = threadIdx.x; y < pitch / V - 1; y += kBiasThreads) {  // the shifted copies, a vector at a time
    const uint4 lo = reinterpret_cast<const uint4*>(copies)[y], hi = reinterpret_cast<const uint4*>(copies)[y + 1];
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int p = 1; p < V; ++p) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 4)
          o[i] = w[i + p < 8 ? i + p : 7];
        else
          o[i] = (p & 1) ? __funnelshift_r(w[i + p / 2], w[i + p / 2 + 1], 16) : w[i + p / 2];
      }
      reinterpret_cast<uint4*>(copies + p * pitch)[y] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
  fence_proxy_async_smem();
  __syncthreads();
  T* out = reinterpret_cast<T*>(a.out) + (static_cast<size_t>(head) * a.q_len + q0) * a.k_len + k0;
  // elements of row r of the tile ahead of its first 16-byte boundary, and those from there on that whole vectors hold
  auto lead_of = [&](int r) {
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(out + static_cast<size_t>(r) * a.k_len) / sizeof(T));
    return min(static_cast<int>((V - at % V) % V), cols);
  };
  auto body_of = [&](int lead) { return last_cols ? (cols - lead) / V * V : cols; };
  // (the lanes of a warp issue their copies one after the other: the rows go round the warps)
  for (int r = (threadIdx.x & 31) * (kBiasThreads / 32) + (threadIdx.x >> 5); r < rows; r += kBiasThreads) {
    const int lead = lead_of(r), body = body_of(lead);
    const int x = rows - 1 - r + lead;
    if (body > 0)
      bulk_store(out + static_cast<size_t>(r) * a.k_len + lead, copies + (x % V) * pitch + x / V * V, static_cast<uint32_t>(body * sizeof(T)));
  }
  tma_store_commit();
  if (a.k_len % V != 0 && (first_cols || last_cols)) {
    // the rows' ragged ends, 2 V - 2 elements at most: 2 V lanes for each row
    for (int i = threadIdx.x; i < rows * 2 * V; i += kBiasThreads) {
      const int r = i / (2 * V), s = i % (2 * V);
      const int lead = lead_of(r);
      const int c = s < V ? s : lead + body_of(lead) + s - V;
      if (s < V ? first_cols && c < lead : last_cols && c < cols) out[static_cast<size_t>(r) * a.k_len + c] = copies[rows - 1 - r + c];
    }
  }
  tma_store_wait_read();
}

// ------------------------------------------------------------------------------------------------ gradient
struct GradArgs {
  const void* grad;  // [batch, heads, q_len, k_len]
  float* partial;    // [heads, buckets, parts]
  int batch, heads, q_len, k_len, q_start;
  int groups;  // CTAs side by side over a row chunk's diagonals
  int chunks, chunk_rows;
  int parts;   // batch * chunks * groups
  int walkers;
  Borders borders;
};

constexpr int kGradWalkers = 192;  // threads that walk down the diagonals, at most
constexpr int kGradOthers = 64;    // threads beside them for the rows' ragged ends (32 to 128: 8 sequences, 12 heads, 509 x 509 17.0,
                                   // 16.4, 25.3 us); all sum the buckets
constexpr int kGradRows = 128;  // rows of a chunk at most: the longest chain of single-precision additions

// A CTA sums the diagonals of up to `kGradRows` rows of one plane (sequence, head), over a range of diagonals, then the
// diagonals of each bucket.  A thread holds 2 V - 1 diagonals (V = elements of 16 bytes) in registers and walks down them,
// V rows and one aligned 16-byte load per row at a time: with every row the matrix's next aligned vector lies
// k_len + 1 elements further on relative to the diagonals, so the vector of row r starts (-r * (k_len + 1)) mod V diagonals
// into the thread's range, a number that only k_len mod V (M) decides and that repeats every V rows.  So every index of
// a register is known at compile time, whatever the row length, and neighbouring threads load neighbouring vectors.
// Rows that do not start on a 16-byte boundary have up to V - 1 elements ahead of their first whole vector and behind
// their last; those are summed by diagonal, a thread each, by threads of their own beside the walk.
template <typename T, int M>
__global__ void __launch_bounds__(kGradWalkers + kGradOthers, 2) relative_bias_grad_kernel(const __grid_constant__ GradArgs a) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  constexpr int kSpanMax = kGradWalkers * V;
  constexpr int kEdge = kGradRows + V;
  __shared__ float low[kSpanMax + V], high[kSpanMax + V], block[kGradWalkers + 1], edge[M != 0 ? 2 : 1][M != 0 ? kEdge : 1];
  __shared__ int first[kMaxBuckets];
  pdl_launch_dependents();
  const int t = threadIdx.x;
  const int walkers = a.walkers;
  const int span = walkers * V;
  for (int i = t; i < a.borders.count; i += blockDim.x) first[i] = a.borders.first[i];
  const int group = blockIdx.x % a.groups;
  const int chunk = blockIdx.x / a.groups;
  const int head = blockIdx.y;
  const int item = blockIdx.z;
  const int q0 = chunk * a.chunk_rows;
  const int rows = min(a.chunk_rows, a.q_len - q0);
  const int k_len = a.k_len;
  const size_t start = ((static_cast<size_t>(item) * a.heads + head) * a.q_len + q0) * k_len;  // element of row q0
  const T* base = reinterpret_cast<const T*>(a.grad) + start;
  // Diagonals are counted as the column of row q0 that they pass.  The range's first one: the leftmost, -(rows - 1),
  // rounded down so that the vectors of the rows q0, q0 + V, ... are aligned there (and V - 1 earlier: a row's vectors start up
  // to that many diagonals further on).
  const int phase = static_cast<int>(start % V);  // elements of row q0 past a boundary
  const int leftmost = -(rows - 1) - (V - 1) + phase;
  const int c_first = -((-leftmost + V - 1) / V) * V - phase + group * span;  // (leftmost <= 0)
  const int c0 = c_first + t * V;
  pdl_wait();
  if constexpr (M != 0) {
    // elements of row r (from q0) ahead of its first boundary
    auto lead_of = [&](int r) { return min((V - static_cast<int>((phase + static_cast<unsigned>(r) * M) % V)) % V, k_len); };
    for (int x = t - walkers; t >= walkers && x < rows + V - 1; x += kGradOthers) {
      // diagonal -(rows - 1) + x on the left, k_len - V + 1 - (rows - 1) + x on the right
      T e[2][V - 1];
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const int d = (side ? k_len - V + 1 + x : x) - (rows - 1);
#pragma unroll
        for (int i = 0; i < V - 1; ++i) {
          const int col = side ? k_len - 1 - i : i;
          const int r = col - d;
          bool take = r >= 0 && r < rows && col >= 0 && col < k_len;
          if (take) {
            const int lead = lead_of(r);
            take = side ? col >= lead + (k_len - lead) / V * V : col < lead;
          }
          e[side][i] = take ? base[static_cast<size_t>(r) * k_len + col] : static_cast<T>(0.f);
        }
      }
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V - 1; ++i) sum += static_cast<float>(e[side][i]);
        edge[side][x] = sum;
      }
    }
  }
  float acc[2 * V - 1];
#pragma unroll
  for (int i = 0; i < 2 * V - 1; ++i) acc[i] = 0.f;
  // One step: V rows, a whole vector of each.
  auto load = [&](uint4 (&v)[V], int n) {
    const int c = c0 + n * V;
    const T* row = base + static_cast<size_t>(n * V) * k_len + c;
    // the V vectors lie in columns c .. c + 3 V - 3
    if (c >= 0 && c + 3 * V - 2 <= k_len && n * V + V <= rows) {
#pragma unroll
      for (int r = 0; r < V; ++r) {
        constexpr int kStep = M + 1;
        v[r] = *reinterpret_cast<const uint4*>(row + r * static_cast<ptrdiff_t>(k_len) + (r + (V * kStep - r * kStep) % V));
      }
    } else {
#pragma unroll
      for (int r = 0; r < V; ++r) {
        constexpr int kStep = M + 1;
        const int shift = (V * kStep - r * kStep) % V;  // static: see above
        const int col = c + r + shift;
        v[r] = make_uint4(0u, 0u, 0u, 0u);
        if (n * V + r < rows && col >= 0 && col + V <= k_len)
          v[r] = *reinterpret_cast<const uint4*>(row + r * static_cast<ptrdiff_t>(k_len) + (r + shift));
      }
    }
  };
  auto add = [&](const uint4 (&v)[V]) {
#pragma unroll
    for (int r = 0; r < V; ++r) {
      constexpr int kStep = M + 1;
      const int shift = (V * kStep - r * kStep) % V;
      const uint32_t w[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (V == 8)
          add_half2(acc[shift + 2 * i], acc[shift + 2 * i + 1], w[i]);
        else
          acc[shift + i] += __uint_as_float(w[i]);
      }
    }
  };
  // The steps of this thread: those whose vectors have a column in the matrix.  The next one's loads are out before this
  // one's values are added.
  const int n0 = c0 + 3 * V - 2 > 0 ? 0 : (-(c0 + 3 * V - 2)) / V + 1;
  const int n1 = min((rows + V - 1) / V, c0 < k_len ? (k_len - 1 - c0) / V + 1 : 0);
  if (t < walkers && n0 < n1) {
    uint4 v[V], w[V];
    load(v, n0);
#pragma unroll 1
    for (int n = n0; n < n1; n += 2) {
      const bool more = n + 1 < n1;
      if (more) load(w, n + 1);
      add(v);
      if (!more) break;
      if (n + 2 < n1) load(v, n + 2);
      add(w);
    }
  }
  // Diagonal t * V + i of the range: the thread's own first V in `low`, what it holds of its right neighbour's in `high`
  if (t < walkers) {
#pragma unroll
    for (int i = 0; i < V; ++i) low[t * V + i] = acc[i];
#pragma unroll
    for (int i = V; i < 2 * V - 1; ++i) high[t * V + i] = acc[i];
    high[t * V + 2 * V - 1] = 0.f;
  }
  if (t == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      high[i] = 0.f;
      low[span + i] = 0.f;
    }
  }
  __syncthreads();
  // The diagonals' sums, in `low`, and those of V diagonals each, which the long runs below take.
  for (int g = t; g <= walkers; g += blockDim.x) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int x = g * V + i;
      float d = low[x] + high[x];
      if constexpr (M != 0) {
        if (x < span) {  // (the rest of the range is the next group's too)
          const int l = c_first + x + (rows - 1), r = l - (k_len - V + 1);
          if (l >= 0 && l < rows + V - 1) d += edge[0][l];
          if (r >= 0 && r < rows + V - 1) d += edge[1][r];
        }
      }
      low[x] = d;
      sum += d;
    }
    block[g] = sum;
  }
  __syncthreads();
  // Distance of diagonal x: x + d_first.  A bucket is a run of diagonals, summed by eight lanes.
  const int d_first = c_first - q0 - a.q_start;
  const int total = a.borders.count * a.borders.sides;
  const int part = (item * a.chunks + chunk) * a.groups + group;
  const int sub = t & 7;
  for (int b0 = (t >> 5) * 4; b0 < total; b0 += blockDim.x / 8) {
    const int b = b0 + ((t >> 3) & 3);
    float sum = 0.f;
    if (b < total) {
      const bool right = b >= a.borders.count;
      const int i = right ? b - a.borders.count : b;
      const bool outermost = i + 1 == a.borders.count;
      int x0 = 0, x1 = span + V;  // the run: x0 <= x < x1
      if (right) {
        x0 = max(x0, max(first[i], 1) - d_first);
        if (!outermost) x1 = min(x1, first[i + 1] - d_first);
      } else {
        if (!outermost) x0 = max(x0, 1 - first[i + 1] - d_first);
        if (i > 0 || a.borders.sides == 2) x1 = min(x1, 1 - first[i] - d_first);
      }
      // ragged ends element by element, what lies between by blocks
      const int g0 = (x0 + V - 1) / V, g1 = x1 / V;
      if (x0 < x1 && g0 < g1) {
        for (int x = x0 + sub; x < g0 * V; x += 8) sum += low[x];
        for (int g = g0 + sub; g < g1; g += 8) sum += block[g];
        for (int x = g1 * V + sub; x < x1; x += 8) sum += low[x];
      } else {
        for (int x = x0 + sub; x < x1; x += 8) sum += low[x];
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sub == 0 && b < total) a.partial[(static_cast<size_t>(head) * total + b) * a.parts + part] = sum;
  }
}

// One warp per (head, bucket): the CTAs' sums, in a fixed order.
__global__ void __launch_bounds__(256) relative_bias_grad_join_kernel(const float* __restrict__ partial, float* __restrict__ out,
                                                                      int heads, int buckets, int parts) {
  pdl_launch_dependents();
  pdl_wait();
  const int at = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= heads * buckets) return;
  double sum = 0.0;
  for (int i = threadIdx.x & 31; i < parts; i += 32) sum += partial[static_cast<size_t>(at) * parts + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) out[static_cast<size_t>(at % buckets) * heads + at / buckets] = static_cast<float>(sum);
}

bool bias_shape_ok(int num_buckets, int max_distance, int bidirectional, int heads, int q_len, int k_len, int q_start) {
  const int sides = bidirectional ? 2 : 1;
  if (num_buckets < 2 * sides || num_buckets > kMaxBuckets || num_buckets % sides != 0) return false;
  if (max_distance <= num_buckets / sides / 2 || max_distance > kMaxDistance) return false;
  // distances stay far inside 32 bits
  const int limit = 1 << 29;
  return heads > 0 && heads <= 65535 && q_len > 0 && q_len <= limit && k_len > 0 && k_len <= limit && q_start >= -limit && q_start <= limit;
}

struct GradSplit {
  int groups, chunks, chunk_rows;
  int walkers;  // of a CTA: no more than the diagonals ask for
  long long parts;
};
GradSplit grad_split(int batch, int heads, int q_len, int k_len, int elem_bytes) {
  GradSplit s;
  const int v = 16 / elem_bytes;
  // Chunks of 128 rows waste least (a chunk of R rows walks R diagonals more than the matrix has columns), but every CTA
  // walks its rows one after the other: calls of few rows take shorter ones, down to 16, while there are fewer than two CTAs to an
  // SM.  us with that line at 1 / 2 / 4 / 8 CTAs to an SM: 8 x 12 heads x 197 x 197 12.7 / 9.8 / 11.3 / 13.7; 16 heads, 1024 x 1024 11.5 / 11.9 /
  // 16.4 / 16.4; 2 x 16 heads x 384 x 384 9.1 / 7.7 / 9.9 / 9.9.  (148 SMs, a B200's: the workspace is asked for without a device.)
  s.chunk_rows = kGradRows;
  while (s.chunk_rows > 16 && static_cast<long long>(batch) * heads * ((q_len + s.chunk_rows - 1) / s.chunk_rows) < 2 * 148) s.chunk_rows /= 2;
  s.chunks = (q_len + s.chunk_rows - 1) / s.chunk_rows;
  const long long vectors = (static_cast<long long>(k_len) + (q_len < s.chunk_rows ? q_len : s.chunk_rows) + 3 * v - 1) / v;
  s.groups = static_cast<int>((vectors + kGradWalkers - 1) / kGradWalkers);
  s.walkers = static_cast<int>(((vectors + s.groups - 1) / s.groups + 31) / 32 * 32);
  s.parts = static_cast<long long>(batch) * s.chunks * s.groups;
  return s;
}

template <typename T, int M>
cudaError_t launch_grad(const GradArgs& a, cudaStream_t stream) {
  const int threads = M != 0 ? a.walkers + kGradOthers : (a.walkers < 128 ? 128 : a.walkers);
  return launch_pdl(relative_bias_grad_kernel<T, M>, dim3(static_cast<unsigned>(a.groups) * a.chunks, a.heads, a.batch), dim3(threads),
                    0, stream, a);
}

template <typename T, typename TableT>
cudaError_t launch_bias(BiasArgs a, cudaStream_t stream) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  // (16 heads, 1024 x 1024 fp16, us by tile: 64 x 1024 12.8, 64 x 512 9.3, 32 x 512 7.7, 64 x 256 7.3, 16 x 256 12.0: enough CTAs that some
  // store while others lay out their diagonals)
  a.cols = a.k_len <= 256 + V ? a.k_len : 256;
  a.rows = a.q_len < 64 ? a.q_len : 64;
  const size_t smem = static_cast<size_t>(V) * ((a.rows + a.cols + 4 * V - 1) / V * V) * sizeof(T);
  const long long tiles_q = (a.q_len + a.rows - 1) / a.rows;
  if (tiles_q > 65535) return cudaErrorInvalidValue;
  return launch_pdl(relative_bias_kernel<T, TableT>, dim3(a.k_len == a.cols ? 1 : (a.k_len - V + a.cols - 1) / a.cols, static_cast<unsigned>(tiles_q), a.heads),
                    dim3(kBiasThreads), smem, stream, a);
}

}  // namespace

}  // namespace bt

using namespace bt;

extern "C" {

int bt_relative_position_bias(const void* table, int table_fp32, int num_buckets, int max_distance, int bidirectional,
                              int head_num, int q_len, int k_len, int q_start, void* out, int out_fp32, void* stream) {
  if (!table || !out || (reinterpret_cast<uintptr_t>(out) & 15u) != 0) return BT_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(table) & (table_fp32 ? 3u : 1u)) != 0) return BT_ERR_INVALID_ARG;
  if (!bias_shape_ok(num_buckets, max_distance, bidirectional, head_num, q_len, k_len, q_start)) return BT_ERR_INVALID_ARG;
  BiasArgs a;
  a.table = table;
  a.out = out;
  a.heads = head_num;
  a.q_len = q_len;
  a.k_len = k_len;
  a.q_start = q_start;
  bucket_borders(&a.borders, num_buckets, max_distance, bidirectional);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (out_fp32)
    e = table_fp32 ? launch_bias<float, float>(a, s) : launch_bias<float, __half>(a, s);
  else
    e = table_fp32 ? launch_bias<__half, float>(a, s) : launch_bias<__half, __half>(a, s);
  if (e == cudaErrorInvalidValue) return BT_ERR_INVALID_ARG;
  return e == cudaSuccess ? BT_OK : BT_ERR_CUDA;
}

int bt_relative_position_bias_grad_workspace(int grad_fp32, int num_buckets, int batch, int head_num, int q_len, int k_len,
                                             size_t* bytes) {
  if (!bytes || batch <= 0 || batch > 65535) return BT_ERR_INVALID_ARG;
  if (!bias_shape_ok(num_buckets, kMaxDistance, 0, head_num, q_len, k_len, 0)) return BT_ERR_INVALID_ARG;
  const GradSplit s = grad_split(batch, head_num, q_len, k_len, grad_fp32 ? 4 : 2);
  if (s.parts > 0x7fffffffLL) return BT_ERR_INVALID_ARG;
  *bytes = static_cast<size_t>(s.parts) * head_num * num_buckets * 4;
  return BT_OK;
}

int bt_relative_position_bias_grad(const void* grad, int grad_fp32, int num_buckets, int max_distance, int bidirectional,
                                   int batch, int head_num, int q_len, int k_len, int q_start, float* grad_table,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (!grad || !grad_table || !workspace) return BT_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(grad) & 15u) != 0 || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0 ||
      (reinterpret_cast<uintptr_t>(grad_table) & 3u) != 0)
    return BT_ERR_INVALID_ARG;
  if (!bias_shape_ok(num_buckets, max_distance, bidirectional, head_num, q_len, k_len, q_start)) return BT_ERR_INVALID_ARG;
  size_t need = 0;
  const int rc = bt_relative_position_bias_grad_workspace(grad_fp32, num_buckets, batch, head_num, q_len, k_len, &need);
  if (rc != BT_OK) return rc;
  if (workspace_bytes < need) return BT_ERR_WORKSPACE;
  const GradSplit split = grad_split(batch, head_num, q_len, k_len, grad_fp32 ? 4 : 2);
  GradArgs a;
  a.grad = grad;
  a.partial = reinterpret_cast<float*>(workspace);
  a.batch = batch;
  a.heads = head_num;
  a.q_len = q_len;
  a.k_len = k_len;
  a.q_start = q_start;
  a.groups = split.groups;
  a.chunks = split.chunks;
  a.chunk_rows = split.chunk_rows;
  a.walkers = split.walkers;
  a.parts = static_cast<int>(split.parts);
  bucket_borders(&a.borders, num_buckets, max_distance, bidirectional);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaErrorInvalidValue;
  if (grad_fp32) {
    switch (k_len % 4) {
      case 0: e = launch_grad<float, 0>(a, s); break;
      case 1: e = launch_grad<float, 1>(a, s); break;
      case 2: e = launch_grad<float, 2>(a, s); break;
      case 3: e = launch_grad<float, 3>(a, s); break;
    }
  } else {
    switch (k_len % 8) {
      case 0: e = launch_grad<__half, 0>(a, s); break;
      case 1: e = launch_grad<__half, 1>(a, s); break;
      case 2: e = launch_grad<__half, 2>(a, s); break;
      case 3: e = launch_grad<__half, 3>(a, s); break;
      case 4: e = launch_grad<__half, 4>(a, s); break;
      case 5: e = launch_grad<__half, 5>(a, s); break;
      case 6: e = launch_grad<__half, 6>(a, s); break;
      case 7: e = launch_grad<__half, 7>(a, s); break;
    }
  }
  if (e == cudaSuccess)
    e = launch_pdl(relative_bias_grad_join_kernel, dim3((head_num * num_buckets + 7) / 8), dim3(256), 0, s,
                   static_cast<const float*>(a.partial), grad_table, head_num, num_buckets, a.parts);
  return e == cudaSuccess ? BT_OK : BT_ERR_CUDA;
}

}  // extern "C"
