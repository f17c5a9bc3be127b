// Log probabilities of given tokens, the entropy of their distributions and
// the top alternatives, with the gradient of the logits.
//
// For one row x of V logits with target t:
//   m = max x, z = sum exp(x - m), lse = m + ln z
//   logprob = x_t - lse
//   entropy = -sum p ln p = ln z - sum exp(x - m) (x - m) / z,   p = exp(x - lse)
//   d logprob / d x_j = [j == t] - p_j
//   d entropy / d x_j = -p_j (x_j - lse + entropy)
// Terms with p = 0 (a logit of -inf) are 0.  A row whose logits are all -inf
// has logprob -inf, entropy 0 and gradient 0; a NaN or +inf in a row makes its
// logprob, entropy and gradient NaN.  m and ln z are kept apart for the
// backward pass: (x - m) - ln z does not round away what x - lse would.
//
// Bound by memory: the forward reads the logits once (running maximum and
// sums), the backward reads them and writes their gradient once.  In the way of
// that stand one exponential a logit (16-bit logits: the units that compute them
// are 62 % busy, fp32 ones half of that) and, with alternatives, the selection at
// a row's end.  Measured back to back over inputs that L2 does not hold, of the
// measured copy bandwidth: 4096 x 50257 bf16 forward 79 us (0.79), top 5 109 us
// (0.57), top 64 168 us; 2048 x 50257 fp32 69 us (0.91); 8192 x 65536 bf16 forward
// 182 us (0.90), backward 316 us (1.04).  Sums are in fp32 in a fixed order.
// More loads on their way (eight groups a thread, 64
// registers) took 91 us instead of 78, all loads of a row's end at once with 48
// registers 83: both spill.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "elem_types.cuh"
#include "host_common.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = B200_LOGPROBS_MAX_TOP;
// Logits of a group: the maximum of each group of the row is kept in shared
// memory while the row streams by.  The top k elements of a row lie in its top
// k groups (groups ordered by maximum, then lower index: an element outside
// them has k elements before it, one in each), so only those are read again.
constexpr int kGroup = 8;
// Longest slice of a row that one block takes when alternatives are wanted:
// 8192 groups, 32 KB of maxima, 32 groups a thread.
constexpr int kTopSlice = 65536;
// Rows this short go to a warp each when there are enough of them to give every
// SM a block, with kWarpTop alternatives at most: no barriers, and eight rows'
// loads side by side.  bf16, us, a block a row -> a warp a row: 100000 x 500
// forward 270 -> 65, backward 214 -> 74, top 5 724 -> 131; 20000 x 5000 98 -> 54,
// 98 -> 83, 179 -> 75 (top 20 195 -> 110); 8192 x 8192 40 -> 32, 47.5 -> 50.5
// (2000 x 8192: 11 -> 13 backward).
constexpr int kWarpRow = 6144;
constexpr int kWarpTop = 24;
// Slices of a row at most when alternatives are wanted: one a thread of the join.
constexpr int kMaxTopVocab = kTopSlice * kThreads;
// Groups of a thread that are on their way at once.
constexpr int kUnroll = 4;

__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// 2^v, subnormal results as 0 (handling them would take four instructions more).
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// max that yields NaN when an operand is NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();

// Running maximum m, z = sum exp(x - m) and w = sum exp(x - m) (x - m).
struct Sums {
  float m, z, w;
};

// Moves sums to a maximum `m` >= s.m.  x - m = (x - s.m) + (s.m - m); a sum
// over nothing (s.m = -inf, z = 0) stays empty.  Where f is 0 the clamp of d
// keeps z d finite, and so 0 * -inf out of w.
__device__ __forceinline__ void rebase(Sums& s, float m) {
  if (s.m == m) return;
  const float d = s.m - m;
  const float f = exp2_approx(d * kLog2e);
  s.w = s.z > 0.0f ? f * fmaf(s.z, fmaxf(d, -1.0e4f), s.w) : (s.z == 0.0f ? 0.0f : s.z);
  s.z = s.z * f;
  s.m = m;
}

__device__ __forceinline__ Sums merge(Sums a, Sums b) {
  const float m = max_nan(a.m, b.m);
  rebase(a, m);
  rebase(b, m);
  return Sums{m, a.z + b.z, a.w + b.w};
}

// Adds a logit.
__device__ __forceinline__ void add_logit(Sums& s, float v) {
  if (!(v <= s.m)) rebase(s, max_nan(s.m, v));
  const float d = v - (s.m == kNegInf ? 0.0f : s.m);
  const float x = exp2_approx(d * kLog2e);
  s.z += x;
  // exp underflows to 0 long before -1e4: the clamp only keeps 0 * -inf out.
  s.w = fmaf(x, fmaxf(d, -1.0e4f), s.w);
}

// max of two packed 16-bit elements; NaN where an operand is.
template <typename T>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Three-input maximum (NaN if one is).
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Logits enter the sums no lower than this, which keeps 0 * -inf out of w, and
// so does the maximum they are summed under: a group that is masked altogether
// has differences of 0, not kClamp<T> minus the lowest value.  It makes no
// difference where the row's maximum is kClampFar<T> or more: what is lifted
// still has probability 0.  Rows below that (all masked with a lowest value)
// are summed again one by one.
template <typename T>
constexpr float kClamp = std::is_same<T, __half>::value ? -65504.0f : -1.0e30f;
template <typename T>
constexpr float kClampFar = std::is_same<T, __half>::value ? -65000.0f : -1.0e29f;

// The maximum that clamped logits with maximum `m` are summed under; -inf stays (nothing to sum).
template <typename T>
__device__ __forceinline__ float sum_base(float m) {
  return m < kClamp<T> && m != kNegInf ? kClamp<T> : m;
}

// A group's maximum, and its logits clamped.
template <typename T, int kPacks>
__device__ __forceinline__ float group_most(const Pack<T, kVec16<T>> (&q)[kPacks]) {
  if constexpr (sizeof(T) == 4) {
    float2 v[kGroup / 2];
    unpack<T, kVec16<T>, kPacks>(q, v);
    return max_nan(max3_nan(max3_nan(v[0].x, v[0].y, v[1].x), v[1].y, v[2].x), max3_nan(v[2].y, v[3].x, v[3].y));
  } else {
    static_assert(kPacks == 1, "a group is one pack");
    const uint32_t w = max_word<T>(max_word<T>(q[0].u[0], q[0].u[1]), max_word<T>(q[0].u[2], q[0].u[3]));
    const float2 m = word_to_pair<T>(w);
    return max_nan(m.x, m.y);
  }
}
template <typename T, int kPacks>
__device__ __forceinline__ void group_values(const Pack<T, kVec16<T>> (&q)[kPacks], float2 (&v)[kGroup / 2]) {
  if constexpr (sizeof(T) == 4) {
    unpack<T, kVec16<T>, kPacks>(q, v);
#pragma unroll
    for (int i = 0; i < kGroup / 2; ++i) v[i] = make_float2(max_nan(v[i].x, kClamp<T>), max_nan(v[i].y, kClamp<T>));
  } else {
    const uint32_t clamp = pair_to_word<T>(pair_of(kClamp<T>));
#pragma unroll
    for (int i = 0; i < kGroup / 2; ++i) v[i] = word_to_pair<T>(max_word<T>(q[0].u[i], clamp));
  }
}

// Adds a group of clamped logits whose maximum before was `mx`.  The sums of a
// thread are pairs: one instruction adds to both.
struct PairSums {
  float m;
  float2 z, w;
};

template <typename T>
__device__ __forceinline__ void add_group(PairSums& s, const float2 (&v)[kGroup / 2], float mx) {
  if (!(mx <= s.m)) {
    Sums a{s.m, s.z.x, s.w.x}, b{s.m, s.z.y, s.w.y};
    const float m = sum_base<T>(max_nan(s.m, mx));
    rebase(a, m);
    rebase(b, m);
    s = PairSums{m, make_float2(a.z, b.z), make_float2(a.w, b.w)};
  }
  const float2 minus_m = pair_of(s.m == kNegInf ? 0.0f : -s.m);
  const float2 log2e = pair_of(kLog2e);
#pragma unroll
  for (int i = 0; i < kGroup / 2; ++i) {
    const float2 d = add2(v[i], minus_m);
    const float2 t = mul2(d, log2e);
    const float2 x = make_float2(exp2_approx(t.x), exp2_approx(t.y));
    s.z = add2(s.z, x);
    s.w = fma2(x, d, s.w);
  }
}

// Sorts after every key with a smaller value, or with the same value and a
// higher index.  NaN is above +inf, and -0 equals +0.
constexpr uint32_t kNanOrder = 0xffff0000u;
__device__ __forceinline__ uint32_t order_bits(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return v != v ? kNanOrder : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long make_key(float v, uint32_t index) {
  return (static_cast<unsigned long long>(order_bits(v)) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long k) { return 0xffffffffu - static_cast<uint32_t>(k); }
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  if (u == kNanOrder) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// Calls one(index, value) or pack(first index, packs) over the logits
// [lo, hi) of a row so that every 16-byte aligned pack is read whole: the
// elements before the first aligned one and after the last go one by one.
template <typename T>
struct Span {
  int64_t head_end, body_end;  // [lo, head_end) single, [head_end, body_end) packs, [body_end, hi) single
  __device__ __forceinline__ Span(const T* row, int64_t lo, int64_t hi) {
    constexpr int kV = kVec16<T>;
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row + lo) & 15u) / sizeof(T);
    head_end = lo + (off ? kV - static_cast<int>(off) : 0);
    if (head_end > hi) head_end = hi;
    body_end = head_end + (hi - head_end) / kV * kV;
  }
};

// The block's sums, for every thread: the maximum first, then one rebase a
// thread and plain sums.
struct MergeBuffer {
  __align__(16) float m[kWarps];
  float2 zw[kWarps];
};
__device__ __forceinline__ Sums block_merge(Sums s, MergeBuffer& buf) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m = s.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) buf.m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) m = max_nan(m, buf.m[i]);
  rebase(s, m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
    s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
  }
  if (lane == 0) buf.zw[warp] = make_float2(s.z, s.w);
  __syncthreads();
  Sums r{m, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    r.z += buf.zw[i].x;
    r.w += buf.zw[i].y;
  }
  return r;
}

// Lowest bit of fp32 that a value of the type can have (other than by its sign).
template <typename T>
constexpr int kLowBit = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;

// Shared memory of the selection in a row (slice) of kRowThreads threads.
template <int kRowThreads>
struct Selection {
  static constexpr int kMost = kRowThreads == 32 ? kWarpTop : kMaxTop;  // alternatives
  static constexpr int kGroups = (kRowThreads == 32 ? kWarpRow : kTopSlice) / kGroup;
  // Candidates whose elements are offered without ranking them: one a thread,
  // about, and no more than `elems` holds.
  static constexpr int kFewCand = kRowThreads == 32 ? kMost : kRowThreads / kGroup;
  float group_max[kGroups];
  // Elements of the top groups, and those before the first and after the last.
  unsigned long long elems[kMost * kGroup + 4 * kGroup];
  // Candidate groups after the threshold: all those of kMost threads at most.
  uint16_t cand[kMost * (kGroups / kRowThreads)];
  unsigned long long bound;
  int count[2];
};
struct Nothing {};

template <int kRowThreads>
__device__ __forceinline__ void row_sync() {
  if constexpr (kRowThreads == 32)
    __syncwarp();
  else
    __syncthreads();
}
template <int kRowThreads>
__device__ __forceinline__ int row_count(bool p) {
  if constexpr (kRowThreads == 32)
    return __popc(__ballot_sync(0xffffffffu, p));
  else
    return __syncthreads_count(p);
}

// A lower bound of the top k of the keys of a row's threads (one each; 0 for
// none; all others differ), which at least k of them (or all) and at most `most`
// reach.  Found bit by bit from the first in which the keys differ: the values'
// bits, of which those below `low` are alike for values of one sign (16-bit
// types), then, if too many values are equal, the indexes'.  `hi` and `lo`: the
// largest and smallest value among the keys.
template <int kRowThreads>
__device__ __forceinline__ unsigned long long bound_by_bits(unsigned long long key, int k, int most, int low,
                                                            uint32_t hi, uint32_t lo) {
  const uint32_t v = static_cast<uint32_t>(key >> 32);
  const int first = 31 - __clz((hi ^ lo) | 1u);
  uint32_t t = first == 31 ? 0u : hi >> (first + 1) << (first + 1);
  int reach = kRowThreads;  // keys that reach t
  for (int bit = first; bit >= low; --bit) {
    const uint32_t u = t | (1u << bit);
    const int c = row_count<kRowThreads>(v >= u);
    if (c >= k) {
      t = u;
      reach = c;
    }
    if (c == k) break;
  }
  if (reach <= most) return static_cast<unsigned long long>(t) << 32;
  // Too many equal values at t (whose bits below `low` are all ones for a
  // negative value, see order_bits): their indexes decide.
  if ((t & 0x80000000u) == 0) t |= (1u << low) - 1;
  const bool tied = key != 0 && v == t;
  const int above = row_count<kRowThreads>(v > t);
  uint32_t at = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t u = at | (1u << bit);
    const int c = above + row_count<kRowThreads>(tied && static_cast<uint32_t>(key) >= u);
    if (c >= k) at = u;
    if (c == k) break;
  }
  return (static_cast<unsigned long long>(t) << 32) | at;
}

// The same for the keys of a warp.
__device__ __forceinline__ unsigned long long warp_bound(unsigned long long key, int k, int low) {
  const uint32_t v = static_cast<uint32_t>(key >> 32);
  if (row_count<32>(key != 0) <= k) return 0;
  return bound_by_bits<32>(key, k, kWarpTop, low, __reduce_max_sync(0xffffffffu, v), __reduce_min_sync(0xffffffffu, v));
}

// The same for the keys of a block, kMaxTop at most.  First try: the value of
// the k-th best of the maxima of `per` neighbouring threads, 1 (keys in the
// first kMaxTop threads only), 4 or 32 (k <= kWarps): three barriers, where one
// a bit takes about fifteen.
struct KthBuffer {
  __align__(16) uint32_t part[kMaxTop];
  uint32_t kth;
  uint32_t most[kWarps], least[kWarps];
};
__device__ __forceinline__ unsigned long long block_bound(unsigned long long key, int k, int per, int low,
                                                          KthBuffer& buf) {
  const uint32_t v = static_cast<uint32_t>(key >> 32);
  const int parts = per == 32 ? kWarps : kMaxTop;
  uint32_t b = v;
  if (per == 4) {
    b = max(b, __shfl_xor_sync(0xffffffffu, b, 1));
    b = max(b, __shfl_xor_sync(0xffffffffu, b, 2));
  } else if (per == 32) {
    b = __reduce_max_sync(0xffffffffu, b);
  }
  const int part = static_cast<int>(threadIdx.x) / per;
  if (threadIdx.x % per == 0 && part < parts) buf.part[part] = b;
  __syncthreads();
  if (threadIdx.x < parts) {
    const uint32_t own = buf.part[threadIdx.x];
    const int i = static_cast<int>(threadIdx.x);
    int before = 0;
    for (int j = 0; j < parts; j += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(&buf.part[j]);
      before += (q.x > own || (q.x == own && j < i)) + (q.y > own || (q.y == own && j + 1 < i)) +
                (q.z > own || (q.z == own && j + 2 < i)) + (q.w > own || (q.w == own && j + 3 < i));
    }
    if (before == k - 1) buf.kth = own;
  }
  __syncthreads();
  const uint32_t kth = buf.kth;
  if (__syncthreads_count(key != 0 && v >= kth) <= kMaxTop) return static_cast<unsigned long long>(kth) << 32;
  const uint32_t most = __reduce_max_sync(0xffffffffu, v), least = __reduce_min_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) {
    buf.most[threadIdx.x >> 5] = most;
    buf.least[threadIdx.x >> 5] = least;
  }
  __syncthreads();
  uint32_t hi = most, lo = least;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    hi = max(hi, buf.most[i]);
    lo = min(lo, buf.least[i]);
  }
  return bound_by_bits<kThreads>(key, k, kMaxTop, low, hi, lo);
}

// A warp's sums, for every thread.
__device__ __forceinline__ Sums warp_merge(Sums s) {
  float m = s.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  rebase(s, m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
    s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
  }
  return s;
}

struct Outputs {
  float* logprob;
  float* entropy;
  float2* stats;       // m, ln z (may be NULL)
  float* top_logprob;  // rows x top
  int64_t* top_index;
};

// The given token's logit; a target outside the vocabulary has no probability to give.
template <typename T>
__device__ __forceinline__ float target_logit(const T* x, int64_t vocab, int64_t target) {
  return target < 0 || target >= vocab ? __uint_as_float(0x7fffffffu) : to_f32(x[target]);
}

__device__ __forceinline__ void write_row(const Outputs& out, int64_t row, bool given, float logit, Sums s) {
  const bool empty = s.m == kNegInf;
  const float ln_z = logf(s.z);
  if (out.stats) out.stats[row] = make_float2(s.m, ln_z);
  out.entropy[row] = empty ? 0.0f : ln_z - s.w / s.z;
  float lp = 0.0f;
  if (given) lp = empty && logit == kNegInf ? kNegInf : (logit - s.m) - ln_z;
  out.logprob[row] = lp;
}

// One slice (blockIdx.x) of a row, by a block or, for short rows, by each of its
// warps (kRowThreads = 32).  With one slice a row, the row's outputs are written here; otherwise the slice's sums and its top
// keys, largest first, go to `part_sums` / `part_keys` and logprobs_join_kernel
// finishes the row.
template <typename T, bool kTop, int kRowThreads>
__global__ void __launch_bounds__(kThreads)
    logprobs_fwd_kernel(const T* __restrict__ logits, const int64_t* __restrict__ targets, int64_t rows, int64_t vocab,
                        int64_t ld, int64_t slice, int top, int64_t ignore, Outputs out, Sums* __restrict__ part_sums,
                        unsigned long long* __restrict__ part_keys) {
  using Sel = Selection<kRowThreads>;
  constexpr int kV = kVec16<T>;
  constexpr int kPacks = kGroup / kV;  // packs of a group
  __shared__ MergeBuffer merge_buf;
  __shared__ KthBuffer kth_buf;
  __shared__ std::conditional_t<kTop, Sel, Nothing> sel_buf[kThreads / kRowThreads];
  pdl_wait();
  const int slices = gridDim.x;
  const int64_t lo = blockIdx.x * slice;
  const int64_t hi = min(lo + slice, vocab);
  constexpr int kRows = kThreads / kRowThreads;  // of a block
  const int tid = threadIdx.x % kRowThreads;
  auto& sel = sel_buf[threadIdx.x / kRowThreads];
  for (int64_t row = static_cast<int64_t>(blockIdx.y) * kRows + threadIdx.x / kRowThreads; row < rows;
       row += static_cast<int64_t>(gridDim.y) * kRows) {
    const T* x = logits + row * ld;
    // Requested now, needed at the row's end.
    const int64_t target = tid == 0 && slices == 1 ? targets[row] : ignore;
    // Groups lie between the slice's first aligned element and its last whole
    // one; up to kV - 1 elements come before them and kGroup + kV - 1 after.
    const Span<T> span(x, lo, hi);
    const T* body = x + span.head_end;
    const int groups = static_cast<int>((span.body_end - span.head_end) / kGroup);
    const int64_t tail = span.head_end + static_cast<int64_t>(groups) * kGroup;
    PairSums ps{kNegInf, make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    float best_max = __uint_as_float(0x7fffffffu);  // the thread's best group: none yet, so any is better
    int best_group = -1;
    auto load = [&](Pack<T, kV> (&q)[kPacks], int g) {
#pragma unroll
      for (int p = 0; p < kPacks; ++p) q[p] = load_pack<T, kV>(body + static_cast<int64_t>(g) * kGroup + p * kV);
    };
    auto add = [&](const Pack<T, kV> (&q)[kPacks], int g) {
      float2 v[kGroup / 2];
      group_values<T, kPacks>(q, v);
      const float mx = group_most<T, kPacks>(q);
      if constexpr (kTop) {
        sel.group_max[g] = mx;
        // Strictly larger only: of equal groups the first stays.
        if (!(mx <= best_max)) {
          best_max = mx;
          best_group = g;
        }
      }
      add_group<T>(ps, v, mx);
    };
    int g = tid;
    // A warp's threads begin with the maximum of their first groups together:
    // few groups exceed it, where of a thread's own maximum some lane's group
    // nearly always does, and all lanes wait for its rebase.
    bool begin = (tid | 31) + (kUnroll - 1) * kRowThreads < groups;
    for (; g + (kUnroll - 1) * kRowThreads < groups; g += kUnroll * kRowThreads) {
      Pack<T, kV> q[kUnroll][kPacks];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) load(q[i], g + i * kRowThreads);
      if (begin) {
        begin = false;
        float m = group_most<T, kPacks>(q[0]);
#pragma unroll
        for (int i = 1; i < kUnroll; ++i) m = max_nan(m, group_most<T, kPacks>(q[i]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        ps.m = sum_base<T>(m);
      }
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) add(q[i], g + i * kRowThreads);
    }
    for (; g < groups; g += kRowThreads) {
      Pack<T, kV> q[kPacks];
      load(q, g);
      add(q, g);
    }
    Sums s = merge(Sums{ps.m, ps.z.x, ps.w.x}, Sums{ps.m, ps.z.y, ps.w.y});
    const bool has_head = lo + tid < span.head_end, has_tail = tail + tid < hi;
    const float head_v = has_head ? to_f32(x[lo + tid]) : kNegInf, tail_v = has_tail ? to_f32(x[tail + tid]) : kNegInf;
    const float target_v = target != ignore ? target_logit(x, vocab, target) : 0.0f;
    if (has_head) add_logit(s, head_v);
    if (has_tail) add_logit(s, tail_v);
    auto row_merge = [&](const Sums& a) { return kRowThreads == 32 ? warp_merge(a) : block_merge(a, merge_buf); };
    s = row_merge(s);
    if (s.m < kClampFar<T> && s.m != kNegInf) {
      s = Sums{kNegInf, 0.0f, 0.0f};
      for (int64_t j = lo + tid; j < hi; j += kRowThreads) add_logit(s, to_f32(x[j]));
      row_sync<kRowThreads>();
      s = row_merge(s);
    }
    if constexpr (kTop) {
      // Threshold: a bound that at least `top` of the threads' best groups and
      // at most Sel::kMost threads reach (or every group does).
      unsigned long long best = best_group >= 0 ? make_key(best_max, best_group) : 0;
      if (s.m != s.m) {
        // A NaN in the row: comparisons above may have dropped it.
        for (int i = tid; i < groups; i += kRowThreads) {
          const unsigned long long k = make_key(sel.group_max[i], i);
          best = k > best ? k : best;
        }
      }
      if (tid == 0) {
        sel.count[0] = sel.count[1] = 0;
        sel.bound = 0;
      }
      unsigned long long thr;
      if constexpr (kRowThreads == 32) {
        __syncwarp();
        thr = warp_bound(best, top, kLowBit<T>);
      } else {
        const int per = groups <= kMaxTop ? 1 : groups < kRowThreads || top > kWarps ? 4 : 32;
        thr = block_bound(best, top, per, kLowBit<T>, kth_buf);
      }
      if (best >= thr) {
        // Maxima below the bound's value (not NaN, nor anything below NaN) are out; the rest by key.
        const float thr_v = thr ? key_value(thr) : kNegInf;
        for (int i = tid; i < groups; i += 4 * kRowThreads) {
          float m[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) m[u] = sel.group_max[min(i + u * kRowThreads, groups - 1)];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int c = i + u * kRowThreads;
            if (c < groups && !(m[u] < thr_v) && make_key(m[u], c) >= thr)
              sel.cand[atomicAdd(&sel.count[0], 1)] = static_cast<uint16_t>(c);
          }
        }
      }
      row_sync<kRowThreads>();
      const int n_cand = sel.count[0];
      unsigned long long least_group = thr;
      if (n_cand > Sel::kFewCand) {
        // Of many candidates the best `top` groups only; the last of them
        // bounds the elements that can be among the top from below.
        for (int i = tid; i < n_cand; i += kRowThreads) {
          const unsigned long long k = make_key(sel.group_max[sel.cand[i]], sel.cand[i]);
          int r = 0;
          for (int j = 0; j < n_cand; ++j) r += make_key(sel.group_max[sel.cand[j]], sel.cand[j]) > k;
          if (r == top - 1) sel.bound = k;
        }
        row_sync<kRowThreads>();
        least_group = sel.bound;
      }
      const uint32_t least = static_cast<uint32_t>(least_group >> 32);
      auto offer = [&](float v, int64_t j) {
        if (order_bits(v) >= least) sel.elems[atomicAdd(&sel.count[1], 1)] = make_key(v, static_cast<uint32_t>(j));
      };
      for (int i = tid; i < n_cand * kGroup; i += kRowThreads) {
        const uint32_t c = sel.cand[i / kGroup];
        if (make_key(sel.group_max[c], c) >= least_group) {
          const int64_t j = span.head_end + static_cast<int64_t>(c) * kGroup + i % kGroup;
          offer(to_f32(x[j]), j);
        }
      }
      if (has_head) offer(head_v, lo + tid);
      if (has_tail) offer(tail_v, tail + tid);
      row_sync<kRowThreads>();
      const int n = sel.count[1];
      const float ln_z = logf(s.z);
      for (int i = tid; i < n; i += kRowThreads) {
        const unsigned long long k = sel.elems[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += sel.elems[j] > k;
        if (r < top) {
          if (slices == 1) {
            out.top_index[row * top + r] = key_index(k);
            out.top_logprob[row * top + r] = s.m == kNegInf ? kNegInf : (key_value(k) - s.m) - ln_z;
          } else {
            part_keys[(row * slices + blockIdx.x) * top + r] = k;
          }
        }
      }
      // A slice shorter than `top` leaves keys over: 0 sorts after every logit.
      if (slices > 1 && tid >= n && tid < top) part_keys[(row * slices + blockIdx.x) * top + tid] = 0;
    }
    if (tid == 0) {
      if (slices == 1)
        write_row(out, row, target != ignore, target_v, s);
      else
        part_sums[row * slices + blockIdx.x] = s;
    }
    row_sync<kRowThreads>();  // the next row reuses the shared arrays
  }
}

// Joins the slices of a row (with alternatives, kThreads of them at most); one
// block a row.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads)
    logprobs_join_kernel(const T* __restrict__ logits, const int64_t* __restrict__ targets, int64_t rows,
                         int64_t vocab, int64_t ld, int slices, int top, int64_t ignore, Outputs out,
                         const Sums* __restrict__ part_sums, const unsigned long long* __restrict__ part_keys) {
  __shared__ MergeBuffer merge_buf;
  __shared__ KthBuffer kth_buf;
  __shared__ unsigned long long elems[kTop ? kMaxTop * kMaxTop : 1];
  __shared__ int count;
  pdl_wait();
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t target = tid == 0 ? targets[row] : ignore;
    const float target_v = target != ignore ? target_logit(logits + row * ld, vocab, target) : 0.0f;
    Sums s{kNegInf, 0.0f, 0.0f};
    for (int i = tid; i < slices; i += kThreads) s = merge(s, part_sums[row * slices + i]);
    s = block_merge(s, merge_buf);
    if constexpr (kTop) {
      // As in a slice: a lower bound that the first keys of at least `top` and
      // at most kMaxTop slices reach.
      const unsigned long long* keys = part_keys + (row * slices + tid) * top;
      if (tid == 0) count = 0;
      const unsigned long long first = tid < slices ? keys[0] : 0;
      const unsigned long long thr = block_bound(first, top, slices <= kMaxTop ? 1 : 4, kLowBit<T>, kth_buf);
      if (first != 0 && first >= thr)
        for (int i = 0; i < top; ++i) {
          const unsigned long long k = keys[i];
          if (k == 0 || k < thr) break;
          elems[atomicAdd(&count, 1)] = k;
        }
      __syncthreads();
      const int n = count;
      const float ln_z = logf(s.z);
      for (int i = tid; i < n; i += kThreads) {
        const unsigned long long k = elems[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += elems[j] > k;
        if (r < top) {
          out.top_index[row * top + r] = key_index(k);
          out.top_logprob[row * top + r] = s.m == kNegInf ? kNegInf : (key_value(k) - s.m) - ln_z;
        }
      }
    }
    if (tid == 0) write_row(out, row, target != ignore, target_v, s);
    __syncthreads();
  }
}

// What the gradient of a row's logits needs of the row.
struct RowGrad {
  float minus_m, minus_ln_z, entropy, gl, gh;
};

// gl ([j == t] - p) - gh p (ln p + entropy)
__device__ __forceinline__ float grad_of(float x, const RowGrad& r, bool is_target) {
  const float d = (x + r.minus_m) + r.minus_ln_z;
  const float p = exp2_approx(d * kLog2e);
  const float g = -p * fmaf(r.gh, fmaxf(d, -1.0e4f) + r.entropy, r.gl);
  return is_target ? g + r.gl : g;
}

// One slice (blockIdx.x) of a row, by a block or, for short rows, by each of its warps.
template <typename T, int kRowThreads>
__global__ void __launch_bounds__(kThreads)
    logprobs_bwd_kernel(const T* __restrict__ logits, const int64_t* __restrict__ targets,
                        const float2* __restrict__ stats, const float* __restrict__ entropy,
                        const float* __restrict__ g_logprob, const float* __restrict__ g_entropy,
                        T* __restrict__ dlogits, int64_t rows, int64_t vocab, int64_t ld, int64_t ldd, int64_t slice,
                        int64_t ignore) {
  constexpr int kV = kVec16<T>;
  pdl_wait();
  const int64_t lo = blockIdx.x * slice;
  const int64_t hi = min(lo + slice, vocab);
  constexpr int kRows = kThreads / kRowThreads;  // of a block
  const int tid = threadIdx.x % kRowThreads;
  for (int64_t row = static_cast<int64_t>(blockIdx.y) * kRows + threadIdx.x / kRowThreads; row < rows;
       row += static_cast<int64_t>(gridDim.y) * kRows) {
    const T* x = logits + row * ld;
    T* d = dlogits + row * ldd;
    const int64_t target = targets[row];
    const float2 st = stats[row];
    float gl = g_logprob && target != ignore ? g_logprob[row] : 0.0f;
    // A target outside the vocabulary: the log probability is NaN, and so is what follows from it.
    if (gl != 0.0f && (target < 0 || target >= vocab)) gl = __uint_as_float(0x7fffffffu);
    const RowGrad r{-st.x, -st.y, entropy[row], gl, g_entropy ? g_entropy[row] : 0.0f};
    if (st.x == kNegInf) {
      // No probability anywhere: nothing depends on the logits.
      for (int64_t j = lo + tid; j < hi; j += kRowThreads) d[j] = from_f32<T>(0.0f);
      continue;
    }
    const Span<T> span(x, lo, hi);
    auto one = [&](int64_t j) { d[j] = from_f32<T>(grad_of(to_f32(x[j]), r, j == target)); };
    if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15u) != 0) {
      // Logits and gradient are aligned differently.
      for (int64_t j = lo + tid; j < hi; j += kRowThreads) one(j);
      continue;
    }
    const float2 minus_m = pair_of(r.minus_m), minus_ln_z = pair_of(r.minus_ln_z), log2e = pair_of(kLog2e);
    const float2 ent = pair_of(r.entropy), gl2 = pair_of(r.gl), gh2 = pair_of(r.gh);
    const T* body = x + span.head_end;
    T* out = d + span.head_end;
    const int packs = static_cast<int>((span.body_end - span.head_end) / kV);
    auto work = [&](const Pack<T, kV>& q, int i) {
      Pack<T, kV> o;
#pragma unroll
      for (int e = 0; e < kV / 2; ++e) {
        float2 f = add2(add2(q.pair(e), minus_m), minus_ln_z);
        const float2 t = mul2(f, log2e);
        // -p (gl + gh (ln p + entropy)); ln p is clamped where p is 0.
        const float2 p = make_float2(-exp2_approx(t.x), -exp2_approx(t.y));
        f = make_float2(fmaxf(f.x, -1.0e4f), fmaxf(f.y, -1.0e4f));
        o.set_pair(e, mul2(p, fma2(gh2, add2(f, ent), gl2)));
      }
      store_pack<T, kV>(out + static_cast<int64_t>(i) * kV, o);
    };
    int i = tid;
    for (; i + (kUnroll - 1) * kRowThreads < packs; i += kUnroll * kRowThreads) {
      Pack<T, kV> q[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) q[u] = load_pack<T, kV>(body + static_cast<int64_t>(i + u * kRowThreads) * kV);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) work(q[u], i + u * kRowThreads);
    }
    for (; i < packs; i += kRowThreads) work(load_pack<T, kV>(body + static_cast<int64_t>(i) * kV), i);
    if (lo + tid < span.head_end) one(lo + tid);
    if (span.body_end + tid < hi) one(span.body_end + tid);
    // The target's element once more, by the thread that wrote its pack.
    if (target >= span.head_end && target < span.body_end && (target - span.head_end) / kV % kRowThreads == tid)
      one(target);
  }
}

int cuda_code(cudaError_t e) { return e == cudaSuccess ? B200_OK : B200_ERR_CUDA; }

int dtype_size(int d) { return d == B200_DTYPE_F32 ? 4 : 2; }
bool dtype_ok(int d) { return d == B200_DTYPE_F16 || d == B200_DTYPE_BF16 || d == B200_DTYPE_F32; }

template <typename Fn>
int with_dtype(int dtype, Fn&& fn) {
  if (dtype == B200_DTYPE_F16) return fn(__half{});
  if (dtype == B200_DTYPE_BF16) return fn(__nv_bfloat16{});
  return fn(float{});
}

// Rows of a launch that are not taken by other blocks: gridDim.y.
unsigned row_blocks(int64_t rows, int per_block) {
  return (unsigned)std::min<int64_t>((rows + per_block - 1) / per_block, 65535);
}

// Slices a row is cut into: enough blocks for the device when rows are few
// (4096 logits each at least), and none longer than the selection can hold.
// The blocks are a constant, four for each SM of a B200, because the workspace's
// size, which is asked for without a device, follows from them.
int64_t row_slices(int64_t rows, int64_t vocab, int top) {
  constexpr int64_t kBlocks = 4 * 148, kLeast = 4096;
  int64_t s = std::max<int64_t>(1, std::min(kBlocks / std::max<int64_t>(rows, 1), vocab / kLeast));
  if (top > 0) s = std::max(std::min<int64_t>(s, kThreads), (vocab + kTopSlice - 1) / kTopSlice);
  return s;
}

// Slice length (a multiple of kGroup) for about `slices` slices, none empty.
int64_t slice_length(int64_t vocab, int64_t slices) { return round_up((vocab + slices - 1) / slices, kGroup); }

}  // namespace
}  // namespace b200

extern "C" int64_t b200_token_logprobs_workspace_size(int64_t rows, int64_t vocab, int top) {
  using namespace b200;
  if (rows < 0 || vocab < 0 || top < 0 || top > kMaxTop) return -B200_ERR_INVALID_ARGUMENT;
  if (vocab > (top > 0 ? kMaxTopVocab : 0x7fffffff)) return -B200_ERR_TOO_LARGE;
  const int64_t s = row_slices(rows, vocab, top);
  if (s <= 1) return 0;
  return round_up(rows * s * (int64_t)sizeof(Sums), 256) + rows * s * top * 8;
}

extern "C" int b200_token_logprobs_fwd(const void* logits, const int64_t* targets, float* logprob, float* entropy,
                                       float* stats, float* top_logprob, int64_t* top_index, int64_t rows,
                                       int64_t vocab, int64_t ld, int top, int64_t ignore_index, int dtype,
                                       void* workspace, int64_t workspace_bytes, void* stream_ptr) {
  using namespace b200;
  if (rows < 0 || vocab < 0 || top < 0 || top > kMaxTop || top > vocab || !dtype_ok(dtype))
    return B200_ERR_INVALID_ARGUMENT;
  if (vocab > (top > 0 ? kMaxTopVocab : 0x7fffffff)) return B200_ERR_TOO_LARGE;
  if (rows == 0) return B200_OK;
  if (vocab == 0 || !logits || !targets || !logprob || !entropy || ld < vocab ||
      (top > 0 && (!top_logprob || !top_index)))
    return B200_ERR_INVALID_ARGUMENT;
  if (!aligned_to(dtype_size(dtype), logits) || !aligned_to(8, targets, stats, top_index) ||
      !aligned_to(4, logprob, entropy, top_logprob))
    return B200_ERR_MISALIGNED;
  const int64_t need = b200_token_logprobs_workspace_size(rows, vocab, top);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))
    return B200_ERR_WORKSPACE;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const int64_t slice = slice_length(vocab, row_slices(rows, vocab, top));
  const int64_t slices = (vocab + slice - 1) / slice;
  const Outputs out{logprob, entropy, reinterpret_cast<float2*>(stats), top_logprob, top_index};
  Sums* sums = static_cast<Sums*>(workspace);
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(
      static_cast<uint8_t*>(workspace) + round_up(rows * slices * (int64_t)sizeof(Sums), 256));
  const bool warp_rows = slices == 1 && vocab <= kWarpRow && top <= kWarpTop && rows >= kWarps * dev.sm_count;
  const dim3 grid((unsigned)slices, row_blocks(rows, warp_rows ? kWarps : 1));
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T* x = static_cast<const T*>(logits);
    auto kern = warp_rows ? (top > 0 ? logprobs_fwd_kernel<T, true, 32> : logprobs_fwd_kernel<T, false, 32>)
                          : (top > 0 ? logprobs_fwd_kernel<T, true, kThreads> : logprobs_fwd_kernel<T, false, kThreads>);
    int rc = cuda_code(launch_gemm(kern, grid, dim3(kThreads), 0, stream, x, targets, rows, vocab, ld, slice, top,
                                   ignore_index, out, sums, keys));
    if (rc || slices == 1) return rc;
    const dim3 jgrid((unsigned)std::min<int64_t>(rows, 0x7fffffff));
    return cuda_code(top > 0 ? launch_gemm(logprobs_join_kernel<T, true>, jgrid, dim3(kThreads), 0, stream, x, targets,
                                           rows, vocab, ld, (int)slices, top, ignore_index, out, sums, keys)
                             : launch_gemm(logprobs_join_kernel<T, false>, jgrid, dim3(kThreads), 0, stream, x,
                                           targets, rows, vocab, ld, (int)slices, top, ignore_index, out, sums, keys));
  });
}

extern "C" int b200_token_logprobs_bwd(const void* logits, const int64_t* targets, const float* stats,
                                       const float* entropy, const float* g_logprob, const float* g_entropy,
                                       void* dlogits, int64_t rows, int64_t vocab, int64_t ld, int64_t ldd,
                                       int64_t ignore_index, int dtype, void* stream_ptr) {
  using namespace b200;
  if (rows < 0 || vocab < 0 || !dtype_ok(dtype)) return B200_ERR_INVALID_ARGUMENT;
  if (vocab > 0x7fffffff) return B200_ERR_TOO_LARGE;
  if (rows == 0 || vocab == 0) return B200_OK;
  if (!logits || !targets || !stats || !entropy || !dlogits || ld < vocab || ldd < vocab)
    return B200_ERR_INVALID_ARGUMENT;
  if (!aligned_to(dtype_size(dtype), logits, dlogits) || !aligned_to(8, targets, stats) ||
      !aligned_to(4, entropy, g_logprob, g_entropy))
    return B200_ERR_MISALIGNED;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  constexpr int64_t kSlice = 16384;
  const int64_t slice = std::min(kSlice, round_up(vocab, kGroup));
  const int64_t slices = (vocab + slice - 1) / slice;
  const bool warp_rows = vocab <= kWarpRow && rows >= kWarps * dev.sm_count;
  const dim3 grid((unsigned)slices, row_blocks(rows, warp_rows ? kWarps : 1));
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto kern = warp_rows ? logprobs_bwd_kernel<T, 32> : logprobs_bwd_kernel<T, kThreads>;
    return cuda_code(launch_gemm(kern, grid, dim3(kThreads), 0, stream,
                                 static_cast<const T*>(logits), targets, reinterpret_cast<const float2*>(stats),
                                 entropy, g_logprob, g_entropy, static_cast<T*>(dlogits), rows, vocab, ld, ldd, slice, ignore_index));
  });
}
