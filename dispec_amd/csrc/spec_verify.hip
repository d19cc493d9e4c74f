// The verdict on drafted tokens: which path of each sequence's tree the target keeps, and the
// token that follows it.  The reference decides a chain on the host side of torch
// (dispec/spec/rejection.py:25-54); here a tree or a chain is decided on the device, from given
// random numbers, so that nothing waits for the host between the forward and the commit.
//
// Node 0 of a sequence is the last token that was kept; row i of the target's probabilities is
// the distribution p_i of the token after node i.
//  * Chain with the draft's probabilities (rejection sampling): after node c, its child with
//    token x is kept where u_c q_c(x) < p_c(x); the first token that is not is replaced by a draw
//    from max(p_c - q_c, 0).  u and the probabilities hold 24 bits, so the product of two is
//    exact in 64 and the decision is the formula's.
//  * Tree of proposed tokens (each its own point distribution): after node c the children are
//    tried in order, the first with u_c < p_c(x_1) + ... + p_c(x) is kept; where none is, the next
//    token is drawn from p_c without the children's tokens.
//  * Both draw the least v with r_0 + ... + r_v > u S, S = sum r.  S and the sums are in 64 bits:
//    the r of a large vocabulary lie closer together than sums in 32 bits resolve.
//
// What it cannot do without: the drafted tokens' probabilities (a gather), and one row of p (and
// q) a sequence, read once.  The rows are cut into slices of kSlice tokens, a workgroup each, so
// that one sequence's row is read by many CUs: every workgroup walks the sequence's tree itself
// (one gather of all nodes' probabilities, then register work), sums its slice and leaves the
// sum; the second launch finds the slice that holds u S and the token in it.
//
// 151936 tokens in fp32: 64 chains of 1 to 9 nodes 13.7 us (78 MB, 5.7 TB/s) and 4.5 for the second
// launch; 8 chains of 6 5.3 and 4.2, 16 trees of 26 7.5 and 4.4: chains of dependent loads (the
// offsets, the nodes, their probabilities, the row).
#include <float.h>

#include "dsp_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 4096;      // tokens of a row per workgroup
constexpr int kPerThread = kSlice / kThreads;
constexpr int kMaxNodes = 1024;   // nodes of one tree (their tokens and probabilities sit in LDS)

struct VBf16 { using store = uint16_t; };
struct VF16 { using store = uint16_t; };
struct VF32 { using store = float; };

template <typename Tag>
__device__ __forceinline__ float value(typename Tag::store x) {
  if constexpr (std::is_same<Tag, VBf16>::value)
    return dsp_bf16lo(x);
  else if constexpr (std::is_same<Tag, VF16>::value)
    return dsp_f16lo(x);
  else
    return x;
}

// What the first launch leaves for the second: the last kept node (-1: no nodes) and its row, the
// tokens kept before it, and the row of the draft's probabilities after it (-1: none was drafted).
struct Info {
  int32_t end, row, len, draft_row;
};
static_assert(sizeof(Info) == 16, "one load");

// One sequence's nodes: those of its first max_q_len that lie inside the rows.
struct Tree {
  int at;  // its first row
  int n;   // nodes (0: none)
};
__device__ __forceinline__ Tree tree_of(const int32_t* __restrict__ cu_q, int b, int max_q_len,
                                        int64_t rows) {
  const int at = cu_q[b];
  const int64_t n = min(min(int64_t(cu_q[b + 1]) - at, int64_t(max_q_len)), rows - at);
  return {at, at < 0 || n < 0 ? 0 : int(n)};
}

// The row of draft probabilities of sequence b's node 0: a sequence of n nodes has n - 1 of them,
// an empty one none.  (Every thread of the workgroup calls it.)
__device__ __forceinline__ int64_t first_draft_row(const int32_t* __restrict__ cu_q, int b) {
  int empty = 0;
  for (int j0 = 0; j0 < b; j0 += kThreads) {
    const int j = j0 + int(threadIdx.x);
    empty += __syncthreads_count(j < b && cu_q[j + 1] <= cu_q[j]);
  }
  return int64_t(cu_q[b]) - b + empty;
}

// A node's parent: the given one where it is an earlier node (else -1, and the node is never
// reached), or, in a chain, the node before it.
__device__ __forceinline__ int parent_of(const int32_t* __restrict__ parents, int at, int i) {
  if (i == 0) return -1;
  if (!parents) return i - 1;
  const int p = parents[at + i];
  return p >= 0 && p < i ? p : -1;
}

// r of token v of the row the next token is drawn from.
__device__ __forceinline__ double rest(float p, float q) {
  const double r = double(p) - double(q);
  return r > 0.0 ? r : 0.0;  // (NaN: 0)
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// One vector of 16 bytes of a row, at any element: rows of an odd vocabulary start anywhere, and
// the memory pipe takes 16-byte loads at any address of a whole element.
template <typename Tag>
struct Vec {
  static constexpr int N = 16 / int(sizeof(typename Tag::store));
  typedef typename Tag::store type
      __attribute__((ext_vector_type(16 / sizeof(typename Tag::store)),
                     aligned(sizeof(typename Tag::store))));
};

template <typename Tag>
__device__ __forceinline__ float at(const typename Vec<Tag>::type& v, int i) {
  return value<Tag>(v[i]);
}

template <typename Tag, bool kChain>
__global__ __launch_bounds__(kThreads) void verify_walk_kernel(
    const int64_t* __restrict__ tokens, const int32_t* __restrict__ parents,
    const typename Tag::store* __restrict__ target, int64_t ts, int64_t rows,
    const typename Tag::store* __restrict__ draft, int64_t ds, int64_t draft_rows,
    const float* __restrict__ u, const int32_t* __restrict__ cu_q, int32_t max_q_len, int64_t V,
    int32_t slices, double* __restrict__ sums, Info* __restrict__ info, int32_t* __restrict__ num,
    int32_t* __restrict__ path, int64_t* __restrict__ out_tokens,
    int32_t* __restrict__ err_count) {
  __shared__ int32_t s_par[kMaxNodes], s_tok[kMaxNodes], s_path[kMaxNodes];
  __shared__ float s_p[kMaxNodes], s_u[kMaxNodes];
  __shared__ int32_t s_len, s_any;
  __shared__ uint32_t s_kids[kSlice / 32];  // tokens of the slice that the last node's children hold
  __shared__ double s_sum[kThreads / 64];
  const int b = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const Tree t = tree_of(cu_q, b, max_q_len, rows);
  const int64_t dr = kChain ? first_draft_row(cu_q, b) : 0;
  // every node's probability after its parent (the chain: whether it is kept)
  for (int i = tid; i < t.n; i += kThreads) {
    const int par = parent_of(parents, t.at, i);
    const int64_t x = tokens[t.at + i];
    const bool ok = par >= 0 && x >= 0 && x < V && (!kChain || (dr >= 0 && dr + par < draft_rows));
    float p = 0.f;
    if (ok) {
      p = value<Tag>(target[(int64_t(t.at) + par) * ts + x]);
      if constexpr (kChain) {
        const float q = value<Tag>(draft[(dr + par) * ds + x]);
        p = double(u[t.at + par]) * double(q) < double(p) ? 1.f : 0.f;
      }
    }
    if constexpr (!kChain) s_u[i] = u[t.at + i];
    if (slice == 0 && par >= 0 && !ok && err_count) atomicAdd(err_count, 1);
    s_par[i] = par;
    s_tok[i] = ok ? int32_t(x) : -1;
    s_p[i] = p;
  }
  for (int i = tid; i < kSlice / 32; i += kThreads) s_kids[i] = 0u;
  if (tid == 0) s_any = 0;
  __syncthreads();
  if (tid < 64) {
    int len = 0;  // kept nodes besides the root
    int cur = 0;
    if (lane == 0) s_path[0] = 0;
    if constexpr (kChain) {
      for (int g = 0; g < t.n; g += 64) {
        const int i = g + lane;
        const uint64_t stop = __ballot(i > 0 && (i >= t.n || s_p[min(i, t.n - 1)] == 0.f));
        const int first = stop ? __ffsll(static_cast<unsigned long long>(stop)) - 1 : 64;
        if (i > 0 && lane < first) s_path[i] = i;
        len = g + first - 1;
        if (stop) break;
      }
      if (t.n == 0) len = 0;
      cur = len;
    } else {
      for (bool more = t.n > 0; more;) {
        more = false;
        const double coin = s_u[cur];
        double sum = 0.0;
        for (int g = 0; g < t.n && !more; g += 64) {
          const int i = min(g + lane, t.n - 1);
          const int par = g + lane < t.n ? s_par[i] : -1;
          const int tok = s_tok[i];
          const float p = s_p[i];
          uint64_t kids = __ballot(par == cur);
          while (kids) {
            const int l = __ffsll(static_cast<unsigned long long>(kids)) - 1;
            kids &= kids - 1;
            const int x = __shfl(tok, l);
            // a token that an earlier child holds counts once
            bool again = (__ballot(par == cur && tok == x && lane < l)) != 0;
            for (int h = 0; h < g && !again; h += 64)
              again = __ballot(s_par[h + lane] == cur && s_tok[h + lane] == x) != 0;
            const float px = __shfl(p, l);
            if (again || !(px > 0.f)) continue;
            sum += double(px);
            if (coin < sum) {
              cur = g + l;
              if (lane == 0) s_path[++len] = cur; else ++len;
              more = true;
              break;
            }
          }
        }
      }
    }
    if (lane == 0) s_len = t.n > 0 ? len : -1;
  }
  __syncthreads();
  const int len = s_len, end = len >= 0 ? s_path[len] : -1;
  if (slice == 0) {
    for (int i = tid; i < max_q_len; i += kThreads) {
      const int64_t o = int64_t(b) * max_q_len + i;
      path[o] = i <= len ? s_path[i] : -1;
      // (the token after the path is the second launch's)
      out_tokens[o] = i < len ? int64_t(s_tok[s_path[i + 1]]) : -1;
    }
  }
  // (nothing was drafted after a chain's last node)
  const bool with_q = kChain && end + 1 < t.n && dr >= 0 && dr + end < draft_rows;
  if (slice == 0 && tid == 0) {
    num[b] = max(len, 0);
    info[b] = Info{end, t.at + end, len, with_q ? int32_t(dr + end) : -1};
  }
  if (len < 0) return;
  const int64_t v0 = int64_t(slice) * kSlice;
  const int nv = int(min(int64_t(kSlice), V - v0));
  if constexpr (!kChain) {
    for (int i = tid; i < t.n; i += kThreads)
      if (s_par[i] == end && s_tok[i] >= v0 && s_tok[i] < v0 + nv) {
        atomicOr(&s_kids[(s_tok[i] - v0) >> 5], 1u << ((s_tok[i] - v0) & 31));
        s_any = 1;
      }
    __syncthreads();
  }
  const bool kids = !kChain && s_any != 0;
  const auto* p = target + (int64_t(t.at) + end) * ts + v0;
  const auto* q = with_q ? draft + (dr + end) * ds + v0 : p;
  using V16 = typename Vec<Tag>::type;
  constexpr int N = Vec<Tag>::N, R = kSlice / N / kThreads;
  double sum = 0.0;
  if (nv == kSlice) {
    V16 pv[R], qv[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      pv[r] = *reinterpret_cast<const V16*>(p + (tid + r * kThreads) * N);
      if (with_q) qv[r] = *reinterpret_cast<const V16*>(q + (tid + r * kThreads) * N);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int v = (tid + r * kThreads) * N + i;
        const bool kid = kids && ((s_kids[v >> 5] >> (v & 31)) & 1u);
        sum += kid ? 0.0 : rest(at<Tag>(pv[r], i), with_q ? at<Tag>(qv[r], i) : 0.f);
      }
  } else {
    for (int v = tid; v < nv; v += kThreads) {
      const bool kid = kids && ((s_kids[v >> 5] >> (v & 31)) & 1u);
      sum += kid ? 0.0 : rest(value<Tag>(p[v]), with_q ? value<Tag>(q[v]) : 0.f);
    }
  }
  sum = wave_sum(sum);
  if (lane == 0) s_sum[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) all += s_sum[w];
    sums[int64_t(b) * slices + slice] = all;
  }
}

// Inclusive sums over a wave's lanes, in their order.
__device__ __forceinline__ double wave_scan(double v) {
  const int lane = __lane_id();
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// One workgroup a sequence.  It is a chain of loads, each of which names the next (what the walk
// left, the slices' sums, the slice's tokens), so the first are sent for together, every wave scans
// the sums by itself (64 slices at a time: one step for 262144 tokens) and the workgroup meets
// twice.
template <typename Tag, bool kChain>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(
    const int64_t* __restrict__ tokens, const int32_t* __restrict__ parents,
    const typename Tag::store* __restrict__ target, int64_t ts, int64_t rows,
    const typename Tag::store* __restrict__ draft, int64_t ds, const float* __restrict__ u_last,
    const int32_t* __restrict__ cu_q, int32_t max_q_len, int64_t V, int32_t slices,
    double* __restrict__ sums, const Info* __restrict__ info, int64_t* __restrict__ out_tokens,
    int32_t* __restrict__ err_count) {
  constexpr int kWaves = kThreads / 64;
  __shared__ double s_wave[kWaves];
  __shared__ int32_t s_first[kWaves], s_last[kWaves];
  __shared__ uint32_t s_kids[kSlice / 32];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  double* mine = sums + int64_t(b) * slices;
  auto sum_of = [&](int s) { return s < slices ? mine[s] : 0.0; };
  double v0 = sum_of(lane);   // the first 64 slices' sums
  const Info seq = info[b];
  const double u = u_last[b];
  const Tree t = kChain ? Tree{0, 0} : tree_of(cu_q, b, max_q_len, rows);
  if (seq.len < 0) return;
  // the last node's children: this thread's nodes
  constexpr int kNodes = kMaxNodes / kThreads;
  int32_t kid[kNodes];
  if constexpr (!kChain) {
#pragma unroll
    for (int i = 0; i < kNodes; ++i) {
      const int at = tid + i * kThreads;
      kid[i] = -1;
      if (at < t.n && parent_of(parents, t.at, at) == seq.end) {
        const int64_t x = tokens[t.at + at];
        kid[i] = x >= 0 && x < V ? int32_t(x) : -1;
      }
    }
    for (int i = tid; i < kSlice / 32; i += kThreads) s_kids[i] = 0u;
  }
  const bool with_q = kChain && seq.draft_row >= 0;
  const auto* prow = target + int64_t(seq.row) * ts;
  const auto* qrow = with_q ? draft + int64_t(seq.draft_row) * ds : prow;
  // this thread's tokens of a slice: kPerThread in a row
  double r[kPerThread];
  auto load = [&](int slice, bool whole) {
    const int64_t first = int64_t(slice) * kSlice;
    const int nv = int(min(int64_t(kSlice), V - first));
    const bool sub = with_q && !whole;
    float pf[kPerThread], qf[kPerThread];
    const int v1 = tid * kPerThread;
    if (v1 + kPerThread <= nv) {
      using V16 = typename Vec<Tag>::type;
      constexpr int N = Vec<Tag>::N;
#pragma unroll
      for (int j = 0; j < kPerThread / N; ++j) {
        const V16 pv = *reinterpret_cast<const V16*>(prow + first + v1 + j * N);
        V16 qv = pv;
        if (sub) qv = *reinterpret_cast<const V16*>(qrow + first + v1 + j * N);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          pf[j * N + i] = at<Tag>(pv, i);
          qf[j * N + i] = sub ? at<Tag>(qv, i) : 0.f;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        const bool in = v1 + i < nv;
        pf[i] = in ? value<Tag>(prow[first + v1 + i]) : 0.f;
        qf[i] = in && sub ? value<Tag>(qrow[first + v1 + i]) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) r[i] = rest(pf[i], qf[i]);
  };
  auto slice_sum = [&]() {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) s += r[i];
    return s;
  };
  // the first 64 slices' running sums and the total of all
  double upto0, all;
  auto total_of = [&]() {
    upto0 = wave_scan(v0);
    all = __shfl(upto0, 63);
    for (int s0 = 64; s0 < slices; s0 += 64) all += wave_sum(sum_of(s0 + lane));
  };
  total_of();
  bool whole = false;
  if (!(all > 0.0)) {
    // nothing is left over (the rows are equal, or the children hold all of it): from the whole
    // row of p
    whole = true;
    __syncthreads();  // every wave has read the sums
    for (int s = 0; s < slices; ++s) {
      load(s, true);
      const double part = wave_sum(slice_sum());
      if (lane == 0) s_wave[wave] = part;
      __syncthreads();
      if (tid == 0) {
        double sum = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += s_wave[w];
        mine[s] = sum;
      }
      __syncthreads();
    }
    v0 = sum_of(lane);
    total_of();
  }
  if (!(all > 0.0 && all <= DBL_MAX)) {
    // a row without a positive, finite sum: no token
    if (tid == 0) {
      if (err_count) atomicAdd(err_count, 1);
      out_tokens[int64_t(b) * max_q_len + seq.len] = -1;
    }
    return;
  }
  const double goal = u * all;
  // the first slice whose sums pass the goal, and the sum before it; where rounding or a u of 1
  // leaves none, the last slice that holds anything
  int slice = -1;
  bool found = false;
  double before = 0.0, upto = upto0, v = v0, ahead = 0.0;
  for (int s0 = 0; !found; ) {
    const uint64_t some = __ballot(v > 0.0), hit = __ballot(v > 0.0 && upto > goal);
    found = hit != 0;
    const int l = found ? __ffsll(static_cast<unsigned long long>(hit)) - 1
                        : (some ? 63 - __clzll(static_cast<long long>(some)) : -1);
    if (l >= 0) {
      slice = s0 + l;
      before = l > 0 ? __shfl(upto, l - 1) : ahead;
    }
    ahead = __shfl(upto, 63);
    s0 += 64;
    if (s0 >= slices) break;
    if (!found) {
      v = sum_of(s0 + lane);
      upto = ahead + wave_scan(v);
    }
  }
  load(slice, whole);
  if constexpr (!kChain) {
    if (!whole) {
      // tokens that the children hold count for nothing
      __syncthreads();  // s_kids is clear
      const int64_t first = int64_t(slice) * kSlice;
#pragma unroll
      for (int i = 0; i < kNodes; ++i)
        if (kid[i] >= first && kid[i] < first + kSlice)
          atomicOr(&s_kids[(kid[i] - first) >> 5], 1u << ((kid[i] - first) & 31));
      __syncthreads();
      static_assert(kPerThread == 16, "a thread's tokens lie in one word of s_kids");
      const uint32_t kids = s_kids[(tid * kPerThread) >> 5] >> (tid * kPerThread & 31);
#pragma unroll
      for (int i = 0; i < kPerThread; ++i)
        if ((kids >> i) & 1u) r[i] = 0.0;
    }
  }
  const double own = slice_sum(), upto_own = wave_scan(own);
  if (lane == 63) s_wave[wave] = upto_own;
  __syncthreads();
  double run = before;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) run += w < wave ? s_wave[w] : 0.0;
  run += upto_own - own;
  int first = -1, last = -1;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    run += r[i];
    if (r[i] > 0.0) {
      if (first < 0 && run > goal) first = tid * kPerThread + i;
      last = tid * kPerThread + i;
    }
  }
  const uint64_t firsts = __ballot(found && first >= 0), lasts = __ballot(last >= 0);
  first = firsts ? __shfl(first, __ffsll(static_cast<unsigned long long>(firsts)) - 1) : -1;
  last = lasts ? __shfl(last, 63 - __clzll(static_cast<long long>(lasts))) : -1;
  if (lane == 0) {
    s_first[wave] = first;
    s_last[wave] = last;
  }
  __syncthreads();
  if (tid == 0) {
    first = -1;
    last = -1;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (first < 0) first = s_first[w];
      if (s_last[w] >= 0) last = s_last[w];
    }
    out_tokens[int64_t(b) * max_q_len + seq.len] =
        int64_t(slice) * kSlice + (first >= 0 ? first : last);
  }
}

// The tokens that the target chose after each node are known: a node is kept where its token is
// the one chosen after its parent.  One wave a sequence: 32 trees of 1 to 61 nodes 3.0 us, three
// dependent loads.
__global__ __launch_bounds__(64) void match_kernel(
    const int64_t* __restrict__ tokens, const int64_t* __restrict__ choice,
    const int32_t* __restrict__ parents, const int32_t* __restrict__ cu_q, int64_t rows,
    int32_t max_q_len, int32_t* __restrict__ num, int32_t* __restrict__ path,
    int64_t* __restrict__ out_tokens) {
  __shared__ int32_t s_par[kMaxNodes];  // the parent of a node that its parent's choice names
  __shared__ int32_t s_path[kMaxNodes];
  const int b = blockIdx.x, lane = threadIdx.x;
  const Tree t = tree_of(cu_q, b, max_q_len, rows);
  for (int i = lane; i < t.n; i += 64) {
    const int par = parent_of(parents, t.at, i);
    s_par[i] = par >= 0 && tokens[t.at + i] == choice[t.at + par] ? par : -1;
  }
  if (lane == 0) s_path[0] = 0;
  __syncthreads();
  int cur = 0, len = 0;
  // (children come after their parents: the search goes on where it stands)
  for (int g = 0; g < t.n;) {
    const int i = g + lane;
    const uint64_t hit = __ballot(i < t.n && i > cur && s_par[min(i, t.n - 1)] == cur);
    if (!hit) {
      g += 64;
      continue;
    }
    cur = g + __ffsll(static_cast<unsigned long long>(hit)) - 1;
    ++len;
    if (lane == 0) s_path[len] = cur;
  }
  __syncthreads();
  for (int i = lane; i < max_q_len; i += 64) {
    const int64_t o = int64_t(b) * max_q_len + i;
    const bool in = t.n > 0 && i <= len;
    path[o] = in ? s_path[i] : -1;
    out_tokens[o] = in ? choice[t.at + s_path[i]] : -1;
  }
  if (lane == 0) num[b] = len;
}

int64_t slices_of(int64_t V) { return (V + kSlice - 1) / kSlice; }

template <typename Tag, bool kChain>
int launch_verify(const int64_t* tokens, const int32_t* parents, const void* target, int64_t ts,
                  int64_t rows, const void* draft, int64_t ds, int64_t draft_rows, const float* u,
                  const float* u_last, const int32_t* cu_q, int32_t B, int32_t max_q_len,
                  int64_t V, void* workspace,
                  int32_t* num, int32_t* path, int64_t* out_tokens, int32_t* err_count,
                  hipStream_t s) {
  using S = typename Tag::store;
  const int slices = int(slices_of(V));
  Info* info = reinterpret_cast<Info*>(workspace);
  double* sums = reinterpret_cast<double*>(info + B);
  verify_walk_kernel<Tag, kChain>
      <<<dim3(unsigned(slices), unsigned(B)), kThreads, 0, s>>>(
          tokens, parents, static_cast<const S*>(target), ts, rows, static_cast<const S*>(draft),
          ds, draft_rows, u, cu_q, max_q_len, V, slices, sums, info, num, path, out_tokens,
          err_count);
  const int st = dsp_launch_status();
  if (st != DSP_OK) return st;
  verify_pick_kernel<Tag, kChain><<<unsigned(B), kThreads, 0, s>>>(
      tokens, parents, static_cast<const S*>(target), ts, rows, static_cast<const S*>(draft), ds,
      u_last, cu_q, max_q_len, V, slices, sums, info, out_tokens, err_count);
  return dsp_launch_status();
}

template <bool kChain, typename... A>
int launch_verify_type(int32_t dtype, A... args) {
  switch (dtype) {
    case DSP_BF16: return launch_verify<VBf16, kChain>(args...);
    case DSP_F16: return launch_verify<VF16, kChain>(args...);
    default: return launch_verify<VF32, kChain>(args...);
  }
}

}  // namespace

extern "C" size_t dsp_verify_workspace_bytes(int32_t B, int64_t V) {
  if (B <= 0 || V <= 0) return 0;
  return size_t(B) * (size_t(slices_of(V)) * sizeof(double) + sizeof(Info));
}

extern "C" int dsp_verify_draft(const int64_t* draft_tokens, const int32_t* parents,
                                const void* target_probs, int64_t target_stride, int64_t num_rows,
                                const void* draft_probs, int64_t draft_stride,
                                int64_t num_draft_rows, const float* uniforms,
                                const float* final_uniforms, const int32_t* cu_q, int32_t B,
                                int32_t max_q_len, int64_t V,
                                int32_t dtype, void* workspace, size_t workspace_bytes,
                                int32_t* num_accepted, int32_t* path, int64_t* tokens,
                                int32_t* err_count, dsp_stream_t stream) {
  DSP_HOST_CHECK(draft_tokens && target_probs && uniforms && final_uniforms && cu_q &&
                     num_accepted && path && tokens,
                 DSP_EINVAL);
  DSP_HOST_CHECK(B >= 0 && B <= 65535 && max_q_len >= 0 && V > 0 && num_rows >= 0 &&
                     num_draft_rows >= 0 && target_stride >= 0 && draft_stride >= 0,
                 DSP_EINVAL);
  DSP_HOST_CHECK(!(parents && draft_probs), DSP_EINVAL);  // draft probabilities: a chain
  DSP_HOST_CHECK(dtype == DSP_BF16 || dtype == DSP_F16 || dtype == DSP_F32, DSP_EUNSUPPORTED);
  DSP_HOST_CHECK(max_q_len <= kMaxNodes && V < (int64_t(1) << 31), DSP_EUNSUPPORTED);
  if (B == 0 || max_q_len == 0) return DSP_OK;
  const int64_t es = dtype == DSP_F32 ? 4 : 2;
  DSP_HOST_CHECK(dsp_aligned(target_probs, es) && (!draft_probs || dsp_aligned(draft_probs, es)),
                 DSP_EALIGN);
  DSP_HOST_CHECK(workspace && workspace_bytes >= dsp_verify_workspace_bytes(B, V),
                 DSP_EWORKSPACE);
  DSP_HOST_CHECK(dsp_aligned(workspace, 16), DSP_EALIGN);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (draft_probs)
    return launch_verify_type<true>(dtype, draft_tokens, parents, target_probs, target_stride,
                                    num_rows, draft_probs, draft_stride, num_draft_rows, uniforms,
                                    final_uniforms, cu_q, B, max_q_len, V, workspace, num_accepted,
                                    path, tokens, err_count, s);
  return launch_verify_type<false>(dtype, draft_tokens, parents, target_probs, target_stride,
                                   num_rows, draft_probs, draft_stride, num_draft_rows, uniforms,
                                   final_uniforms, cu_q, B, max_q_len, V, workspace, num_accepted,
                                   path, tokens, err_count, s);
}

extern "C" int dsp_match_draft(const int64_t* draft_tokens, const int64_t* target_tokens,
                               const int32_t* parents, const int32_t* cu_q, int64_t num_rows,
                               int32_t B, int32_t max_q_len, int32_t* num_accepted, int32_t* path,
                               int64_t* tokens, dsp_stream_t stream) {
  DSP_HOST_CHECK(draft_tokens && target_tokens && cu_q && num_accepted && path && tokens,
                 DSP_EINVAL);
  DSP_HOST_CHECK(B >= 0 && max_q_len >= 0 && num_rows >= 0, DSP_EINVAL);
  DSP_HOST_CHECK(max_q_len <= kMaxNodes, DSP_EUNSUPPORTED);
  if (B == 0 || max_q_len == 0) return DSP_OK;
  match_kernel<<<unsigned(B), 64, 0, static_cast<hipStream_t>(stream)>>>(
      draft_tokens, target_tokens, parents, cu_q, num_rows, max_q_len, num_accepted, path, tokens);
  return dsp_launch_status();
}
