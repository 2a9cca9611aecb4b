// A teacher's k largest logits, and the loss of a student against them with
// its gradient, gfx950.
//
// topk: the k largest of a row, largest first, equal ones by lowest index,
// and rest = log sum exp(t_i / T) over the classes that were not taken.
//
// distill: with u_j = v_j / T of the slots that name a class, the teacher's
// answer is q = softmax over (u_1 .. u_k, rest): one probability for each
// named class and one, q_r, for all others together. The student's is
// p = softmax(z / T), p_r its sum over the classes that no slot names.
//
//   loss = sum_j q_j log(q_j / p_{i_j}) + q_r log(q_r / p_r)
//   dz_i = (g / T) (p_i - sum of the q_j that name i)     i named
//   dz_i = (g / T) p_i (1 - q_r / p_r)                    the rest
//
// The rest has a maximum and a sum of its own: as 1 - (what is named) it
// would lose all its digits where a few classes hold nearly everything. The
// loss is summed as q log(q / p) - q + p, whose terms do not cancel where the
// two answers are near to each other; q and p both sum to one, so the sum is
// the same.
//
// One block takes a row. All sums are made in a fixed order: the same inputs
// give the same bits.

#include "common.h"
#include "distill.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;

// Sum of exp2((z - m) c) over a set of z, with the set's largest for m. An
// empty set, or one of -inf alone, is {kLowest, 0}.
struct Sum {
  float m, s;
};

// One instruction; results below 2^-126 are 0.
DFD_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

DFD_DEV void add(Sum& a, float z, float c) {
  if (z > a.m) {
    a.s = a.s * exp2_fast((a.m - z) * c) + 1.f;
    a.m = z;
  } else {
    // equal: also where both are +inf, whose difference is no number
    a.s += z == a.m ? 1.f : exp2_fast((z - a.m) * c);
  }
}

DFD_DEV Sum join(const Sum& a, const Sum& b, float c) {
  if (a.m == b.m) return {a.m, a.s + b.s};
  return a.m > b.m ? Sum{a.m, a.s + b.s * exp2_fast((b.m - a.m) * c)}
                   : Sum{b.m, b.s + a.s * exp2_fast((a.m - b.m) * c)};
}

DFD_DEV Sum wave_join(Sum v, float c) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    const Sum o = {__shfl_xor(v.m, off), __shfl_xor(v.s, off)};
    v = lane & off ? join(o, v, c) : join(v, o, c);
  }
  return v;
}

// Every thread gets the block's sum.
template <int THREADS>
DFD_DEV Sum block_join(Sum v, float c, Sum* lds) {
  v = wave_join(v, c);
  if (THREADS == kWave) return v;
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = lds[0];
  for (int w = 1; w < THREADS / kWave; ++w) v = join(v, lds[w], c);
  return v;
}

// A row as aligned vectors: head elements before the first one, body vectors,
// tail elements after the last.
template <typename T, int VEC>
struct Row {
  const T* p;
  int head, body, tail;
  DFD_DEV Row(const T* row, int n) : p(row) {
    const unsigned off = (unsigned)(reinterpret_cast<unsigned long long>(row) % (VEC * sizeof(T)));
    head = off ? (int)((VEC * sizeof(T) - off) / sizeof(T)) : 0;
    if (head > n) head = n;
    body = (n - head) / VEC;
    tail = n - head - body * VEC;
  }
  DFD_DEV DfdVec<T, VEC> load(int v) const { return dfd_vload<T, VEC>(p + head + (long long)v * VEC); }
  DFD_DEV DfdVec<T, VEC> load_once(int v) const {
    return dfd_vload_once<T, VEC>(p + head + (long long)v * VEC);
  }
  DFD_DEV int first(int v) const { return head + v * VEC; }
  DFD_DEV int edges() const { return head + tail; }
  DFD_DEV int edge(int e) const { return e < head ? e : head + body * VEC + (e - head); }
  DFD_DEV float at(int i) const { return DfdCvt<T>::to_f32(p[i]); }
};

// f(vector, its number) for the thread's vectors of a row. Four loads are in
// flight at a time; those beyond the row load its last vector again and are
// dropped, which costs less than a branch around each. ONCE: past the caches.
template <int THREADS, bool ONCE, typename T, int VEC, typename F>
DFD_DEV void stream(const Row<T, VEC>& row, F f) {
  constexpr int U = 4;
  for (int v = threadIdx.x; v < row.body; v += U * THREADS) {
    DfdVec<T, VEC> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int w = v + u * THREADS;
      const int at = w < row.body ? w : row.body - 1;
      x[u] = ONCE ? row.load_once(at) : row.load(at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * THREADS < row.body) f(x[u], v + u * THREADS);
  }
}

// The sum of a stream of vectors at one exponential a value. The exponent is
// the difference times c, for every finite value as near as a product's
// rounding leaves it; z c less a rounded m c would be one instruction fewer
// (8192 x 32000 bf16, the loss: 93 us, and 94 so), but from |m c| of 2^31 on
// that rounding alone takes the sum beyond fp32. A NaN or +inf makes the sum a
// NaN.
struct FastSum {
  Sum sum = {kLowest, 0.f};
  template <int N>
  DFD_DEV void add(const float (&z)[N], float c) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
    if (top > sum.m) {
      sum.s *= exp2_fast((sum.m - top) * c);
      sum.m = top;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) sum.s += exp2_fast((z[i] - sum.m) * c);
  }
};

template <typename T, int VEC>
DFD_DEV void to_floats(const DfdVec<T, VEC>& x, float (&z)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) z[i] = DfdCvt<T>::to_f32(x.v[i]);
}

// Order-preserving keys: any NaN is the largest, -0 and 0 are equal, and 0 is
// below every value's key.
DFD_DEV unsigned key_of(float f) {
  if (f != f) return 0xffffffffu;
  const unsigned u = f == 0.f ? 0u : __float_as_uint(f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// The leading bits of a key that can differ from the rest of it.
template <typename T> constexpr int key_bits() { return 32; }
template <> constexpr int key_bits<__hip_bfloat16>() { return 16; }
template <> constexpr int key_bits<__half>() { return 19; }

constexpr unsigned kOffKey = ~0xff800000u;  // the key of -inf

// The place of each thread that says yes among them, in thread order.
template <int THREADS>
DFD_DEV int block_rank(bool yes, int* lds, int& total) {
  const unsigned long long mask = __ballot(yes);
  const int lane = threadIdx.x & (kWave - 1);
  const int wid = threadIdx.x / kWave;
  int rank = __popcll(mask & ((1ull << lane) - 1));
  if (THREADS == kWave) {
    total = __popcll(mask);
    return rank;
  }
  __syncthreads();  // lds may still be read
  if (lane == 0) lds[wid] = __popcll(mask);
  __syncthreads();
  total = 0;
  for (int w = 0; w < THREADS / kWave; ++w) {
    if (w == wid) rank += total;
    total += lds[w];
  }
  return rank;
}

// ---------------------------------------------------------------------------
// topk
// ---------------------------------------------------------------------------
//
// One pass over the row: every thread takes its vectors in up to kParts parts
// and keeps the largest value and the sum of each. A key that k of the threads'
// largest reach is at most the row's k-th largest: what lies below that bound
// is not taken. Only the parts whose largest reaches it (about k of
// them) hold candidates; their elements are read again, from the cache, by all
// threads together, and sorted into candidates and rest. A candidate's rank is
// the number of greater ones. -inf is no candidate (nothing is said of a class
// that is switched off), so a row may have fewer than k.
//
// Many values equal to the bound can leave more candidates than fit; then the
// row is searched as a whole (topk_wide).

constexpr int kParts = 8;

template <int THREADS>
constexpr int topk_cap() {
  return THREADS == 64 ? 512 : 1024;
}

template <int THREADS>
struct TopkLds {
  unsigned long long cand[topk_cap<THREADS>()];
  float left[topk_cap<THREADS>()];  // candidates that were not taken, by rank
  unsigned short hot[THREADS * kParts];  // part * THREADS + thread
  Sum sums[THREADS / kWave];
  int counts[THREADS / kWave];
  unsigned bounds[THREADS / kWave];
  int n;
};

// A key that at least k of the threads' keys reach, near to the largest such:
// each wave finds its own (k / waves)-th largest by counting lanes, bit by bit,
// and the least of these is taken. (The block's k-th largest itself takes a
// barrier for each bit: by 256 threads 39 us for 2961 x 9591 fp16, k = 23, and
// 31 so.)
template <int THREADS, int BITS>
DFD_DEV unsigned topk_bound(unsigned key, int k, unsigned* lds) {
  constexpr int kWaves = THREADS / kWave;
  const int own = (k + kWaves - 1) / kWaves;
  unsigned bound = 0;
  for (int b = 31; b > 31 - BITS; --b) {
    const unsigned test = bound | (1u << b);
    const int n = __popcll(__ballot(key >= test));
    if (n >= own) bound = test;
    if (n == own) break;
  }
  if (kWaves > 1) {
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = bound;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) bound = lds[w] < bound ? lds[w] : bound;
  }
  // the bits that a narrow type does not have are ones in a negative value's key
  return bound >> 31 ? bound : bound | (unsigned)((1ull << (32 - BITS)) - 1);
}

template <int THREADS>
DFD_DEV int block_total(int mine, int& lds) {
  __syncthreads();
  if (threadIdx.x == 0) lds = 0;
  __syncthreads();
  if (mine) atomicAdd(&lds, mine);
  __syncthreads();
  return lds;
}

// Fills lds.cand with exactly the k to take; returns the sum of this thread's
// share of the others. At least k keys reach bound, which is no -inf.
template <typename T, int THREADS>
DFD_DEV Sum topk_wide(const T* row, int classes, int k, float c, unsigned bound,
                      TopkLds<THREADS>& lds) {
  const int tid = threadIdx.x;
  auto above = [&](unsigned key) {
    int mine = 0;
    for (int i = tid; i < classes; i += THREADS) mine += key_of(DfdCvt<T>::to_f32(row[i])) > key;
    return block_total<THREADS>(mine, lds.n);
  };
  // the k-th largest key: the bound itself if values equal to it are what
  // there are many of, or else by bisection
  unsigned kth = bound;
  if (above(bound) >= k) {
    kth = 0;
    for (int b = 31; b >= 0; --b) {
      const unsigned test = kth | (1u << b);
      if (above(test - 1) >= k) kth = test;
    }
  }
  __syncthreads();
  if (tid == 0) lds.n = 0;
  __syncthreads();
  for (int i = tid; i < classes; i += THREADS) {
    const unsigned key = key_of(DfdCvt<T>::to_f32(row[i]));
    if (key > kth) {  // fewer than k of them
      const int at = atomicAdd(&lds.n, 1);
      lds.cand[at] = ((unsigned long long)key << 32) | (unsigned)~i;
    }
  }
  __syncthreads();
  int have = lds.n;
  for (int base = 0; have < k; base += THREADS) {
    const int i = base + tid;
    const bool equal = i < classes && key_of(DfdCvt<T>::to_f32(row[i])) == kth;
    int total;
    const int at = have + block_rank<THREADS>(equal, lds.counts, total);
    if (equal && at < k) lds.cand[at] = ((unsigned long long)kth << 32) | (unsigned)~i;
    have += total;
  }
  __syncthreads();
  if (tid == 0) lds.n = k;
  // of the last tile some may be left over: those after the last one taken
  unsigned lowest = 0xffffffffu;
  for (int i = tid; i < k; i += THREADS)
    if ((unsigned)(lds.cand[i] >> 32) == kth) {
      const unsigned inv = (unsigned)lds.cand[i];
      lowest = inv < lowest ? inv : lowest;
    }
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    const unsigned o = __shfl_xor(lowest, off);
    lowest = o < lowest ? o : lowest;
  }
  __syncthreads();
  if ((tid & (kWave - 1)) == 0) lds.counts[tid / kWave] = (int)lowest;
  __syncthreads();
  for (int w = 0; w < THREADS / kWave; ++w)
    lowest = (unsigned)lds.counts[w] < lowest ? (unsigned)lds.counts[w] : lowest;
  const int last = (int)~lowest;  // the highest index taken of those equal to kth
  Sum mine = {kLowest, 0.f};
  for (int i = tid; i < classes; i += THREADS) {
    const float z = DfdCvt<T>::to_f32(row[i]);
    const unsigned key = key_of(z);
    if (key < kth || (key == kth && i > last)) add(mine, z, c);
  }
  return mine;
}

template <typename T, int VEC, int THREADS>
__global__ __launch_bounds__(THREADS) void topk_kernel(
    const T* __restrict__ logits, long long row_stride, int classes, int k, float inv_t,
    T* __restrict__ values, long long* __restrict__ indices, float* __restrict__ rest) {
  __shared__ TopkLds<THREADS> lds;
  constexpr int kCap = topk_cap<THREADS>();
  constexpr int kBits = key_bits<T>();
  const int tid = threadIdx.x;
  const long long r = blockIdx.x;
  const T* p = logits + r * row_stride;
  const Row<T, VEC> row(p, classes);
  const float c = inv_t * kLog2e;

  // part q: vectors from q * step on, `per` for each thread
  constexpr int U = 4;
  const int rounds = (row.body + U * kParts * THREADS - 1) / (U * kParts * THREADS);
  const int per = U * (rounds > 0 ? rounds : 1);
  const int step = per * THREADS;
  Sum part[kParts];  // {largest value, sum}
#pragma unroll
  for (int q = 0; q < kParts; ++q) {
    part[q] = {-__builtin_inff(), 0.f};
    if (q * step >= row.body) continue;  // the same for the whole block
    const int end = (q + 1) * step < row.body ? (q + 1) * step : row.body;
    FastSum fast;
    for (int v = q * step + tid; v < end; v += U * THREADS) {
      DfdVec<T, VEC> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int w = v + u * THREADS;
        x[u] = row.load(w < end ? w : end - 1);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + u * THREADS < end) {
          float z[VEC];
          to_floats(x[u], z);
          fast.add(z, c);
        }
    }
    // (the largest of a set counts as 1, so an empty sum has seen -inf alone)
    if (fast.sum.s != 0.f) part[q] = fast.sum;
    if (part[q].s != part[q].s) {  // a NaN or +inf among them
      part[q] = {-__builtin_inff(), 0.f};
      for (int v = q * step + tid; v < end; v += THREADS)
        for (int i = 0; i < VEC; ++i) add(part[q], row.at(row.first(v) + i), c);
    }
  }
  // a NaN leaves its mark in the sum alone
  auto key_of_part = [&](int q) { return part[q].s != part[q].s ? 0xffffffffu : key_of(part[q].m); };
  unsigned key = 0;
  if (tid < row.body) {
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      const unsigned o = key_of_part(q);
      key = o > key ? o : key;
    }
  }
  if (tid == 0) lds.n = 0;
  const unsigned bound = topk_bound<THREADS, kBits>(key, k, lds.bounds);

  // the hot parts' list, in a fixed order; the sum of the others
  Sum mine = {kLowest, 0.f};
  unsigned hot = 0;
  int before = 0, count = 0;  // hot parts of lower lanes, and of the wave
#pragma unroll
  for (int q = 0; q < kParts; ++q) {
    const unsigned o = key_of_part(q);
    const bool is = o >= bound && o > kOffKey;
    if (is) hot |= 1u << q;
    else if (part[q].s > 0.f) mine = join(mine, part[q], c);
    const unsigned long long all = __ballot(is);
    before += __popcll(all & ((1ull << (tid & (kWave - 1))) - 1));
    count += __popcll(all);
  }
  int nhot = count;
  if (THREADS > kWave) {
    if ((tid & (kWave - 1)) == 0) lds.counts[tid / kWave] = count;
    __syncthreads();
    nhot = 0;
    for (int w = 0; w < THREADS / kWave; ++w) {
      if (w == tid / kWave) before += nhot;
      nhot += lds.counts[w];
    }
  }
#pragma unroll
  for (int q = 0; q < kParts; ++q)
    if (hot >> q & 1) lds.hot[before++] = (unsigned short)(q * THREADS + tid);
  __syncthreads();
  auto sift = [&](float z, int i) {
    const unsigned o = key_of(z);
    if (o >= bound && o > kOffKey) {
      const int at = atomicAdd(&lds.n, 1);
      if (at < kCap) lds.cand[at] = ((unsigned long long)o << 32) | (unsigned)~i;
    } else {
      add(mine, z, c);
    }
  };
  for (int w = tid; w < nhot * per; w += THREADS) {
    const int h = w / per;
    const int q = lds.hot[h] / THREADS;
    const int v = q * step + (w - h * per) * THREADS + lds.hot[h] % THREADS;
    if (v < row.body) {
      const DfdVec<T, VEC> x = row.load(v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sift(DfdCvt<T>::to_f32(x.v[i]), row.first(v) + i);
    }
  }
  for (int e = tid; e < row.edges(); e += THREADS) sift(row.at(row.edge(e)), row.edge(e));
  __syncthreads();
  if (lds.n > kCap) {
    mine = topk_wide<T, THREADS>(p, classes, k, c, bound, lds);
    __syncthreads();
  }
  const int n = lds.n;
  for (int i = tid; i < n; i += THREADS) {
    const unsigned long long own = lds.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += lds.cand[j] > own;
    const int at = (int)~(unsigned)own;
    if (rank < k) {
      const T x = p[at];
      values[r * k + rank] = x;
      indices[r * k + rank] = at;
    } else {
      lds.left[rank - k] = row.at(at);
    }
  }
  for (int i = n + tid; i < k; i += THREADS) {
    values[r * k + i] = DfdCvt<T>::from_f32(-__builtin_inff());
    indices[r * k + i] = -1;
  }
  __syncthreads();
  for (int i = tid; i < n - k; i += THREADS) add(mine, lds.left[i], c);
  const Sum all = block_join<THREADS>(mine, c, lds.sums);
  if (tid == 0) rest[r] = all.s == 0.f ? -__builtin_inff() : all.m * inv_t + logf(all.s);
}

// ---------------------------------------------------------------------------
// distill
// ---------------------------------------------------------------------------

DFD_DEV float load_as(const void* p, LogitType type, long long i) {
  switch (type) {
    case LogitType::kBf16:
      return DfdCvt<__hip_bfloat16>::to_f32(static_cast<const __hip_bfloat16*>(p)[i]);
    case LogitType::kF16: return DfdCvt<__half>::to_f32(static_cast<const __half*>(p)[i]);
    default: return static_cast<const float*>(p)[i];
  }
}

// What the backward pass needs of a row.
struct RowStats {
  float m_rest, coef;   // rest: dz = (g / T) coef exp2((z - m_rest) c)
  float m, inv_s;       // named: p = exp2((z - m) c) inv_s
  float u_top, inv_q;   // q_j = exp(u_j - u_top) inv_q
  float state, unused;
};
static_assert(sizeof(RowStats) == kDistillStats * sizeof(float), "stats");

constexpr float kTeaches = 0.f, kTwice = 1.f, kNothing = 2.f, kBadIndex = 3.f;

template <typename T, int VEC, int THREADS, bool ONCE>
__global__ __launch_bounds__(THREADS) void distill_fwd_kernel(
    const T* __restrict__ logits, long long row_stride, int classes, int k, float inv_t,
    const void* __restrict__ values, LogitType vtype, const long long* __restrict__ indices,
    const float* __restrict__ rest, float* __restrict__ loss, RowStats* __restrict__ stats) {
  extern __shared__ unsigned bits[];  // one for each class: named by a slot
  __shared__ int s_index[kMaxTopK];
  __shared__ float s_u[kMaxTopK], s_z[kMaxTopK];
  __shared__ unsigned char s_first[kMaxTopK];  // the first slot that names its class
  __shared__ Sum sums[THREADS / kWave];
  __shared__ int twice, bad;
  const int tid = threadIdx.x;
  const long long r = blockIdx.x;
  const Row<T, VEC> row(logits + r * row_stride, classes);
  const float c = inv_t * kLog2e;
  // a vector's bits begin at a multiple of VEC
  const int pad = row.head ? VEC - row.head : 0;
  const int words = (classes + pad + 31) / 32;
  for (int i = tid; i < words; i += THREADS) bits[i] = 0;
  if (tid == 0) twice = bad = 0;
  __syncthreads();
  for (int j = tid; j < k; j += THREADS) {
    const long long at = indices[r * k + j];
    const bool in = at >= 0 && at < classes;
    s_index[j] = in ? (int)at : -1;
    s_u[j] = in ? load_as(values, vtype, r * k + j) * inv_t : -__builtin_inff();
    s_z[j] = in ? row.at((int)at) : -__builtin_inff();
    s_first[j] = 1;
    if (at >= classes) bad = 1;
    if (in) {
      const unsigned b = (unsigned)at + pad;
      if (atomicOr(&bits[b / 32], 1u << (b % 32)) >> (b % 32) & 1) twice = 1;
    }
  }
  __syncthreads();
  if (twice)
    for (int j = tid; j < k; j += THREADS)
      for (int i = 0; i < j; ++i)
        if (s_index[i] == s_index[j]) s_first[j] = 0;

  // Vectors without a named class are summed as they stream by; the others
  // are left to the first slot that names a class of theirs.
  const unsigned char* marks = reinterpret_cast<const unsigned char*>(bits);
  constexpr unsigned kAll = (1u << VEC) - 1;
  auto marks_of = [&](int v) {
    const int b = row.first(v) + pad;
    return (unsigned)(marks[b / 8] >> (b % 8)) & kAll;
  };
  auto named_at = [&](int i) { return marks[(i + pad) / 8] >> ((i + pad) % 8) & 1; };
  FastSum fast;
  stream<THREADS, ONCE>(row, [&](const DfdVec<T, VEC>& x, int v) {
    if (marks_of(v)) return;
    float z[VEC];
    to_floats(x, z);
    fast.add(z, c);
  });
  Sum mine = fast.sum;
  for (int e = tid; e < row.edges(); e += THREADS)
    if (!named_at(row.edge(e))) add(mine, row.at(row.edge(e)), c);
  __syncthreads();  // s_first
  for (int j = tid; j < k; j += THREADS) {
    const int i = s_index[j] - row.head;
    if (i < 0 || i >= row.body * VEC || !s_first[j]) continue;
    const int v = i / VEC;
    const unsigned mark = marks_of(v);
    if (mark & ((1u << (i % VEC)) - 1)) continue;
    const DfdVec<T, VEC> x = row.load(v);
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (!(mark >> e & 1)) add(mine, DfdCvt<T>::to_f32(x.v[e]), c);
  }
  const Sum others = block_join<THREADS>(mine, c, sums);
  if (tid >= kWave) return;

  // the first wave: the row's few named classes
  const float inf = __builtin_inff();
  const float u_rest = rest ? rest[r] : -inf;
  Sum named = {kLowest, 0.f};
  float u_top = u_rest;
  bool none = u_rest == u_rest;  // no NaN among the teacher's logits
  for (int j = tid; j < k; j += kWave) {
    u_top = fmaxf(u_top, s_u[j]);
    none &= s_u[j] == s_u[j];
    if (s_index[j] >= 0 && s_first[j]) add(named, s_z[j], c);
  }
  named = wave_join(named, c);
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) u_top = fmaxf(u_top, __shfl_xor(u_top, off));
  const bool nothing = u_top == -inf && __all(none);
  float q_sum = tid == 0 ? expf(u_rest - u_top) : 0.f;
  for (int j = tid; j < k; j += kWave)
    if (s_index[j] >= 0) q_sum += expf(s_u[j] - u_top);
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) q_sum += __shfl_xor(q_sum, off);
  const Sum all = join(others, named, c);
  const float log_q = logf(q_sum), log_s = logf(all.s);
  float sum = 0.f;
  auto term = [&](float lq, float lp) {
    const float q = expf(lq);
    if (q > 0.f) sum += q * (lq - lp) + (twice ? 0.f : expf(lp) - q);
    else if (!twice) sum += expf(lp);
  };
  for (int j = tid; j < k; j += kWave)
    if (s_index[j] >= 0) term(s_u[j] - u_top - log_q, (s_z[j] - all.m) * inv_t - log_s);
  float p_rest = 0.f;
  const float q_rest = expf(u_rest - u_top - log_q);
  if (others.s != 0.f) {
    const float lp = (others.m - all.m) * inv_t + logf(others.s) - log_s;
    p_rest = expf(lp);
    if (tid == 0) term(u_rest - u_top - log_q, lp);
  } else if (tid == 0 && q_rest > 0.f) {
    sum = inf;  // the teacher sees classes that the student rules out
  }
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
  if (tid == 0) {
    loss[r] = bad ? __builtin_nanf("") : nothing ? 0.f : sum;
    RowStats s;
    s.m_rest = others.s == 0.f ? 0.f : others.m;
    s.coef = others.s == 0.f ? 0.f : (p_rest - q_rest) / others.s;
    s.m = all.m;
    s.inv_s = 1.f / all.s;
    s.u_top = u_top;
    s.inv_q = 1.f / q_sum;
    s.state = bad ? kBadIndex : nothing ? kNothing : twice ? kTwice : kTeaches;
    s.unused = 0.f;
    stats[r] = s;
  }
}

template <typename T, int VEC, int THREADS, bool ONCE>
__global__ __launch_bounds__(THREADS) void distill_bwd_kernel(
    const T* __restrict__ logits, long long row_stride, int classes, int k, float inv_t,
    const void* __restrict__ values, LogitType vtype, const long long* __restrict__ indices,
    const RowStats* __restrict__ stats, const float* __restrict__ upstream,
    long long upstream_stride, T* __restrict__ grad) {
  const int tid = threadIdx.x;
  // from the last row on: what the forward pass read last may still be cached
  const long long r = gridDim.x - 1 - blockIdx.x;
  const Row<T, VEC> row(logits + r * row_stride, classes);
  const float c = inv_t * kLog2e;
  T* out = grad + r * classes;
  const RowStats s = stats[r];
  const float g = upstream[r * upstream_stride] * inv_t;
  if (s.state >= kNothing) {
    const T fill = DfdCvt<T>::from_f32(s.state == kNothing ? 0.f : __builtin_nanf(""));
    DfdVec<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = fill;
    for (int v = tid; v < row.body; v += THREADS) dfd_vstore<T, VEC>(out + row.first(v), o);
    for (int e = tid; e < row.edges(); e += THREADS) out[row.edge(e)] = fill;
    return;
  }
  const float coef = s.coef * g;
  auto of_rest = [&](float z) { return DfdCvt<T>::from_f32(exp2_fast((z - s.m_rest) * c) * coef); };
  stream<THREADS, ONCE>(row, [&](const DfdVec<T, VEC>& x, int v) {
    float z[VEC];
    to_floats(x, z);
    DfdVec<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = of_rest(z[i]);
    dfd_vstore_once<T, VEC>(out + row.first(v), o);
  });
  for (int e = tid; e < row.edges(); e += THREADS)
    out[row.edge(e)] = of_rest(row.at(row.edge(e)));
  // the named classes' gradients take the place of what was just written
  __syncthreads();
  for (int j = tid; j < k; j += THREADS) {
    const long long at = indices[r * k + j];
    // (the forward pass has looked at them, but they may have changed since)
    if (at < 0 || at >= classes) continue;
    float q = 0.f;
    if (s.state == kTwice) {
      for (int i = 0; i < k; ++i)
        if (indices[r * k + i] == at)
          q += expf(load_as(values, vtype, r * k + i) * inv_t - s.u_top) * s.inv_q;
    } else {
      q = expf(load_as(values, vtype, r * k + j) * inv_t - s.u_top) * s.inv_q;
    }
    // (the exponential that keeps results below 2^-126)
    const float p = expf((row.at((int)at) - s.m) * inv_t) * s.inv_s;
    out[at] = DfdCvt<T>::from_f32((p - q) * g);
  }
}

#define LOGIT_TYPE(VAL, ...)                                                 \
  switch (VAL) {                                                             \
    case LogitType::kF32: { using T = float; __VA_ARGS__; break; }           \
    case LogitType::kBf16: { using T = __hip_bfloat16; __VA_ARGS__; break; } \
    case LogitType::kF16: { using T = __half; __VA_ARGS__; break; }          \
  }
#define ROW_THREADS(VAL, LARGEST, ...)                                  \
  switch (VAL) {                                                        \
    case 64: { constexpr int N = 64; __VA_ARGS__; break; }              \
    case 256: { constexpr int N = 256; __VA_ARGS__; break; }            \
    default: { constexpr int N = LARGEST; __VA_ARGS__; break; }         \
  }

}  // namespace

template <typename T, int THREADS>
static void topk_launch(const TopkArgs& a, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const T* z = static_cast<const T*>(a.logits);
  T* values = static_cast<T*>(a.values);
  const float inv_t = 1.f / a.temperature;
  const dim3 grid((unsigned)a.rows);
  // every thread has to have elements for the bound to be one
  if (a.classes >= V * (THREADS + 1))
    topk_kernel<T, V, THREADS><<<grid, THREADS, 0, stream>>>(
        z, a.row_stride, a.classes, a.k, inv_t, values, a.indices, a.rest);
  else
    topk_kernel<T, 1, THREADS><<<grid, THREADS, 0, stream>>>(
        z, a.row_stride, a.classes, a.k, inv_t, values, a.indices, a.rest);
}

static hipError_t topk_rows(const TopkArgs& a, hipStream_t stream) {
  // A wave alone has no barriers to wait at, and many rows hide its own time;
  // more threads shorten a row's. us by 64, 256 and 512 threads: bf16, k = 16,
  // 4096 x 16000: 36, 44, 59; 4096 x 32000: 63, 65, 76; fp16, k = 12, 4929 x
  // 3925: 20, 36, 60; k = 64, 4096 x 65536: -, 128, 138; fp32, k = 20, 100 x
  // 10000: 15, 10, 10; bf16, 1 x 131072: -, 23, 19. A bound needs k / waves of a wave's
  // 64 lanes, and fewer than half of them to be near: fp32, k = 250, 2000 x
  // 10000: -, 638, 90.
  const bool one_wave = a.k <= 32 && (a.classes <= 2048 || (a.rows >= 1024 && a.classes <= 32768));
  const bool many = a.k > 160 || (a.rows <= 256 && a.classes > 16384);
  const int threads = one_wave ? 64 : many ? 512 : 256;
  LOGIT_TYPE(a.type, {
    switch (threads) {
      case 64: topk_launch<T, 64>(a, stream); break;
      case 256: topk_launch<T, 256>(a, stream); break;
      default: topk_launch<T, 512>(a, stream); break;
    }
  });
  return hipGetLastError();
}

// Logits that the 256 MB of cache hold are still there for the backward pass;
// of larger ones the loads pass by it. Forward and backward us, so and
// otherwise: 8192 x 32000 bf16 (524 MB) 92 + 180 and 123 + 176, 513 x 49999
// fp32 (103 MB) 27 + 44 and 24 + 34.
static bool past_caches(const DistillArgs& a) {
  return a.rows * a.classes * (a.type == LogitType::kF32 ? 4 : 2) > 256ll << 20;
}

static hipError_t fwd_rows(const DistillArgs& a, hipStream_t stream) {
  // bf16: 1536 x 2048: 10.5 us by 64 threads, 11.4 by 256; 8192 x 32000 (all
  // through the cache): 147 us by 256, 170 by 64; 32 x 131072: 24 us by 256, 18
  // by 512, 17 by 1024.
  const int threads = a.classes <= 4096 ? 64 : a.rows <= 512 ? 512 : 256;
  const float inv_t = 1.f / a.temperature;
  const int bytes = (a.classes + 16 + 31) / 32 * 4;
  const bool once = past_caches(a);
  LOGIT_TYPE(a.type, ROW_THREADS(threads, 512, {
               constexpr int V = 16 / sizeof(T);
               auto launch = [&](auto kernel) {
                 kernel<<<dim3((unsigned)a.rows), N, bytes, stream>>>(
                     static_cast<const T*>(a.logits), a.row_stride, a.classes, a.k, inv_t,
                     a.values, a.vtype, a.indices, a.rest, a.loss,
                     reinterpret_cast<RowStats*>(a.stats));
               };
               if (once) launch(distill_fwd_kernel<T, V, N, true>);
               else launch(distill_fwd_kernel<T, V, N, false>);
             }));
  return hipGetLastError();
}

static hipError_t bwd_rows(const DistillArgs& a, hipStream_t stream) {
  // bf16: 1536 x 1000: 4.6 us by 64 threads, 4.5 by 256, 7.4 by 1024; 1024 x
  // 16384: 13 us by 256, 15 by 64; 8192 x 32000: 212 us by 256, 178 by 1024
  // (a copy's rate).
  const int threads = a.classes <= 1024 ? 64 : a.classes <= 16384 ? 256 : 1024;
  const float inv_t = 1.f / a.temperature;
  LOGIT_TYPE(a.type, ROW_THREADS(threads, 1024, {
               constexpr int V = 16 / sizeof(T);
               const T* z = static_cast<const T*>(a.logits);
               T* grad = static_cast<T*>(a.grad);
               // both rows' vectors lie alike, or elements go one by one
               const bool alike =
                   (reinterpret_cast<unsigned long long>(z) -
                    reinterpret_cast<unsigned long long>(grad)) % 16 == 0 &&
                   (a.row_stride - a.classes) * (long long)sizeof(T) % 16 == 0;
               auto launch = [&](auto kernel) {
                 kernel<<<dim3((unsigned)a.rows), N, 0, stream>>>(
                     z, a.row_stride, a.classes, a.k, inv_t, a.values, a.vtype, a.indices,
                     reinterpret_cast<const RowStats*>(a.stats), a.upstream,
                     a.upstream_stride, grad);
               };
               if (!alike) launch(distill_bwd_kernel<T, 1, N, false>);
               else if (past_caches(a)) launch(distill_bwd_kernel<T, V, N, true>);
               else launch(distill_bwd_kernel<T, V, N, false>);
             }));
  return hipGetLastError();
}

// HIP takes fewer than 2^32 threads a launch: more rows go in several.
constexpr long long kMostRows = 1ll << 21;

static const void* at(const void* p, LogitType type, long long i) {
  return static_cast<const char*>(p) + i * (type == LogitType::kF32 ? 4 : 2);
}
static void* at(void* p, LogitType type, long long i) {
  return static_cast<char*>(p) + i * (type == LogitType::kF32 ? 4 : 2);
}

// f of the args of each part of the rows.
template <typename Args, typename Skip, typename F>
static hipError_t in_parts(const Args& all, Skip skip, F f) {
  Args a = all;
  hipError_t e = hipSuccess;
  for (long long left = all.rows; left > 0 && e == hipSuccess; left -= a.rows) {
    a.rows = left < kMostRows ? left : kMostRows;
    e = f(a);
    skip(a, a.rows);
  }
  return e;
}

hipError_t topk_logits_launch(const TopkArgs& args, hipStream_t stream) {
  return in_parts(
      args,
      [](TopkArgs& a, long long n) {
        a.logits = at(a.logits, a.type, n * a.row_stride);
        a.values = at(a.values, a.type, n * a.k);
        a.indices += n * a.k;
        a.rest += n;
      },
      [&](const TopkArgs& a) { return topk_rows(a, stream); });
}

static void distill_skip(DistillArgs& a, long long n) {
  a.logits = at(a.logits, a.type, n * a.row_stride);
  a.values = at(a.values, a.vtype, n * a.k);
  a.indices += n * a.k;
  a.stats += n * kDistillStats;
  if (a.rest) a.rest += n;
  if (a.loss) a.loss += n;
  if (a.upstream) a.upstream += n * a.upstream_stride;
  if (a.grad) a.grad = at(a.grad, a.type, n * a.classes);
}

hipError_t distill_fwd(const DistillArgs& args, hipStream_t stream) {
  return in_parts(args, distill_skip, [&](const DistillArgs& a) { return fwd_rows(a, stream); });
}

hipError_t distill_bwd(const DistillArgs& args, hipStream_t stream) {
  return in_parts(args, distill_skip, [&](const DistillArgs& a) { return bwd_rows(a, stream); });
}
