// Operators over rows of logits of a whole vocabulary: log probabilities of given tokens with entropy and top alternatives, the
// distillation loss against a teacher's top logits, and the gradients of both.
//
// Times in the comments are medians over replays of a captured graph of a few calls on the same buffers, so that what fits the last-level
// cache (256 MB) may come from it; where two ways stand side by side, both were timed on one card when the choice between them was made.
#include <type_traits>

#include "row_math.h"

namespace tk {
namespace {

constexpr float NEG_INF = -__builtin_inff();

constexpr float LOG2E = 1.44269504088896340736f, LOG2E_REST = (float)(1.44269504088896340736 - (double)LOG2E), LN2 = 0.69314718055994530942f;
constexpr int MAX_GRID = 1 << 23;  // workgroups of a launch (2^32 threads are its limit)
constexpr int GROUP = 64;      // consecutive columns whose largest logit is kept while a row streams by
constexpr int MAX_CHUNKS = 256;  // pieces that a row is split into where there are few rows
constexpr int LEAST_CHUNK = 4096;

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// What a call needs of the temperature: exponentials are taken to the base two, exp((x - m) / t) = 2^((x - m) c2).
struct Scales {
  float inv_t, c2;
};

// ---- the pass over the logits -------------------------------------------------------------------------------
// Softmax statistics of the logits seen so far, as one pass takes them: m the largest, k = m c2 rounded to a whole number, s = sum 2^d and
// e = sum 2^d d with d = x c2 - k.  The product and the difference are one operation and one rounding, and a larger m rescales both sums by
// a power of two, exactly: s' = 2^(k - k') s, e' = 2^(k - k') (e + s (k - k')).  (x - m) c2 in two operations, which needs no whole number,
// took 4 to 7 % longer with alternatives, where the vector unit bounds the pass; x c2 - m c2 with m c2 rounded is off by 1e-6 between lanes
// whose m differ.  From |m c2| = 2^24 on, numbers of 32 bits are further apart than one, and m c2 - k may be anything up to that distance.
// So k is taken from a little above: no d is much above zero, and no sum overflows that a larger logit (behind logits masked with -1e10,
// say) brings back to nothing.  The sums of a row whose largest logit is so large are left to Workgroup::wide().  d is bounded by D_MIN in
// products only, where -inf times a probability of zero stands for zero; 2^D_MIN is zero in 32 bits.
constexpr float D_MIN = -300.f, K_MAX = 3.3e38f, WIDE = 2.f;
struct Softmax {
  float m, k, s, e;
  float offset;  // of a row's whole sums: k - m c2, what its logarithms are off by from those around m
  static __device__ __forceinline__ float reference(float m, float c2) {
    const float x = m * c2;
    return fminf(fmaxf(rintf(fmaf(fabsf(x), 0x1p-23f, x)), -K_MAX), K_MAX);
  }
  static __device__ __forceinline__ Softmax nothing() { return {NEG_INF, -K_MAX, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ void raise(float to, float c2) {
    const float old = k;
    m = to;
    k = reference(to, c2);
    const float d = old - k, f = __builtin_amdgcn_exp2f(d);
    e = f * fmaf(s, fmaxf(d, D_MIN), e);
    s *= f;
  }
};

// Order of a logit as an unsigned number of BITS; the two zeros are one value, and no logit's number is zero.
template <int DT>
struct Key {
  static constexpr int SHIFT = DT == TK_F32 ? 0 : DT == TK_BF16 ? 16 : 13, BITS = 32 - SHIFT;
  static __device__ __forceinline__ uint32_t of(float f) { return ordered_key(f + 0.0f) >> SHIFT; }
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint32_t low = (1u << SHIFT) - 1u;
    return key_to_float(k << SHIFT | (k >> (BITS - 1) ? 0u : low));
  }
};

__device__ __forceinline__ uint64_t entry_of(uint32_t key, int column) { return (uint64_t)key << 32 | (uint32_t)~column; }

struct RowResult {
  float m, log_s, entropy;  // log_s = ln sum exp((x - m) / t)
  bool bad, empty;
  __device__ __forceinline__ RowResult(const Softmax& r) : m(r.m) {
    bad = !(r.s >= 0.f) || r.m == __builtin_inff();
    empty = !bad && r.s == 0.f;
    const float l = logf(r.s);
    log_s = bad ? __builtin_nanf("") : empty ? NEG_INF : fmaf(LN2, r.offset, l);
    entropy = bad ? __builtin_nanf("") : empty ? 0.f : l - LN2 * (r.e / r.s);
  }
  __device__ __forceinline__ float logprob(float x, float inv_t) const { return bad ? __builtin_nanf("") : empty ? NEG_INF : (x - m) * inv_t - log_s; }
};

// What a row's results take from single elements, requested before the row streams by.
template <int DT>
struct Token {
  float x = 0.f;
  bool live;
  __device__ __forceinline__ Token(const tk_vocab_desc& d, int t, const void* row) {
    const int64_t at = index_at(d.tokens, d.tokens_i64, t);
    live = at >= 0 && at < d.vocab;
    if (live) x = RowType<DT>::load(row, at);
  }
};

// The teacher's entry j of row t: its index, or -1 where it carries no weight, and its logit.
__device__ __forceinline__ int teacher_entry(const tk_vocab_desc& d, int t, int j, float* q) {
  *q = load_any(d.teacher_logits, d.teacher_dtype, (int64_t)t * d.teacher_stride_m + j);
  const int64_t i = index_at(d.teacher_indx, d.teacher_indx_i64, (int64_t)t * d.teacher_indx_stride_m + j);
  return i < 0 || i >= d.vocab || *q == NEG_INF ? -1 : (int)i;
}

enum { LOGPROBS = 0, LOGPROBS_TOP = 1, DISTILL = 2 };

template <int DT>
__device__ __forceinline__ const void* logits_row(const tk_vocab_desc& d, int t) {
  return static_cast<const char*>(d.logits) + (int64_t)t * d.logits_stride_m * RowType<DT>::BYTES;
}

// A row from the sixteen-byte boundary at or in front of it: place `begin` is its column 0, what lies in front is not touched.  Loads that
// do not begin at such boundaries take a quarter longer (4096 x 130001 bf16 222 us, x 130000 180).
struct Placed {
  const void* base;
  int begin;
};
template <int DT>
__device__ __forceinline__ Placed placed(const void* row) {
  const int begin = (int)(reinterpret_cast<uintptr_t>(row) & 15) / RowType<DT>::BYTES;
  return {static_cast<const char*>(row) - begin * RowType<DT>::BYTES, begin};
}

// ---- a row by a workgroup of THREADS lanes: four waves, or one for short rows, of which the chip then holds four times as many ----------
template <int THREADS>
struct Workgroup {
  static constexpr int WAVES = THREADS / 64;
  static constexpr int MANY = THREADS == 64 ? 256 : 512;  // candidates that are ranked by counting
  static constexpr int ENTRIES = TK_VOCAB_MAX_TEACHER / 256;  // teacher entries a lane

  // A row's statistics in every lane, from those of the lanes; `buf`: 3 * WAVES floats of LDS.
  static __device__ __forceinline__ Softmax block_softmax(Softmax r, float c2, float* buf) {
    const float m = block_max<THREADS>(r.m, buf);
    r.raise(m, c2);
    r.offset = fmaf(-m, c2, r.k);
    r.s = wave_sum_f32(r.s);
    r.e = wave_sum_f32(r.e);
    if constexpr (WAVES == 1) return r;
    if ((threadIdx.x & 63) == 0) {
      buf[WAVES + (threadIdx.x >> 6)] = r.s;
      buf[2 * WAVES + (threadIdx.x >> 6)] = r.e;
    }
    __syncthreads();
    r.s = buf[WAVES];
    r.e = buf[2 * WAVES];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      r.s += buf[WAVES + w];
      r.e += buf[2 * WAVES + w];
    }
    return r;
  }

  // The sums of a row whose largest logit is finite but lies WIDE or more from its whole number (nothing but masked logits, say):
  // differences from m first, element by element.
  template <int DT>
  static __device__ __forceinline__ Softmax wide(const void* row, int V, Softmax r, float c2, float* buf) {
    if (!(r.m > NEG_INF && r.m < __builtin_inff() && !(fabsf(r.offset) < WIDE))) return r;
    float s = 0.f, e = 0.f;
    for (int v = threadIdx.x; v < V; v += THREADS) {
      const float d = (RowType<DT>::load(row, v) - r.m) * c2, p = __builtin_amdgcn_exp2f(d);
      s += p;
      e = fmaf(p, fmaxf(d, D_MIN), e);
    }
    __syncthreads();
    r.s = block_sum<THREADS>(s, buf);
    __syncthreads();
    r.e = block_sum<THREADS>(e, buf);
    r.offset = 0.f;
    return r;
  }

  // Places [c0, c1) of a row from `begin` on; `keys` takes the order numbers of the groups' largest logits (group = place / GROUP; c0 is a
  // multiple of GROUP).  U vectors of 16 bytes a lane are under way while the U before them are summed.
  template <int DT, bool ENTROPY, bool TOP, int U, bool ONCE>
  static __device__ __forceinline__ Softmax stream(const void* row, int begin, int c0, int c1, float c2, uint32_t* keys) {
    typedef RowType<DT> R;
    constexpr int VE = R::VE, STEP = THREADS * VE * U;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * 64 * VE;
    Softmax r = Softmax::nothing();
    const auto fetch = [&](row_u32x4 (&raw)[U], int base) {
      const int at = base + (int)threadIdx.x * VE;
      if (base >= begin && base + STEP <= c1) {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = ONCE ? R::load_vec_once(row, at + u * THREADS * VE) : R::load_vec(row, at + u * THREADS * VE);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = R::load_vec_in(row, at + u * THREADS * VE, begin, c1, R::NEG_INF_BITS);
      }
    };
    row_u32x4 next[U];
    fetch(next, c0);
    for (int base = c0; base < c1; base += STEP) {
      const int at = base + (int)threadIdx.x * VE;
      row_u32x4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = next[u];
      if (base + STEP < c1) fetch(next, base + STEP);
      __builtin_amdgcn_sched_barrier(0);  // (the requests first)
      const auto sum = [&](auto last) {  // (a row's last step: the waves skip as a whole what lies behind it)
        const auto there = [&](int u) { return !decltype(last)::value || base + u * THREADS * VE + wave < c1; };
        float mx[U], top = NEG_INF;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          mx[u] = NEG_INF;
          if (!there(u)) continue;
          mx[u] = R::element(raw[u], 0);
#pragma unroll
          for (int e = 1; e < VE; ++e) mx[u] = fmaxf(mx[u], R::element(raw[u], e));
          top = fmaxf(top, mx[u]);
        }
        if (top > r.m) r.raise(top, c2);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!there(u)) continue;
          float s = 0.f, en = 0.f;
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float d = fmaf(R::element(raw[u], e), c2, -r.k), p = __builtin_amdgcn_exp2f(d);
            s += p;
            if (ENTROPY) en = fmaf(p, fmaxf(d, D_MIN), en);
          }
          r.s += s;
          r.e += en;
          if (TOP) {
            uint32_t x = Key<DT>::of(mx[u]);
#define TK_STEP(ctrl)                                                                        \
  {                                                                                          \
    const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, ctrl, 0xF, 0xF, true);     \
    x = o > x ? o : x;                                                                       \
  }
            TK_STEP(TK_DPP_QUAD_XOR1)
            TK_STEP(TK_DPP_QUAD_XOR2)
            TK_STEP(TK_DPP_ROW_HALF_MIRROR)
            if (VE == 4) TK_STEP(TK_DPP_ROW_MIRROR)
#undef TK_STEP
            const int c = at + u * THREADS * VE;
            if ((threadIdx.x & (GROUP / VE - 1)) == 0 && c < c1) keys[c / GROUP] = x;
          }
        }
      };
      if (base + STEP <= c1)
        sum(std::false_type());
      else
        sum(std::true_type());
    }
    return r;
  }

  // ---- the k largest ------------------------------------------------------------------------------------------
  // A row's k largest logits lie in the k groups whose largest logits are the largest (equal ones: the lower groups): were one of them in
  // another group, each of these k groups would hold an element in front of it.  So the selection looks at a number per group, and then at
  // the k groups' elements again: the rest of the row is read once, whatever stands in it.  A bound from below narrows both: k threads'
  // largest group numbers are at least the k-th largest of the threads' largest ones, so that only groups, and then only elements, from
  // there on can be among the k; as a rule they are few more than k, which are ranked by counting.  Where they are many (equal logits,
  // logits masked to one value, neighbours sorted together), each of the two selections finds the k-th largest number bit by bit with a
  // count over the workgroup, and takes the equal ones by a prefix sum in the order of the columns.
  struct SelectLds {
    int count[2][WAVES];
    int scan[WAVES];
    int n_groups, n_found;
    alignas(16) uint32_t most[THREADS];
    int group[MANY];
    uint64_t found[MANY];  // key << 32 | ~column: a larger one comes first
  };
  // Calls take(slot, i) for the k first of n items in the order (larger key, then lower i), slots by i; at least k keys are not 0.  A
  // thread looks at consecutive items.  This is the way for the rows that the ranking does not serve: it reads the keys again for each bit.
  template <int BITS, class KeyOf, class F>
  static __device__ __forceinline__ void select(int n, int k, SelectLds& lds, KeyOf&& key_of, F&& take) {
    const int per = (n + THREADS - 1) / THREADS, i0 = (int)threadIdx.x * per, i1 = i0 + per < n ? i0 + per : n;
    uint32_t from = 0;
    bool exact = false;  // k keys are >= from
    for (int b = BITS - 1; b >= 0 && !exact; --b) {
      const uint32_t at = from | 1u << b;
      int mine = 0;
      for (int i = i0; i < i1; ++i) mine += key_of(i) >= at;
      mine = wave_scan_i32(mine);
      if ((threadIdx.x & 63) == 63) lds.count[b & 1][threadIdx.x >> 6] = mine;
      __syncthreads();
      int c = lds.count[b & 1][0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) c += lds.count[b & 1][w];
      if (c >= k) from = at;
      exact = c == k;
    }
    // all larger ones, and the first of the equal ones
    int larger = 0, equal = 0;
    for (int i = i0; i < i1; ++i) {
      const uint32_t key = key_of(i);
      larger += key > from;
      equal += key == from;
    }
    const int mine = larger | equal << 16, upto = wave_scan_i32(mine);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) lds.scan[threadIdx.x >> 6] = upto;
    __syncthreads();
    int before = upto - mine, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < (int)(threadIdx.x >> 6)) before += lds.scan[w];
      all += lds.scan[w];
    }
    const int need = k - (all & 0xFFFF);  // equal ones that are taken
    int l = before & 0xFFFF, q = before >> 16;
    for (int i = i0; i < i1; ++i) {
      const uint32_t key = key_of(i);
      if (key > from || (key == from && q < need)) take(l + (q < need ? q : need), i);
      l += key > from;
      q += key == from;
    }
  }

  // The k-th largest of the threads' numbers, each wave by itself; 1 (less than any logit's) where fewer than k threads have one.
  template <int BITS>
  static __device__ __forceinline__ uint32_t kth_of_threads(uint32_t mine, int k, SelectLds& lds) {
    lds.most[threadIdx.x] = mine;
    __syncthreads();
    typedef uint32_t own __attribute__((ext_vector_type(WAVES == 1 ? 2 : WAVES)));  // (a lane's share of them; a wave alone has one)
    own share;
    if constexpr (WAVES == 1)
      share = own{mine, 0u};
    else
      share = reinterpret_cast<const own*>(lds.most)[threadIdx.x & 63];
    uint32_t from = 0;
    for (int b = BITS - 1; b >= 0; --b) {
      const uint32_t at = from | 1u << b;
      int c = 0;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) c += __builtin_popcountll(__ballot(share[i] >= at));
      if (c < k) continue;
      from = at;
      if (c == k) break;
    }
    return from ? from : 1u;
  }

  // Leaves at least the k largest of places [begin, end) of a row in lds.found, in any order, and returns how many; from the groups'
  // numbers.
  template <int DT>
  static __device__ __forceinline__ int top_of_row(const void* row, int begin, int end, int k, const uint32_t* group_keys, SelectLds& lds) {
    typedef RowType<DT> R;
    constexpr int VE = R::VE, BITS = Key<DT>::BITS, OWN = 8;
    const int groups = (end + GROUP - 1) / GROUP;
    // (four waves have passed a barrier since the pass wrote the groups' numbers; one has not, and its lanes read each other's)
    if constexpr (WAVES == 1) __syncthreads();
    if (threadIdx.x == 0) lds.n_groups = lds.n_found = 0;
    uint32_t most = 0, own[OWN];  // (the first OWN of a thread's stay in registers)
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int g = i * THREADS + (int)threadIdx.x;
      own[i] = g < groups ? group_keys[g] : 0u;
      most = own[i] > most ? own[i] : most;
    }
    for (int g = OWN * THREADS + (int)threadIdx.x; g < groups; g += THREADS) most = group_keys[g] > most ? group_keys[g] : most;
    if (groups < k)  // a row so short that the threads' elements tell more
      for (int v = (int)threadIdx.x * VE; v < end; v += THREADS * VE) {
        const row_u32x4 raw = R::load_vec_in(row, v, begin, end, R::NEG_INF_BITS);
        uint32_t mx = 0;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const uint32_t one = Key<DT>::of(R::element(raw, e));
          mx = one > mx ? one : mx;
        }
        most = v == (int)threadIdx.x * VE || mx > most ? mx : most;
      }
    const uint32_t from = kth_of_threads<BITS>(most, k, lds);
    const auto add_group = [&](uint32_t key, int g) {
      if (key < from) return;
      const int slot = atomicAdd(&lds.n_groups, 1);
      if (slot < MANY) lds.group[slot] = g;
    };
#pragma unroll
    for (int i = 0; i < OWN; ++i) add_group(own[i], i * THREADS + (int)threadIdx.x);
    for (int g = OWN * THREADS + (int)threadIdx.x; g < groups; g += THREADS) add_group(group_keys[g], g);
    __syncthreads();
    const int n_groups = lds.n_groups;
    if (n_groups <= MANY) {
      constexpr int PER = GROUP / VE;
      for (int v = threadIdx.x; v < n_groups * PER; v += THREADS) {
        const int at = lds.group[v / PER] * GROUP + v % PER * VE;
        const row_u32x4 raw = R::load_vec_in(row, at, begin, end, R::NEG_INF_BITS);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const uint32_t one = Key<DT>::of(R::element(raw, e));
          if (one >= from && at + e >= begin && at + e < end) {
            const int i = atomicAdd(&lds.n_found, 1);
            if (i < MANY) lds.found[i] = entry_of(one, at + e - begin);
          }
        }
      }
      __syncthreads();
      const int n = lds.n_found;
      if (n <= MANY) return n;
    }
    const int n = k < groups ? k : groups;
    select<BITS>(groups, n, lds, [&](int i) { return group_keys[i]; }, [&](int to, int i) { lds.group[to] = i; });
    __syncthreads();
    const auto place = [&](int i) { return lds.group[i / GROUP] * GROUP + i % GROUP; };
    const auto element = [&](int i) { return place(i) >= begin && place(i) < end ? Key<DT>::of(R::load(row, place(i))) : 0u; };
    select<BITS>(n * GROUP, k, lds, element, [&](int to, int i) { lds.found[to] = entry_of(element(i), place(i) - begin); });
    __syncthreads();
    return k;
  }

  // ---- what comes out of a row's statistics ---------------------------------------------------------------------
  template <int DT, bool TOP>
  static __device__ __forceinline__ void finish_logprobs(const tk_vocab_desc& d, Scales sc, int t, Placed row, const Token<DT>& token, const Softmax& r,
                                                  const uint32_t* group_keys, SelectLds* lds) {
    const RowResult o(r);
    if (threadIdx.x == 0) {
      d.logprobs[t] = token.live ? o.logprob(token.x, sc.inv_t) : 0.f;
      d.entropy[t] = o.entropy;
      if (d.stats) {
        d.stats[t] = o.m;
        d.stats[(int64_t)d.n_rows + t] = o.log_s;
      }
    }
    if constexpr (TOP) {
      const int64_t out = (int64_t)t * d.k;
      if (o.bad) {
        if ((int)threadIdx.x < d.k) {
          d.top_indx[out + threadIdx.x] = -1;
          d.top_logprobs[out + threadIdx.x] = __builtin_nanf("");
        }
        return;
      }
      const int n = top_of_row<DT>(row.base, row.begin, row.begin + d.vocab, d.k, group_keys, *lds);
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint64_t mine = lds->found[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += lds->found[j] > mine;
        if (rank < d.k) {
          d.top_indx[out + rank] = (int)~(uint32_t)mine;
          d.top_logprobs[out + rank] = o.logprob(Key<DT>::value((uint32_t)(mine >> 32)), sc.inv_t);
        }
      }
    }
  }

  // The teacher's entries of a thread: their logits, -inf where they carry no weight, and the student's at their indices.
  template <int DT>
  struct Teacher {
    float q[ENTRIES], x[ENTRIES];
    __device__ __forceinline__ Teacher(const tk_vocab_desc& d, int t, const void* row) {
#pragma unroll
      for (int i = 0; i < ENTRIES; ++i) {
        const int j = i * THREADS + (int)threadIdx.x;
        q[i] = NEG_INF;
        x[i] = 0.f;
        if (j < d.n_teacher) {
          const int at = teacher_entry(d, t, j, &q[i]);
          if (at >= 0)
            x[i] = RowType<DT>::load(row, at);
          else
            q[i] = NEG_INF;
        }
      }
    }
  };

  template <int DT>
  static __device__ __forceinline__ void finish_distill(const tk_vocab_desc& d, Scales sc, int t, const Teacher<DT>& teacher, const Softmax& r, float (*buf)[WAVES]) {
    const RowResult o(r);
    float qm = NEG_INF, qs = 0.f, loss = 0.f;
    int bad = 0;
#pragma unroll
    for (int i = 0; i < ENTRIES; ++i) {
      qm = fmaxf(qm, teacher.q[i]);
      bad |= teacher.q[i] != teacher.q[i];
    }
    qm = block_max<THREADS>(qm, buf[0]);
    bad = __syncthreads_or(bad) || qm == __builtin_inff();
#pragma unroll
    for (int i = 0; i < ENTRIES; ++i)
      if (teacher.q[i] != NEG_INF) qs += expf((teacher.q[i] - qm) * sc.inv_t);
    qs = block_sum<THREADS>(qs, buf[1]);
    const float log_qs = bad ? __builtin_nanf("") : logf(qs);
#pragma unroll
    for (int i = 0; i < ENTRIES; ++i)
      if (teacher.q[i] != NEG_INF) {
        const float la = (teacher.q[i] - qm) * sc.inv_t - log_qs, a = expf(la);
        if (a != 0.f) loss = fmaf(a, la - o.logprob(teacher.x[i], sc.inv_t), loss);
      }
    loss = block_sum<THREADS>(loss, buf[2]);
    if (threadIdx.x == 0) {
      d.loss[t] = loss;
      if (d.stats) {
        d.stats[t] = o.m;
        d.stats[(int64_t)d.n_rows + t] = o.log_s;
      }
      if (d.teacher_stats) {
        d.teacher_stats[t] = bad ? __builtin_nanf("") : qm;
        d.teacher_stats[(int64_t)d.n_rows + t] = log_qs;
      }
    }
  }

  struct RowLds {
    float softmax[3 * WAVES];
    float teacher[3][WAVES];
    SelectLds select;
  };

  template <int DT, int OP>
  using Single = std::conditional_t<OP == DISTILL, Teacher<DT>, Token<DT>>;
  template <int DT, int OP>
  static __device__ __forceinline__ void finish(const tk_vocab_desc& d, Scales sc, int t, Placed row, const Single<DT, OP>& single, const Softmax& r,
                                         const uint32_t* keys, RowLds& lds) {
    if constexpr (OP == DISTILL)
      finish_distill<DT>(d, sc, t, single, r, lds.teacher);
    else
      finish_logprobs<DT, OP == LOGPROBS_TOP>(d, sc, t, row, single, r, keys, &lds.select);
  }
};

// A row a workgroup, from the first logit to the results; the groups' numbers stay in LDS (dynamic, with OP == LOGPROBS_TOP).  Bound by the
// logits' one read, and with alternatives by the vector unit as well: 4096 x 131072 bf16 174 us (6.2 TB/s), with 64 alternatives 195 (5.5);
// 2048 x 32000 fp32 43.7 (6.0).
template <int DT, int OP, int THREADS, int U>
__global__ __launch_bounds__(THREADS) void vocab_rows_kernel(tk_vocab_desc d, Scales sc, int t0, int keep_from) {
  typedef Workgroup<THREADS> W;
  extern __shared__ uint32_t keys[];
  __shared__ typename W::RowLds lds;
  const int t = t0 + (int)blockIdx.x;
  const void* row = logits_row<DT>(d, t);
  const typename W::template Single<DT, OP> single(d, t, row);
  const Placed p = THREADS == 64 ? Placed{row, 0} : placed<DT>(row);  // (a short row is over before it pays)
  const int end = p.begin + d.vocab;
  const Softmax mine = THREADS == 64 || t >= keep_from ? W::template stream<DT, OP != DISTILL, OP == LOGPROBS_TOP, U, false>(p.base, p.begin, 0, end, sc.c2, keys)
                                                       : W::template stream<DT, OP != DISTILL, OP == LOGPROBS_TOP, U, THREADS != 64>(p.base, p.begin, 0, end, sc.c2, keys);
  const Softmax r = W::template wide<DT>(row, d.vocab, W::block_softmax(mine, sc.c2, lds.softmax), sc.c2, lds.softmax);
  W::template finish<DT, OP>(d, sc, t, p, single, r, keys, lds);
}

// Few rows: pieces of a row (61 x 50001 fp16 with 8 alternatives 12.2 us, both launches: latencies one after the other, not bytes), whose
// statistics and groups' numbers go through the workspace to vocab_join_kernel.
typedef Workgroup<256> Wide;
template <int DT, int OP>
__global__ __launch_bounds__(256) void vocab_chunk_kernel(tk_vocab_desc d, Scales sc, int chunk, int n_chunks, float* parts, uint32_t* keys, int groups) {
  __shared__ float buf[3 * Wide::WAVES];
  const int t = blockIdx.x / n_chunks, c = blockIdx.x % n_chunks, c0 = c * chunk;
  const Placed p = placed<DT>(logits_row<DT>(d, t));
  const int end = p.begin + d.vocab, c1 = end - c0 < chunk ? end : c0 + chunk;
  const Softmax r =
      Wide::block_softmax(Wide::stream<DT, OP != DISTILL, OP == LOGPROBS_TOP, 2, false>(p.base, p.begin, c0, c1, sc.c2, keys + (int64_t)t * groups), sc.c2, buf);
  if (threadIdx.x < 3) parts[((int64_t)t * n_chunks + c) * 3 + threadIdx.x] = threadIdx.x == 0 ? r.m : threadIdx.x == 1 ? r.s : r.e;
}

template <int DT, int OP>
__global__ __launch_bounds__(256) void vocab_join_kernel(tk_vocab_desc d, Scales sc, int n_chunks, const float* parts, const uint32_t* keys, int groups) {
  __shared__ Wide::RowLds lds;
  const int t = blockIdx.x;
  const void* row = logits_row<DT>(d, t);
  const Wide::Single<DT, OP> single(d, t, row);
  Softmax r = Softmax::nothing();
  if ((int)threadIdx.x < n_chunks) {
    const float* p = parts + ((int64_t)t * n_chunks + threadIdx.x) * 3;
    r = {p[0], Softmax::reference(p[0], sc.c2), p[1], p[2], 0.f};
  }
  r = Wide::wide<DT>(row, d.vocab, Wide::block_softmax(r, sc.c2, lds.softmax), sc.c2, lds.softmax);
  Wide::finish<DT, OP>(d, sc, t, placed<DT>(row), single, r, keys + (int64_t)t * groups, lds);
}

// Gradients from this size on are read and written with the read-once hint: they would only push the logits, which come from the last-level
// cache in part, out of it (forward and backward, us without and with: 2048 x 32000 fp32, 262 MB, 159, 129; 4096 x 131072 bf16, 1074 MB,
// 604, 590; 1000 x 50001 fp16, 100 MB, 79, 74.5; 200 x 32000 bf16, 13 MB, 18, 18, where whoever reads the gradient next may find it
// cached).
constexpr int64_t ONCE_BYTES = 64 << 20;
// The forward pass reads its logits with the hint, too (nothing follows it: 4096 x 131072 bf16 189, 165, 2048 x 32000 fp32 48.6, 42.6), but
// where a backward pass is to follow, the last rows without: that many bytes are still cached when it begins with them (forward and
// backward, all rows hinted, none, the last 192 MB not: 2048 x 32000 fp32 143, 129, 127; 2048 x 64000 281, 270, 263; 4096 x 96000 bf16 422,
// 416, 400; 4096 x 131072 542, 586, 548; 8192 x 100000 978, 924, 960).
constexpr int64_t KEPT_BYTES = 192 << 20;

// Pieces that the rows of a call are split into: about four workgroups a CU; no more, since a second launch joins them (us, pieces for 500,
// 1000 and 2048 workgroups: 1000 x 131072 bf16 with 20 alternatives 61, 61, 76; 300 x 131072 22.9, 22.5, 23.4; 100 x 131072 13.4, 12.6,
// 11.8; 61 x 50001 fp16 with 8 13.1, 14.4, 16.3).  From some 400 rows on whole rows are as fast or faster, which this rule does not know
// (in pieces and whole: 400 x 50001 fp16 15.5, 13.8; 600 19.9, 17.4; 999 27.6, 22.1, with 20 alternatives 37.4, 28.5; 400 x 131072 bf16
// 25.6, 27.8; 600 33.4, 33.7; 999 50.2, 46.3; 999 x 32000 fp32 28.3, 24.1).
struct Split {
  int n, chunk, groups;
  int64_t parts_bytes, bytes;
};
// `shift`: columns that the rows' addresses may add in front.
Split split_of(int32_t n_rows, int64_t vocab, int32_t k, int shift) {
  Split s;
  vocab += shift;
  const int64_t want = cdiv(1000, n_rows > 0 ? n_rows : 1), most = cdiv(vocab, LEAST_CHUNK);
  int64_t n = want < most ? want : most;
  n = n < MAX_CHUNKS ? n : MAX_CHUNKS;
  const int64_t chunk = cdiv(cdiv(vocab, n), LEAST_CHUNK) * LEAST_CHUNK;
  s.chunk = (int)(chunk < vocab ? chunk : vocab);
  s.n = (int)cdiv(vocab, s.chunk);
  s.groups = k ? (int)cdiv(vocab, GROUP) : 0;
  s.parts_bytes = cdiv((int64_t)n_rows * s.n * 12, 16) * 16;
  s.bytes = s.n > 1 ? s.parts_bytes + (int64_t)n_rows * s.groups * 4 : 0;
  return s;
}

Scales scales_of(const tk_vocab_desc* d) { return {(float)(1.0 / d->temperature), (float)(1.4426950408889634 / d->temperature)}; }

// Rows of up to SHORT_ROW columns have a wave each, where there are enough of them (us, a workgroup and a wave: 16000 x 1000 bf16 22.9,
// 12.1, its gradient 35, 19; x 4000 23.5, 28, its gradient 52, 56), longer ones with alternatives up to SHORT_TOP, whose ranking is the
// same work for four waves and one (with 20: 16000 x 2000 71, 34; x 4000 74, 44; x 8000 84, 67; x 16000 121, 118).  No more of those than
// half a wave ranks, nor more teacher entries than four a lane.
constexpr int SHORT_ROW = 2048, SHORT_TOP = 8192;

template <int DT, int OP>
int32_t forward(const tk_vocab_desc* d, hipStream_t stream, const char* who) {
  const bool aligned = ((reinterpret_cast<uintptr_t>(d->logits) | (uintptr_t)(d->logits_stride_m * RowType<DT>::BYTES)) & 15) == 0;
  const Split s = split_of(d->n_rows, d->vocab, OP == LOGPROBS_TOP ? d->k : 0, aligned ? 0 : RowType<DT>::VE - 1);
  const Scales sc = scales_of(d);
  if (s.n == 1) {
    // Four vectors a lane under way, or two: two waste less of a row's last step and start sooner, four carry long rows when the chip is
    // full of them; us with two, four (statistics alone; * with 64 alternatives): 1000 x 131072 bf16 49.3, 46.0 (* 60.6, 58.8), 1500 66.5,
    // 67.4 (* 78.9, 79.9), 2048 91.3, 94.8 (* 103, 106), 3000 134, 131 (* 151, 147), 4096 174, 174 (* 196, 195); x 50001 fp16 1000 23.6,
    // 22.7 (* 34.0, 34.5), 2048 40.0, 42.5 (* 53.5, 59.3), 4096 75.6, 73.3 (* 92.9, 94.7); x 32000 fp32 1000 23.7, 24.1 (* 31.9, 32.7),
    // 2048 46.4, 43.7 (* 57.6, 57.6), 4096 83.5, 82.5 (* 104, 100); 16000 x 4000 bf16 with 20 alternatives 74, 90.
    constexpr int STEP = 4 * 256 * RowType<DT>::VE;
    const bool wave = d->n_rows >= 1000 && (OP == LOGPROBS_TOP ? d->k <= 32 && d->vocab <= SHORT_TOP : d->vocab <= SHORT_ROW)
                      && (OP != DISTILL || d->n_teacher <= 64 * Workgroup<64>::ENTRIES);
    auto f = wave ? vocab_rows_kernel<DT, OP, 64, 2> : d->n_rows >= 2048 && d->vocab >= 6 * STEP ? vocab_rows_kernel<DT, OP, 256, 4> : vocab_rows_kernel<DT, OP, 256, 2>;
    const int64_t row_bytes = (int64_t)d->vocab * RowType<DT>::BYTES, kept = d->stats ? KEPT_BYTES / row_bytes : 0;
    const int keep_from = d->n_rows * row_bytes < ONCE_BYTES ? 0 : (int)(d->n_rows > kept ? d->n_rows - kept : 0);
    for (int64_t t = 0; t < d->n_rows; t += MAX_GRID) {
      const int rows = (int)(d->n_rows - t < MAX_GRID ? d->n_rows - t : MAX_GRID);
      hipLaunchKernelGGL(f, dim3(rows), dim3(wave ? 64 : 256), OP == LOGPROBS_TOP ? s.groups * 4 : 0, stream, *d, sc, (int)t, keep_from);
    }
    return check_launch(who);
  }
  if (!d->workspace) return fail(TK_ERR_INVALID, "%s: null workspace", who);
  float* parts = static_cast<float*>(d->workspace);
  uint32_t* keys = reinterpret_cast<uint32_t*>(static_cast<char*>(d->workspace) + s.parts_bytes);
  hipLaunchKernelGGL((vocab_chunk_kernel<DT, OP>), dim3((unsigned)(d->n_rows * s.n)), dim3(256), 0, stream, *d, sc, s.chunk, s.n, parts, keys, s.groups);
  hipLaunchKernelGGL((vocab_join_kernel<DT, OP>), dim3(d->n_rows), dim3(256), 0, stream, *d, sc, s.n, parts, keys, s.groups);
  return check_launch(who);
}

// ---- gradients ----------------------------------------------------------------------------------------------
// A piece of a row a workgroup: one read and one write of the row's size, which bound it (forward and backward of 1000 x 50001 bf16 57.9
// us, 5.2 TB/s).  With p = 2^d2, d2 = (x - m) c2 - log2 s:
//   log probabilities   g = p (A + B d2) everywhere, A = -(d_lp + d_h H) / t, B = -d_h ln 2 / t, and d_lp / t more at the token
//   distillation        g = p G, G = d_loss / t, and a_j G less at the teacher's entry j
// The teacher's few columns are written once more at the end, by the piece that they lie in: looking each column up while the row streams
// by cost as much as the row where a wave's columns hold some of them (2000 x 1500 fp16 with 50 entries 31 us).
constexpr int GRAD_CHUNK = 16384;

template <int DT, int OP, int THREADS, bool ONCE>
__global__ __launch_bounds__(THREADS) void vocab_backward_kernel(tk_vocab_desc d, Scales sc, int t0, int n_chunks, int chunk) {
  typedef RowType<DT> R;
  constexpr int VE = R::VE, U = 2, STEP = THREADS * VE * U;
  // (from the last row back: its logits were read last and may still be in the last-level cache)
  const unsigned place = gridDim.x - 1 - blockIdx.x;
  const int t = t0 + (int)(place / (unsigned)n_chunks);
  const void* row = logits_row<DT>(d, t);
  const int c0 = (int)(place % (unsigned)n_chunks) * chunk;
  const int c1 = d.vocab - c0 < chunk ? d.vocab : c0 + chunk;
  void* out = static_cast<char*>(d.d_logits) + (int64_t)t * d.d_logits_stride_m * R::BYTES;
  // ln s / ln 2 in two parts: rounded to one number it is off by 7e-7 near 17, and every p of the row with it.  The second part is a factor
  // of the row's A and B.
  const float m = d.stats[t], log_s = d.stats[(int64_t)d.n_rows + t], log2_s = log_s * LOG2E;
  const float rest = __builtin_amdgcn_exp2f(-fmaf(log_s, LOG2E_REST, fmaf(log_s, LOG2E, -log2_s)));
  float A, B = 0.f, more = 0.f, qm = 0.f, log_qs = 0.f;
  int token = -1;
  bool zero;
  if constexpr (OP == DISTILL) {
    qm = d.teacher_stats[t];
    log_qs = d.teacher_stats[(int64_t)d.n_rows + t];
    const float g = d.d_loss ? d.d_loss[t * d.d_loss_stride] : 0.f;
    zero = g == 0.f || log_s == NEG_INF || qm == NEG_INF;  // (sums of nothing)
    A = qm == qm ? g * sc.inv_t : qm;
  } else {
    const int64_t at = index_at(d.tokens, d.tokens_i64, t);
    const bool live = at >= 0 && at < d.vocab;
    const float g_lp = live && d.d_logprobs ? d.d_logprobs[t * d.d_logprobs_stride] : 0.f, g_h = d.d_entropy ? d.d_entropy[t * d.d_entropy_stride] : 0.f;
    zero = (g_lp == 0.f && g_h == 0.f) || log_s == NEG_INF;  // (a sum of nothing)
    token = live ? (int)at : -1;
    A = -(g_lp + g_h * d.entropy[t]) * sc.inv_t;
    B = -g_h * LN2 * sc.inv_t;
    more = g_lp * sc.inv_t;
  }
  const float Ap = A * rest, Bp = B * rest;
  const auto gradient = [&](float x) {
    const float d2 = fmaf(x - m, sc.c2, -log2_s), p = __builtin_amdgcn_exp2f(d2);
    return OP == DISTILL ? p * Ap : p * fmaf(fmaxf(d2, D_MIN), Bp, Ap);
  };
  for (int base = c0; base < c1; base += STEP) {
    const int at = base + (int)threadIdx.x * VE;
    if (zero) {
#pragma unroll
      for (int u = 0; u < U; ++u) R::store_vec_to(out, at + u * THREADS * VE, c1, row_u32x4{0, 0, 0, 0});
      continue;
    }
    const bool full = base + STEP <= c1;
    row_u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = at + u * THREADS * VE;
      raw[u] = !full ? R::load_vec_to(row, v, c1, R::NEG_INF_BITS) : ONCE ? R::load_vec_once(row, v) : R::load_vec(row, v);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = at + u * THREADS * VE;
      float g[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) g[e] = gradient(R::element(raw[u], e));
      if (OP != DISTILL && (unsigned)(token - v) < (unsigned)VE)
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (v + e == token) g[e] += more;
      if (!full)
        R::store_vec_to(out, v, c1, R::pack(g));
      else if (ONCE)
        R::store_vec_once(out, v, R::pack(g));
      else
        R::store_vec(out, v, R::pack(g));
    }
  }
  if constexpr (OP == DISTILL) {
    if (zero) return;
    // [n_teacher] columns, [n_teacher] logits, [chunk / 32] a bit a column that an entry names, whether two name one
    extern __shared__ uint32_t lds[];
    const int n = d.n_teacher;
    uint32_t *column = lds, *logit = lds + n, *named = lds + 2 * n, *twice = named + chunk / 32;
    for (int i = threadIdx.x; i <= chunk / 32; i += THREADS) named[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += THREADS) {
      float q;
      const int v = teacher_entry(d, t, j, &q);
      column[j] = (uint32_t)v;
      logit[j] = f32_bits(q);
      const uint32_t bit = 1u << ((v - c0) & 31);
      if (v >= c0 && v < c1 && (atomicOr(&named[(v - c0) >> 5], bit) & bit)) *twice = 1;
    }
    // (this wave's part of the row has arrived where the second writing of a column finds it)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const auto weight = [&](int j) { return expf((bits_f32(logit[j]) - qm) * sc.inv_t - log_qs); };
    for (int j = threadIdx.x; j < n; j += THREADS) {
      const int v = (int)column[j];
      if (v < c0 || v >= c1) continue;
      float a = 0.f;
      if (!*twice)
        a = weight(j);
      else  // (all entries that name a column write the same)
        for (int i = 0; i < n; ++i)
          if ((int)column[i] == v) a += weight(i);
      R::store(out, v, fmaf(-a, A, gradient(R::load(row, v))));
    }
  }
}

template <int DT, int OP>
int32_t backward(const tk_vocab_desc* d, hipStream_t stream, const char* who) {
  // pieces of up to GRAD_CHUNK columns; fewer where that leaves less than sixteen workgroups a CU
  const int64_t want = cdiv(4096, d->n_rows), most = cdiv(d->vocab, 2048), least = cdiv(d->vocab, GRAD_CHUNK);
  const int64_t n = want > most ? most : want < least ? least : want;
  const int64_t chunk = cdiv(cdiv(d->vocab, n), 2048) * 2048;
  const int n_chunks = (int)cdiv(d->vocab, chunk), rows = MAX_GRID / n_chunks;
  const bool wave = d->n_rows >= 1000 && d->vocab <= SHORT_ROW, once = (int64_t)d->n_rows * d->vocab * RowType<DT>::BYTES >= ONCE_BYTES;
  auto f = wave ? vocab_backward_kernel<DT, OP, 64, false> : once ? vocab_backward_kernel<DT, OP, 256, true> : vocab_backward_kernel<DT, OP, 256, false>;
  for (int64_t t = 0; t < d->n_rows; t += rows) {
    const int now = (int)(d->n_rows - t < rows ? d->n_rows - t : rows);
    hipLaunchKernelGGL(f, dim3((unsigned)(now * n_chunks)), dim3(wave ? 64 : 256), OP == DISTILL ? d->n_teacher * 8 + chunk / 8 + 4 : 0, stream, *d, scales_of(d),
                       (int)t, n_chunks, (int)chunk);
  }
  return check_launch(who);
}

int32_t check(const tk_vocab_desc* d, const char* who) {
  if (!d) return fail(TK_ERR_INVALID, "%s: null descriptor", who);
  if (d->n_rows < 0 || d->vocab <= 0) return fail(TK_ERR_INVALID, "%s: bad sizes %d x %d", who, d->n_rows, d->vocab);
  if (d->vocab > 1 << 30) return fail(TK_ERR_UNSUPPORTED, "%s: %d columns, at most 2^30", who, d->vocab);
  if (!(d->temperature >= 1.17549435e-38f) || d->temperature == __builtin_inff())  // (a smaller one has no reciprocal)
    return fail(TK_ERR_INVALID, "%s: the temperature must be a positive, finite normal number", who);
  if (!is_row_dtype(d->logits_dtype)) return fail(TK_ERR_UNSUPPORTED, "%s: logits are fp32, bf16 or fp16", who);
  if (d->n_rows && !d->logits) return fail(TK_ERR_INVALID, "%s: null logits", who);
  return TK_OK;
}

int32_t check_teacher(const tk_vocab_desc* d, const char* who) {
  if (d->n_teacher < 0) return fail(TK_ERR_INVALID, "%s: bad number of teacher entries %d", who, d->n_teacher);
  if (d->n_teacher > TK_VOCAB_MAX_TEACHER) return fail(TK_ERR_UNSUPPORTED, "%s: %d teacher entries a row, at most %d", who, d->n_teacher, TK_VOCAB_MAX_TEACHER);
  if (!is_row_dtype(d->teacher_dtype)) return fail(TK_ERR_UNSUPPORTED, "%s: teacher logits are fp32, bf16 or fp16", who);
  if (d->n_rows && d->n_teacher && (!d->teacher_logits || !d->teacher_indx)) return fail(TK_ERR_INVALID, "%s: null teacher", who);
  return TK_OK;
}

}  // namespace
}  // namespace tk

using namespace tk;

// f<type of the logits, op>(descriptor, stream, name)
#define TK_VOCAB_CALL(f, op, who)                                                                                                            \
  (d->logits_dtype == TK_F32 ? f<TK_F32, op> : d->logits_dtype == TK_BF16 ? f<TK_BF16, op> : f<TK_F16, op>)(d, static_cast<hipStream_t>(stream), who)

extern "C" int64_t tk_vocab_workspace_bytes(int32_t n_rows, int32_t vocab, int32_t k) {
  if (n_rows <= 0 || vocab <= 0) return 0;
  int64_t most = 0;  // (of what the logits' type and addresses may call for)
  for (int shift : {0, 3, 7}) {
    const int64_t n = split_of(n_rows, vocab, k, shift).bytes;
    most = n > most ? n : most;
  }
  return most;
}

extern "C" int32_t tk_token_logprobs(const tk_vocab_desc* d, tk_stream_t stream) {
  if (int32_t e = check(d, "tk_token_logprobs")) return e;
  if (d->k < 0 || d->k > d->vocab) return fail(TK_ERR_INVALID, "tk_token_logprobs: %d alternatives of %d", d->k, d->vocab);
  if (d->k > TK_VOCAB_MAX_TOP || (d->k && d->vocab > TK_VOCAB_MAX_TOP_COLUMNS))
    return fail(TK_ERR_UNSUPPORTED, "tk_token_logprobs: at most %d alternatives, of at most %d columns", TK_VOCAB_MAX_TOP, TK_VOCAB_MAX_TOP_COLUMNS);
  if (d->n_rows == 0) return TK_OK;
  if (!d->tokens || !d->logprobs || !d->entropy || (d->k && (!d->top_logprobs || !d->top_indx))) return fail(TK_ERR_INVALID, "tk_token_logprobs: null pointer");
  return d->k ? TK_VOCAB_CALL(forward, LOGPROBS_TOP, "tk_token_logprobs") : TK_VOCAB_CALL(forward, LOGPROBS, "tk_token_logprobs");
}

extern "C" int32_t tk_token_logprobs_backward(const tk_vocab_desc* d, tk_stream_t stream) {
  if (int32_t e = check(d, "tk_token_logprobs_backward")) return e;
  if (d->n_rows == 0) return TK_OK;
  if (!d->tokens || !d->entropy || !d->stats || !d->d_logits) return fail(TK_ERR_INVALID, "tk_token_logprobs_backward: null pointer");
  return TK_VOCAB_CALL(backward, LOGPROBS, "tk_token_logprobs_backward");
}

extern "C" int32_t tk_distill_topk(const tk_vocab_desc* d, tk_stream_t stream) {
  if (int32_t e = check(d, "tk_distill_topk")) return e;
  if (int32_t e = check_teacher(d, "tk_distill_topk")) return e;
  if (d->n_rows == 0) return TK_OK;
  if (!d->loss) return fail(TK_ERR_INVALID, "tk_distill_topk: null pointer");
  return TK_VOCAB_CALL(forward, DISTILL, "tk_distill_topk");
}

extern "C" int32_t tk_distill_topk_backward(const tk_vocab_desc* d, tk_stream_t stream) {
  if (int32_t e = check(d, "tk_distill_topk_backward")) return e;
  if (int32_t e = check_teacher(d, "tk_distill_topk_backward")) return e;
  if (d->n_rows == 0) return TK_OK;
  if (!d->stats || !d->teacher_stats || !d->d_logits) return fail(TK_ERR_INVALID, "tk_distill_topk_backward: null pointer");
  return TK_VOCAB_CALL(backward, DISTILL, "tk_distill_topk_backward");
}
