// Categorical loss against a target and a teacher's top logits, per row of
// logits z[0..V):
//
//   l1 = ln sum exp(z),  lT = ln sum exp(z / T)
//   p  = softmax over the teacher's entries of t / T  (entries with id in [0, V))
//   loss = [target in [0, V)]  ce_weight (l1 - z[target]) + z_weight l1^2
//        + [a teacher entry]   kd_weight T^2 sum_e p_e (ln p_e - z[id_e] / T + lT)
//
// the first line being the categorical head's cross-entropy with z-loss
// (confluence/confluence/loss.py:33-170). Gradient for an upstream g:
//
//   dz_v = g ( [target] ((ce_weight + 2 z_weight l1) softmax(z)_v - ce_weight 1[v = target])
//            + [teacher] kd_weight T (softmax(z / T)_v - sum over e with id_e = v of p_e) )
//
// Forward: one pass over the row; a thread keeps a running maximum m and the
// sums of exp(z - m) and exp((z - m) / T), rescaled when m grows, so that no
// logit is read twice. m, the logarithms of the two sums (l1 = m + ln s1,
// lT = m / T + ln sT; apart, so that logits far from zero lose nothing) and,
// apart in the same way, the teacher's maximum and the logarithm of its sum
// are kept for the backward, which is elementwise: no sum over the row, and
// the few columns that a target or an entry names are written once more by the
// thread that owns the first entry of that id, with all of them (equal ids
// included) added in a fixed order: the same bits on every run. Statistics,
// sums and losses are fp32; the gradient is rounded once to the logits' type.
// Rows without target and entries read no logits.

namespace rt {
namespace distill {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxEntries = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct Weights {
  float inv_t, ce, z, kd, t;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// 16 bytes of a row, kept as words: 16-bit elements are only taken apart in
// pairs.
template <typename T>
struct __align__(16) Pack {
  static constexpr int kN = 16 / sizeof(T);
  uint32_t w[4];
};
template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const Pack<T>* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  return {{u.x, u.y, u.z, u.w}};
}
template <typename T>
__device__ __forceinline__ uint32_t minus_inf_word() {
  return sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
}
__device__ __forceinline__ float2 pair_of(const Pack<float>& p, int i) {
  return make_float2(__uint_as_float(p.w[2 * i]), __uint_as_float(p.w[2 * i + 1]));
}
__device__ __forceinline__ float2 pair_of(const Pack<__nv_bfloat16>& p, int i) { return unpack_bf16x2(p.w[i]); }
__device__ __forceinline__ float2 pair_of(const Pack<__half>& p, int i) {
  return __half22float2(*reinterpret_cast<const __half2*>(&p.w[i]));
}
__device__ __forceinline__ void set_pair(Pack<float>& p, int i, float2 f) {
  p.w[2 * i] = __float_as_uint(f.x);
  p.w[2 * i + 1] = __float_as_uint(f.y);
}
__device__ __forceinline__ void set_pair(Pack<__nv_bfloat16>& p, int i, float2 f) { p.w[i] = pack_bf16x2(f.x, f.y); }
__device__ __forceinline__ void set_pair(Pack<__half>& p, int i, float2 f) {
  const __half2 h = __floats2half2_rn(f.x, f.y);
  p.w[i] = *reinterpret_cast<const uint32_t*>(&h);
}

// The 16-byte steps of a row: rows of odd widths start anywhere, so up to
// kN - 1 elements lie before the first step and behind the last.
template <typename T>
struct Steps {
  int head, count, rest;  // elements before, steps, elements outside the steps
  __device__ __forceinline__ Steps(long long offset, int V) {
    constexpr int n = Pack<T>::kN;
    head = min(V, (int)((n - offset % n) % n));
    count = (V - head) / n;
    rest = V - count * n;
  }
  __device__ __forceinline__ int outside(int i) const { return i < head ? i : i + count * Pack<T>::kN; }
};

__device__ __forceinline__ float exp_of(float x) { return fast_exp2(x * kLog2e); }
__device__ __forceinline__ float2 exp2_pair(float2 x) { return make_float2(fast_exp2(x.x), fast_exp2(x.y)); }
__device__ __forceinline__ float2 two(float x) { return make_float2(x, x); }
__device__ __forceinline__ bool named(int id, int V) { return id >= 0 && id < V; }

// TM: what is known of the temperature, to spend one exponential per element
// where two would be needed (two exceed the MUFU's rate on bf16 logits from
// HBM): 1, 2 and 4 take exp(z) as that power of exp(z / T); 0 is any other.
template <int TM>
__device__ __forceinline__ float power(float e) {
  return TM == 1 ? e : TM == 2 ? e * e : (e * e) * (e * e);
}

// A running maximum and the sums of exp(z - m), exp((z - m) / T) below it.
struct Online {
  float m, s1, sT;
};

// c = log2(e) / T
template <int TM>
__device__ __forceinline__ void raise_max(Online& a, float m, float c) {
  if (m > a.m) {  // -inf stays -inf: a row (so far) of -inf only has no terms
    const float e = fast_exp2((a.m - m) * c);
    a.s1 *= TM == 0 ? exp_of(a.m - m) : power<TM>(e);
    a.sT *= e;
    a.m = m;
  }
}

// Adds U steps of 16 bytes: their maximum first, then their terms.
template <typename T, int TM, int U>
__device__ __forceinline__ void add_steps(Online& a, const Pack<T> (&p)[U], float c) {
  constexpr int n = Pack<T>::kN;
  float m = a.m;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float2 f = pair_of(p[u], i);
      m = fmax3(m, f.x, f.y);
    }
  raise_max<TM>(a, m, c);
  const float2 off = two(a.m == -INFINITY ? 0.f : -a.m);
  float2 s1 = make_float2(a.s1, 0.f), sT = make_float2(a.sT, 0.f);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float2 x = fadd2(pair_of(p[u], i), off);
      const float2 e = exp2_pair(fmul2(x, two(c)));
      sT = fadd2(sT, e);
      if (TM == 0) s1 = fadd2(s1, exp2_pair(fmul2(x, two(kLog2e))));
      if (TM == 2) s1 = ffma2(e, e, s1);
      if (TM == 4) {
        const float2 e2 = fmul2(e, e);
        s1 = ffma2(e2, e2, s1);
      }
    }
  a.sT = sT.x + sT.y;
  a.s1 = TM == 1 ? a.sT : s1.x + s1.y;
}

template <int TM>
__device__ __forceinline__ void add_one(Online& a, float z, float c) {
  raise_max<TM>(a, z, c);
  const float x = a.m == -INFINITY ? z : z - a.m;
  const float e = fast_exp2(x * c);
  a.sT += e;
  a.s1 = TM == 1 ? a.sT : a.s1 + (TM == 0 ? exp_of(x) : power<TM>(e));
}

// 16-byte step i of a row, or one of -inf behind its last (which adds nothing).
template <typename T>
__device__ __forceinline__ Pack<T> step_or_nothing(const Pack<T>* p, int i, int count) {
  const uint32_t m = minus_inf_word<T>();
  Pack<T> q = {{m, m, m, m}};
  if (i < count) q = load_pack(p + i);
  return q;
}

constexpr int kBatch = 4;  // loads of a row in flight per thread

// The first steps of a thread's share of a row: first, first + stride, ...
template <typename T>
struct Batch {
  Pack<T> q[kBatch];
  __device__ __forceinline__ void load(const T* z, const Steps<T>& st, int i, int stride) {
    const Pack<T>* p = reinterpret_cast<const Pack<T>*>(z + st.head);
    if (i + (kBatch - 1) * stride < st.count) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) q[u] = load_pack(p + i + u * stride);
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) q[u] = step_or_nothing(p, i + u * stride, st.count);
    }
  }
};

// This thread's share of a row, of which `q` holds the first steps.
template <typename T, int TM>
__device__ __forceinline__ Online scan_row(const T* z, const Steps<T>& st, Batch<T>& q, int first, int stride,
                                           float c) {
  Online a = {-INFINITY, 0.f, 0.f};
  if (st.count <= kBatch / 2 * stride) {  // a short row: half a batch (30000 x 300 bf16, forward: 20.5 -> 17.7 us)
    Pack<T> half[kBatch / 2];
#pragma unroll
    for (int u = 0; u < kBatch / 2; ++u) half[u] = q.q[u];
    if (first < st.count) add_steps<T, TM, kBatch / 2>(a, half, c);
  } else if (first < st.count) {
    add_steps<T, TM, kBatch>(a, q.q, c);
  }
  for (int i = first + kBatch * stride; i < st.count; i += kBatch * stride) {
    q.load(z, st, i, stride);
    add_steps<T, TM, kBatch>(a, q.q, c);
  }
  for (int j = first; j < st.rest; j += stride) add_one<TM>(a, to_f32(z[st.outside(j)]), c);
  return a;
}

__device__ __forceinline__ float warp_max(float x) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
  return m;
}

// The warp's sums, brought to its maximum first (every lane gets them).
template <int TM>
__device__ __forceinline__ Online warp_merge(Online a, float c) {
  raise_max<TM>(a, warp_max(a.m), c);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    if (TM != 1) a.s1 += __shfl_xor_sync(0xFFFFFFFFu, a.s1, off);
    a.sT += __shfl_xor_sync(0xFFFFFFFFu, a.sT, off);
  }
  if (TM == 1) a.s1 = a.sT;
  return a;
}

// A row's teacher entries, by a warp: lane l holds entries l, l + 32, ...
struct Teacher {
  int id[kMaxEntries / 32];
  float t[kMaxEntries / 32];
  __device__ __forceinline__ void load(const int32_t* ids, const float* tl, int K, int lane) {
#pragma unroll
    for (int j = 0; j < kMaxEntries / 32; ++j) {
      id[j] = -1;
      t[j] = -INFINITY;
      if (32 * j < K && lane + 32 * j < K) {
        id[j] = ids[lane + 32 * j];
        t[j] = tl[lane + 32 * j];
      }
    }
  }
  // Whether one of them counts: a column of the row, and not -inf.
  __device__ __forceinline__ bool any(int K, int V) {
    bool some = false;
#pragma unroll
    for (int j = 0; j < kMaxEntries / 32; ++j)
      if (32 * j < K) {
        if (!named(id[j], V) || t[j] == -INFINITY) id[j] = -1;
        some = some || id[j] >= 0;
      }
    return __any_sync(0xFFFFFFFFu, some);
  }
};

// What a teacher adds to the loss, but for the row's m and ln sT: with
// x = t - max t and p = exp(x / T), the Kullback-Leibler sum is
//   ln sT + (m - z_ref) / T + kl,  kl = sum p (x - (z_e - z_ref)) / T / sum p - ln sum p
struct TeacherSums {
  float kl, z_ref, top, ls;  // top = max t, ls = ln sum exp((t - top) / T)
};

template <typename T>
__device__ __forceinline__ TeacherSums teacher_sums(const Teacher& te, const T* row, int K, float inv_t) {
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  float z[kMaxEntries / 32], top = -INFINITY, z_ref = -INFINITY, s = 0.f, u = 0.f;
#pragma unroll
  for (int j = 0; j < kMaxEntries / 32; ++j)
    if (32 * j < K) {
      z[j] = te.id[j] >= 0 ? to_f32(row[te.id[j]]) : -INFINITY;
      if (te.id[j] >= 0) top = fmaxf(top, te.t[j]);
    }
  top = warp_max(top);
#pragma unroll
  for (int j = 0; j < kMaxEntries / 32; ++j)
    if (32 * j < K) z_ref = fmaxf(z_ref, z[j]);
  z_ref = warp_max(z_ref);
  if (z_ref == -INFINITY) z_ref = 0.f;
#pragma unroll
  for (int j = 0; j < kMaxEntries / 32; ++j)
    if (32 * j < K && te.id[j] >= 0) {
      const float x = te.t[j] - top;
      const float p = exp_of(x * inv_t);
      s += p;
      if (p != 0.f) u += p * ((x - (z[j] - z_ref)) * inv_t);
    }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s += __shfl_xor_sync(kAll, s, off);
    u += __shfl_xor_sync(kAll, u, off);
  }
  const float ls = logf(s);
  return {u / s - ls, z_ref, top, ls};  // ls is NaN if one of t is
}

// Loss and statistics of a row: m, ln s1, ln sT, the teacher's logarithm (-inf:
// no teacher), and its maximum in an array behind all rows' first four.
__device__ __forceinline__ void finish_row(const Online& a, const TeacherSums& ts, bool hard, bool soft,
                                           float z_target, const Weights& w, float* loss, float4* stats,
                                           float* teacher_top) {
  const float ls1 = logf(a.s1), lsT = logf(a.sT), l1 = a.m + ls1;
  float total = 0.f;
  if (soft) total = w.kd * w.t * w.t * (ts.kl + (a.m - ts.z_ref) * w.inv_t + lsT);
  if (hard) total += w.ce * ((a.m - z_target) + ls1) + w.z * l1 * l1;
  *loss = total;
  *stats = make_float4(a.m, ls1, lsT, soft ? ts.ls : -INFINITY);
  *teacher_top = ts.top;
}

__device__ __forceinline__ void finish_dead_row(float* loss, float4* stats, float* teacher_top) {
  *loss = 0.f;
  *stats = make_float4(0.f, 0.f, 0.f, -INFINITY);
  *teacher_top = 0.f;
}

// One warp per row (short rows).
template <typename T, int TM>
__global__ void __launch_bounds__(kThreads) distill_fwd_warp_kernel(
    const T* __restrict__ logits, long long rows, int V, const int32_t* __restrict__ target,
    const int32_t* __restrict__ ids, const float* __restrict__ teacher, int K, Weights w, float* __restrict__ loss,
    float4* __restrict__ stats, float* __restrict__ tops) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= rows) return;  // a whole warp
  const T* z = logits + row * V;
  const int tgt = target ? target[row] : -1;
  Teacher te;
  te.load(ids + row * K, teacher + row * K, K, lane);
  const bool hard = named(tgt, V), soft = te.any(K, V);
  if (!hard && !soft) {
    if (lane == 0) finish_dead_row(loss + row, stats + row, tops + row);
    return;
  }
  const float c = w.inv_t * kLog2e;
  const Steps<T> st(row * V, V);
  Batch<T> q;
  q.load(z, st, lane, 32);
  const float z_target = hard ? to_f32(z[tgt]) : 0.f;
  TeacherSums ts = {0.f, 0.f, 0.f, 0.f};
  if (soft) ts = teacher_sums(te, z, K, w.inv_t);
  const Online a = warp_merge<TM>(scan_row<T, TM>(z, st, q, lane, 32, c), c);
  if (lane == 0) finish_row(a, ts, hard, soft, z_target, w, loss + row, stats + row, tops + row);
}

// One block per row, or a cluster of gridDim.x / rows blocks whose sums the
// first joins through distributed shared memory. The last warp of a block has
// no share of the row: it looks after the teacher, so that its gathers and
// sums run beside the row's (7 x 100003 fp32: 8.4 -> 6.4 us).
constexpr int kRowThreads = kThreads + 32;

template <typename T, int TM>
__global__ void __launch_bounds__(kRowThreads, 4) distill_fwd_kernel(
    const T* __restrict__ logits, long long rows, int V, const int32_t* __restrict__ target,
    const int32_t* __restrict__ ids, const float* __restrict__ teacher, int K, Weights w, float* __restrict__ loss,
    float4* __restrict__ stats, float* __restrict__ tops) {
  namespace cg = cooperative_groups;
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  __shared__ Online s_part[kWarps], s_block;
  __shared__ TeacherSums s_teacher;
  __shared__ float s_target;
  __shared__ int s_soft;
  const cg::cluster_group cluster = cg::this_cluster();
  const int split = cluster.num_blocks(), part = cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = blockIdx.x / split;
  const T* z = logits + row * V;
  const int tgt = target ? target[row] : -1;
  const bool hard = named(tgt, V);
  Teacher te;
  if (warp == kWarps) {
    te.load(ids + row * K, teacher + row * K, K, lane);
    const bool soft = te.any(K, V);
    if (lane == 0) s_soft = soft;
  }
  if (!hard) {  // the row counts only if its teacher does
    __syncthreads();
    if (!s_soft) {  // the whole cluster
      if (threadIdx.x == 0 && part == 0) finish_dead_row(loss + row, stats + row, tops + row);
      return;
    }
  }
  const float c = w.inv_t * kLog2e;
  const Steps<T> st(row * V, V);
  if (warp < kWarps) {
    const int first = part * kThreads + (int)threadIdx.x, stride = split * kThreads;
    Batch<T> q;
    q.load(z, st, first, stride);
    const Online a = warp_merge<TM>(scan_row<T, TM>(z, st, q, first, stride, c), c);
    if (lane == 0) s_part[warp] = a;
  } else if (part == 0) {
    __syncwarp();
    TeacherSums ts = {0.f, 0.f, 0.f, 0.f};
    if (s_soft) ts = teacher_sums(te, z, K, w.inv_t);
    if (lane == 0) {
      s_teacher = ts;
      s_target = hard ? to_f32(z[tgt]) : 0.f;
    }
  }
  __syncthreads();
  Online a = {-INFINITY, 0.f, 0.f};
  if (warp == 0) {
    if (lane < kWarps) a = s_part[lane];
    a = warp_merge<TM>(a, c);
  }
  if (split > 1) {
    if (threadIdx.x == 0) s_block = a;
    cluster.sync();
    if (part == 0 && warp == 0) {
      if (lane > 0) a = {-INFINITY, 0.f, 0.f};
      if (lane > 0 && lane < split) a = *cluster.map_shared_rank(&s_block, lane);
      a = warp_merge<TM>(a, c);
    }
    cluster.sync();  // the other blocks' memory stays until it has been read
  }
  if (part == 0 && threadIdx.x == 0)
    finish_row(a, s_teacher, hard, s_soft, s_target, w, loss + row, stats + row, tops + row);
}

// What turns a logit into its gradient, but for the named columns:
// c1 softmax(z) + ct softmax(z / T).
template <int TM>
struct RowGrad {
  float m, c, k1, kT, c1, ct;  // k1, kT: log2 of the sums
  __device__ __forceinline__ RowGrad(const float4& st, const Weights& w, bool hard, bool soft, float g) {
    m = st.x;
    c = w.inv_t * kLog2e;
    k1 = st.y * kLog2e;
    kT = st.z * kLog2e;
    c1 = hard ? g * (w.ce + 2.f * w.z * (st.x + st.y)) : 0.f;
    ct = soft ? g * w.kd * w.t : 0.f;
    // exp(z - m) / s1 = (exp((z - m) / T) / sT)^TM * sT^TM / s1
    if (TM != 0) c1 *= fast_exp2((float)TM * kT - k1);
  }
  __device__ __forceinline__ float2 dense(float2 z) const {
    const float2 x = fadd2(z, two(-m));
    const float2 e = exp2_pair(ffma2(x, two(c), two(-kT)));
    if (TM == 1) return fmul2(e, two(c1 + ct));
    if (TM == 2) return fmul2(e, ffma2(e, two(c1), two(ct)));
    if (TM == 4) return fmul2(e, ffma2(fmul2(e, fmul2(e, e)), two(c1), two(ct)));
    const float2 f = exp2_pair(ffma2(x, two(kLog2e), two(-k1)));
    return ffma2(f, two(c1), fmul2(e, two(ct)));
  }
  __device__ __forceinline__ float dense(float z) const { return dense(two(z)).x; }
};

// Entry e's column gets all that names it: the teacher's share of every entry
// of that id and the target, by the first such entry (e = K: the target, if
// no entry has its id). s_id and s_p are the row's entries (id -1: none), z
// the logit of that column.
template <typename T, int TM>
__device__ __forceinline__ void named_column(const RowGrad<TM>& rg, float z, T* dz, const int* s_id, const float* s_p,
                                             int id, int e, int K, int tgt, float target_part) {
  float p = 0.f;
  bool first = true;
#pragma unroll 8
  for (int f = 0; f < K; ++f) {
    const bool same = s_id[f] == id;
    p += same ? s_p[f] : 0.f;
    first = first && !(same && f < e);
  }
  if (!first) return;
  float d = rg.dense(z) - rg.ct * p;
  if (id == tgt) d -= target_part;
  dz[id] = from_f32<T>(d);
}

// Logits are read for the last time and gradients written once: with
// streaming (evict-first) accesses, which at 4096 x 65537 bf16 take the
// backward from 199 to 184 us.
template <typename T>
__device__ __forceinline__ Pack<T> load_streaming(const Pack<T>* p) {
  const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
  return {{u.x, u.y, u.z, u.w}};
}

template <typename T, int TM>
__device__ __forceinline__ void write_step(const RowGrad<TM>& rg, Pack<T>& q, Pack<T>* d) {
#pragma unroll
  for (int j = 0; j < Pack<T>::kN / 2; ++j) set_pair(q, j, rg.dense(pair_of(q, j)));
  __stcs(reinterpret_cast<uint4*>(d), make_uint4(q.w[0], q.w[1], q.w[2], q.w[3]));
}
template <typename T, int TM, int U>
__device__ __forceinline__ void write_steps(const RowGrad<TM>& rg, const Pack<T>* p, Pack<T>* d, int i, int stride) {
  Pack<T> q[U];
#pragma unroll
  for (int u = 0; u < U; ++u) q[u] = load_streaming(p + i + u * stride);
#pragma unroll
  for (int u = 0; u < U; ++u) write_step(rg, q[u], d + i + u * stride);
}

// The dense gradient of steps [begin, end) of a row, this thread's being
// begin + first, + stride, ..., U loads in flight; zeros without `live`.
template <typename T, int TM, int U>
__device__ __forceinline__ void write_row(const RowGrad<TM>& rg, bool live, const T* z, T* dz, const Steps<T>& st,
                                          int begin, int end, int first, int stride) {
  const Pack<T>* p = reinterpret_cast<const Pack<T>*>(z + st.head);
  Pack<T>* d = reinterpret_cast<Pack<T>*>(dz + st.head);
  int i = begin + first;
  if (!live) {
    for (; i < end; i += stride) __stcs(reinterpret_cast<uint4*>(d + i), make_uint4(0u, 0u, 0u, 0u));
    return;
  }
  for (; i + (U - 1) * stride < end; i += U * stride) write_steps<T, TM, U>(rg, p, d, i, stride);
  if (i < end) {  // the last steps, all of their loads first
    Pack<T> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = load_streaming(p + min(i + u * stride, end - 1));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * stride < end) write_step(rg, q[u], d + i + u * stride);
  }
}

// Of a warp's entries, one a lane with `same` the lanes of its id: the sum of
// the id's shares, in the lanes' order.
__device__ __forceinline__ float shares_of_id(uint32_t same, bool counts, float p, int lane) {
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  if (!__any_sync(kAll, counts && (same & (same - 1u)) != 0u)) return p;  // no id twice
  float sum = 0.f;
  uint32_t left = counts ? same : 0u;
  while (__any_sync(kAll, left != 0u)) {  // as often as the most frequent id is there
    const float q = __shfl_sync(kAll, p, left ? __ffs(left) - 1 : lane);
    sum += left ? q : 0.f;
    left &= left - 1u;
  }
  return sum;
}

// Slots of a warp's table of named columns: twice the entries, so that a free
// one is near. Backward of 32768 x 256 fp32 with 64 entries: 34 us, 58 with
// every entry held against every other.
constexpr int kSlotBits = 8, kSlots = 1 << kSlotBits;
static_assert(kSlots >= 2 * kMaxEntries && kSlotBits * kMaxEntries / 32 <= 32, "table of named columns");

// One warp per row (short rows).
template <typename T, int TM>
__global__ void __launch_bounds__(kThreads) distill_bwd_warp_kernel(
    const T* __restrict__ logits, long long rows, int V, const int32_t* __restrict__ target,
    const int32_t* __restrict__ ids, const float* __restrict__ teacher, int K, Weights w,
    const float4* __restrict__ stats, const float* __restrict__ tops, const float* __restrict__ grad,
    T* __restrict__ dlogits) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  __shared__ int s_key[kWarps][kSlots];
  __shared__ float s_share[kWarps][kSlots];
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= rows) return;  // a whole warp
  const T* z = logits + row * V;
  T* dz = dlogits + row * V;
  const float4 st4 = stats[row];
  const float top = tops[row];
  const int tgt = target && named(target[row], V) ? target[row] : -1;
  const bool hard = tgt >= 0, soft = st4.w != -INFINITY, live = hard || soft;
  const float g = live ? grad[row] : 0.f;
  const RowGrad<TM> rg(st4, w, hard, soft, g);
  const Steps<T> st(row * V, V);
  // up to 32 entries: one a lane, its logit and the target's ahead of their use
  const bool few = K <= 32;
  int id = -1;
  float p = 0.f, x = 0.f, x_target = 0.f;
  if (soft && few && lane < K) {
    const int c = ids[row * K + lane];
    const float t = teacher[row * K + lane];
    if (named(c, V)) {
      id = c;
      x = to_f32(z[c]);
      p = exp_of((t - top) * w.inv_t - st4.w);
    }
  }
  if (hard) x_target = to_f32(z[tgt]);
  // more: their shares by id, in a table; the first entry of an id keeps its slot
  int* key = s_key[threadIdx.x >> 5];
  float* share = s_share[threadIdx.x >> 5];
  int own[kMaxEntries / 32];
  uint32_t own_slots = 0u;
  if (soft && !few) {
#pragma unroll
    for (int i = 0; i < kSlots; i += 32) key[i + lane] = -1;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kMaxEntries / 32; ++j) {
      own[j] = -1;
      if (32 * j >= K) continue;
      int c = -1;
      float q = 0.f;
      if (32 * j + lane < K) {
        c = ids[row * K + 32 * j + lane];
        c = named(c, V) ? c : -1;
        q = c >= 0 ? exp_of((teacher[row * K + 32 * j + lane] - top) * w.inv_t - st4.w) : 0.f;
      }
      const uint32_t same = __match_any_sync(kAll, c);
      q = shares_of_id(same, c >= 0, q, lane);
      if (c >= 0 && __ffs(same) - 1 == lane) {
        uint32_t i = (uint32_t)c * 2654435769u >> (32 - kSlotBits);  // multiplicative hashing, then the next slots
        int k;
        while ((k = atomicCAS(key + i, -1, c)) != -1 && k != c) i = (i + 1) % kSlots;
        if (k == -1) {
          own[j] = c;
          own_slots |= i << (kSlotBits * j);
          share[i] = q;
        } else {
          share[i] += q;
        }
      }
      __syncwarp();
    }
  }
  write_row<T, TM, 4>(rg, live, z, dz, st, 0, st.count, lane, 32);
  for (int i = lane; i < st.rest; i += 32) {
    const int c = st.outside(i);
    dz[c] = from_f32<T>(live ? rg.dense(to_f32(z[c])) : 0.f);
  }
  if (!live) return;
  __syncwarp();  // the named columns, after the dense values
  bool target_named = false;  // among the entries
  if (few) {
    const uint32_t same = __match_any_sync(kAll, id);
    p = shares_of_id(same, id >= 0, p, lane);
    target_named = __any_sync(kAll, hard && id == tgt);
    if (id >= 0 && __ffs(same) - 1 == lane)
      dz[id] = from_f32<T>(rg.dense(x) - rg.ct * p - (id == tgt ? g * w.ce : 0.f));
  } else if (soft) {
    float x[kMaxEntries / 32];
#pragma unroll
    for (int j = 0; j < kMaxEntries / 32; ++j)
      if (own[j] >= 0) x[j] = to_f32(z[own[j]]);
#pragma unroll
    for (int j = 0; j < kMaxEntries / 32; ++j)
      if (own[j] >= 0) {
        const float q = share[own_slots >> (kSlotBits * j) & (kSlots - 1)];
        target_named = target_named || own[j] == tgt;
        dz[own[j]] = from_f32<T>(rg.dense(x[j]) - rg.ct * q - (own[j] == tgt ? g * w.ce : 0.f));
      }
    target_named = __any_sync(kAll, target_named);
  }
  if (hard && !target_named && lane == 0) dz[tgt] = from_f32<T>(rg.dense(x_target) - g * w.ce);
}

// Blocks of `span` steps of a row: gridDim.x = rows * parts. Six blocks per SM,
// with up to 56 bytes a thread spilled: backward, us, 6 / 5 / 4 per SM, 4096 x
// 65537 bf16 at T = 2 194 / 197 / 210, at T = 1.5 193 / 203 / 222; but 2048 x
// 65536 fp32 at T = 1 186 / 179 / 182.
template <typename T, int TM>
__global__ void __launch_bounds__(kThreads, 6) distill_bwd_kernel(
    const T* __restrict__ logits, long long rows, int V, const int32_t* __restrict__ target,
    const int32_t* __restrict__ ids, const float* __restrict__ teacher, int K, Weights w,
    const float4* __restrict__ stats, const float* __restrict__ tops, const float* __restrict__ grad, int parts,
    int span, T* __restrict__ dlogits) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  __shared__ int s_id[kMaxEntries];
  __shared__ float s_p[kMaxEntries];
  const int part = (int)(blockIdx.x % parts);
  const long long row = blockIdx.x / parts;
  const T* z = logits + row * V;
  T* dz = dlogits + row * V;
  const float4 st4 = stats[row];
  const float top = tops[row];
  const int tgt = target && named(target[row], V) ? target[row] : -1;
  const bool hard = tgt >= 0, soft = st4.w != -INFINITY, live = hard || soft;
  const float g = live ? grad[row] : 0.f;
  const RowGrad<TM> rg(st4, w, hard, soft, g);
  const Steps<T> st(row * V, V);
  const int begin = part * span, end = min(st.count, begin + span);
  const bool last = part == parts - 1;  // with the elements outside the steps
  // the row's entries; thread e holds entry e and, behind them, the target,
  // if its column is this part's, with the logit there ahead of its use
  const int entries = soft ? K : 0, e = threadIdx.x;
  int id = e == entries ? tgt : -1;
  if (e < entries) {
    const int c = ids[row * K + e];
    if (named(c, V)) id = c;
    s_id[e] = id;
    s_p[e] = id >= 0 ? exp_of((teacher[row * K + e] - top) * w.inv_t - st4.w) : 0.f;
  }
  const int step = id < st.head ? -1 : (id - st.head) / Pack<T>::kN;  // -1, count: outside
  if (!((step >= begin && step < end) || (last && id >= 0 && (step < 0 || step >= st.count)))) id = -1;
  const float x = id >= 0 ? to_f32(z[id]) : 0.f;
  write_row<T, TM, 4>(rg, live, z, dz, st, begin, end, threadIdx.x, kThreads);
  if (last)
    for (int i = threadIdx.x; i < st.rest; i += kThreads) {
      const int c = st.outside(i);
      dz[c] = from_f32<T>(live ? rg.dense(to_f32(z[c])) : 0.f);
    }
  if (!live) return;
  __syncthreads();  // the named columns, after the dense values
  if (id >= 0) named_column<T, TM>(rg, x, dz, s_id, s_p, id, e, entries, tgt, g * w.ce);
}

// Whether a row is taken by one warp: short rows always, longer ones while
// there are rows enough for 16 warps per SM. Measured, block against warp per
// row (forward / backward, us): 8192 x 1024 fp32 41 / 23 against 8.5 / 14,
// 8192 x 4096 bf16 58 / 63 against 15 / 29, 2048 x 16384 bf16 19 / 27 against
// 19 / 47, 512 x 4096 bf16 6.4 / 4.1 against 6.4 / 6.1.
inline bool warp_per_row(int64_t rows, long long row_bytes, bool backward) {
  return row_bytes <= 4096 || (rows >= 16 * 148 && row_bytes <= (backward ? 16384 : 32768));
}
// Steps of 16 bytes that a block of the backward takes.
constexpr int kSpan = 16 * kThreads;

bool valid(int64_t rows, int32_t vocab, int32_t dtype, int32_t entries, float temperature, float ce, float z, float kd) {
  return rows >= 0 && rows <= INT32_MAX && vocab > 0 && entries >= 0 && dtype >= RT_FP32 && dtype <= RT_FP16 &&
         temperature > 0.f && std::isnormal(temperature * temperature) &&  // and with it 1 / T is finite
         std::isfinite(ce) && std::isfinite(z) && std::isfinite(kd);
}

}  // namespace distill
}  // namespace rt

namespace rt {
namespace distill {

// Calls f with the logits' type and what is known of the temperature.
template <typename F>
int with_types(int32_t dtype, float temperature, const F& f) {
  auto typed = [&](auto* z) {
    if (temperature == 1.f) return f(z, std::integral_constant<int, 1>());
    if (temperature == 2.f) return f(z, std::integral_constant<int, 2>());
    if (temperature == 4.f) return f(z, std::integral_constant<int, 4>());
    return f(z, std::integral_constant<int, 0>());
  };
  if (dtype == RT_FP32) return typed(static_cast<float*>(nullptr));
  if (dtype == RT_BF16) return typed(static_cast<__nv_bfloat16*>(nullptr));
  return typed(static_cast<__half*>(nullptr));
}

// Blocks per row of the forward: more than one (a cluster) for few rows, while
// each still has 2048 elements. One block against a cluster of 8, us: 1 x
// 131072 bf16 13.6 / 6.3, 7 x 100003 fp32 12.6 / 6.4, 32 x 65537 bf16 8.5 /
// 6.4; 300 x 50001 bf16 12.7 against 14.5 in clusters of 2.
int row_split(int64_t rows, int32_t vocab) {
  int split = 1;
  while (split < 8 && rows * split <= 128 && vocab >= 2 * split * 2048) split *= 2;
  return split;
}

}  // namespace distill
}  // namespace rt

extern "C" int rt_distill_loss(const void* logits, int32_t dtype, int64_t rows, int32_t vocab, const int32_t* target,
                               const int32_t* teacher_ids, const float* teacher_logits, int32_t entries,
                               float temperature, float ce_weight, float z_weight, float kd_weight, float* loss,
                               float* stats, void* stream) {
  using namespace rt;
  if (!distill::valid(rows, vocab, dtype, entries, temperature, ce_weight, z_weight, kd_weight))
    return RT_ERR_INVALID_ARGUMENT;
  if (entries > distill::kMaxEntries) return RT_ERR_UNSUPPORTED;
  if (rows == 0) return RT_OK;
  if (!ok16(logits) || !loss || !ok16(stats) || (entries > 0 && (!teacher_ids || !teacher_logits)))
    return RT_ERR_INVALID_ARGUMENT;
  DeviceGuard guard(logits);
  if (guard.status() != RT_OK) return guard.status();
  const distill::Weights w = {1.f / temperature, ce_weight, z_weight, kd_weight, temperature};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float4* st = reinterpret_cast<float4*>(stats);
  float* tops = stats + 4 * rows;
  return distill::with_types(dtype, temperature, [&](auto* type, auto tm) {
    using T = std::remove_pointer_t<decltype(type)>;
    const T* z = static_cast<const T*>(logits);
    if (distill::warp_per_row(rows, (long long)vocab * (int)sizeof(T), false))
      return launch_pdl("distill_fwd_warp_kernel launch", distill::distill_fwd_warp_kernel<T, tm.value>,
                        dim3((unsigned)((rows + distill::kWarps - 1) / distill::kWarps)), dim3(distill::kThreads), 0,
                        s, z, rows, vocab, target, teacher_ids, teacher_logits, entries, w, loss, st, tops);
    const int split = distill::row_split(rows, vocab);
    return launch_pdl_cluster("distill_fwd_kernel launch", distill::distill_fwd_kernel<T, tm.value>,
                              dim3((unsigned)(rows * split)), dim3(distill::kRowThreads), split, s, z, rows, vocab,
                              target, teacher_ids, teacher_logits, entries, w, loss, st, tops);
  });
}

extern "C" int rt_distill_loss_bwd(const void* logits, int32_t dtype, int64_t rows, int32_t vocab,
                                   const int32_t* target, const int32_t* teacher_ids, const float* teacher_logits,
                                   int32_t entries, float temperature, float ce_weight, float z_weight,
                                   float kd_weight, const float* stats, const float* grad, void* dlogits,
                                   void* stream) {
  using namespace rt;
  if (!distill::valid(rows, vocab, dtype, entries, temperature, ce_weight, z_weight, kd_weight))
    return RT_ERR_INVALID_ARGUMENT;
  if (entries > distill::kMaxEntries) return RT_ERR_UNSUPPORTED;
  if (rows == 0) return RT_OK;
  if (!ok16(logits) || !ok16(stats) || !grad || !ok16(dlogits) || (entries > 0 && (!teacher_ids || !teacher_logits)))
    return RT_ERR_INVALID_ARGUMENT;
  DeviceGuard guard(logits);
  if (guard.status() != RT_OK) return guard.status();
  const distill::Weights w = {1.f / temperature, ce_weight, z_weight, kd_weight, temperature};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const float4* st = reinterpret_cast<const float4*>(stats);
  const float* tops = stats + 4 * rows;
  return distill::with_types(dtype, temperature, [&](auto* type, auto tm) {
    using T = std::remove_pointer_t<decltype(type)>;
    const T* z = static_cast<const T*>(logits);
    T* dz = static_cast<T*>(dlogits);
    if (distill::warp_per_row(rows, (long long)vocab * (int)sizeof(T), true))
      return launch_pdl("distill_bwd_warp_kernel launch", distill::distill_bwd_warp_kernel<T, tm.value>,
                        dim3((unsigned)((rows + distill::kWarps - 1) / distill::kWarps)), dim3(distill::kThreads), 0,
                        s, z, rows, vocab, target, teacher_ids, teacher_logits, entries, w, st, tops, grad, dz);
    // parts of kSpan steps, smaller ones while that leaves fewer blocks than run at once
    const int steps = vocab / (16 / (int)sizeof(T));  // at least as many as any row has
    int span = distill::kSpan;
    while (span > distill::kThreads && rows * ((steps + span - 1) / span) < 6 * 148) span /= 2;
    const long long parts = std::max(1, (steps + span - 1) / span);
    if (rows * parts > INT32_MAX) return (int)RT_ERR_INVALID_ARGUMENT;
    return launch_pdl("distill_bwd_kernel launch",
                      distill::distill_bwd_kernel<T, tm.value>, dim3((unsigned)(rows * parts)),
                      dim3(distill::kThreads), 0, s, z, rows, vocab, target, teacher_ids, teacher_logits, entries, w, st,
                      tops, grad, (int)parts, span, dz);
  });
}
