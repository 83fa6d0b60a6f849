// Losses over a vocabulary: distillation from a teacher's top logits, cross entropy with a label, or both, and the logits'
// gradient.  Per row, with z the logits, y the label, (id_k, t_k) the teacher's present entries, T the temperature and a the
// teacher's weight:
//
//   p = softmax over k of t_k / T,  q = softmax over the vocabulary of z / T,  s = softmax of z
//   loss = (1 - a) (log sum exp z - z_y) + a T^2 sum_k p_k (log p_k - log q[id_k])
//   dz_j = g [ (1 - a) (s_j - [j = y]) + a T (q_j - sum of p_k with id_k = j) ]
//
// A row without a label loses the first term, a row without present entries the second; with neither, or with all
// logits at -inf, the loss is 0 and the gradient zero.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "granule.cuh"

namespace tp {

constexpr int kMaxTop = 1024;

struct LossArgs {
  const void* logits;
  long long ld;
  int rows, V;
  const void* labels;            // null: none
  OuterIndex label_at;
  long long ignore;
  int labels64;
  const void* tid;               // teacher's ids and logits, null: none
  const void* tlog;
  OuterIndex tid_at, tlog_at;
  int top, tid64, tlog_dtype;
  float temperature, weight;     // weight = a
  float* loss;                   // [rows]
  float* stats;                  // [rows][4]: largest logit (0 where all are -inf), sum of exp(z - largest), of exp((z - largest) / T)
  void* dlogits;
  long long ldd;
  const float* grad_loss;        // [rows], stride ldg; null: 1
  long long ldg;
  float grad_scale;
  int* status;                   // word for waits that ran out
};

// dtype of the logits: what loss_<type>.cu instantiates.  mode: 1 loss and stats, 2 gradient from stats, 3 both.
int loss_launch_fp16(const LossArgs& a, int mode, cudaStream_t s);
int loss_launch_bf16(const LossArgs& a, int mode, cudaStream_t s);
int loss_launch_fp32(const LossArgs& a, int mode, cudaStream_t s);

enum { kLossFwd = 1, kLossBwd = 2 };   // bits of mode

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// Loads are kept as they come and looked at when they are needed: the first use of a value is what waits for it.
struct RawLabel {
  long long y;
  __device__ __forceinline__ void load(const LossArgs& a, int row) {
    if (a.labels) y = load_id(a.labels, a.label_at(row), a.labels64);
  }
  __device__ __forceinline__ int get(const LossArgs& a) const {      // -1: no term
    return !a.labels || a.weight == 1.0f || y == a.ignore || y < 0 || y >= a.V ? -1 : static_cast<int>(y);
  }
};
// Entry k of a row's teacher: its id or -1, and its logit (-inf where it is absent).
struct RawEntry {
  long long v;
  uint32_t bits;
  __device__ __forceinline__ void load(const LossArgs& a, int row, int k) {
    v = load_id(a.tid, a.tid_at(row) + k, a.tid64);
    const long long i = a.tlog_at(row) + k;
    bits = a.tlog_dtype == 2 ? static_cast<const uint32_t*>(a.tlog)[i] : static_cast<const uint16_t*>(a.tlog)[i];
  }
  __device__ __forceinline__ int id(const LossArgs& a) const { return v >= 0 && v < a.V ? static_cast<int>(v) : -1; }
  __device__ __forceinline__ float logit(const LossArgs& a) const {
    if (id(a) < 0) return -INFINITY;
    if (a.tlog_dtype == 2) return __uint_as_float(bits);
    if (a.tlog_dtype == 1) return __uint_as_float(bits << 16);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  }
};

// A row as 16-byte pieces of memory ("granules"): granule g holds elements [g N - lead, g N - lead + N), of which those
// outside [0, V) are not the row's.
template <typename T> struct RowPieces {
  static constexpr int N = Granule<T>::N;
  const T* row;
  int lead, V, count;
  __device__ __forceinline__ RowPieces(const T* r, int v) : row(r), V(v) {
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    count = V > 0 ? (lead + V + N - 1) / N : 0;      // (the address of an empty row may be anything)
  }
  __device__ __forceinline__ bool edge(int g) const { return (g == 0 && lead > 0) || (g + 1) * N > lead + V; }
  // An edge with -inf in the place of the elements that are not the row's: of a granule in hand, or reading the others only.
  __device__ uint4 mask_edge(const uint4& u, int g) const {
    float f[N];
    Granule<T>::unpack(u, f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = g * N - lead + j;
      if (i < 0 || i >= V) f[j] = -INFINITY;
    }
    return Granule<T>::pack(f);
  }
  __device__ uint4 load_edge(int g) const {
    float f[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = g * N - lead + j;
      f[j] = i >= 0 && i < V ? Elem<T>::to_f(row[i]) : -INFINITY;
    }
    return Granule<T>::pack(f);
  }
  __device__ __forceinline__ uint4 load(int g) const {
    return edge(g) ? load_edge(g) : __ldg(reinterpret_cast<const uint4*>(row - lead) + g);
  }
  // `wide`: a whole granule, and the written row lies on the same offset from a 16-byte boundary as the row read.
  __device__ __forceinline__ void store(T* out, int g, const float (&f)[N], bool wide) const {
    if (wide) {
      *reinterpret_cast<uint4*>(out + (g * N - lead)) = Granule<T>::pack(f);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = g * N - lead + j;
        if (i >= 0 && i < V) out[i] = Elem<T>::from_f(f[j]);
      }
    }
  }
};

// Largest values of granules, in pairs where they are 16-bit.  (A NaN is passed over; it comes back in the sums.)
template <typename T> struct GranuleMax {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  static __device__ __forceinline__ T2 pair(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
  T2 m;
  __device__ __forceinline__ GranuleMax() : m(pair(std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u)) {}
  __device__ __forceinline__ void add(const uint4& u) {
    m = __hmax2(m, __hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w))));
  }
  __device__ __forceinline__ float get() const { return fmaxf(Elem<T>::to_f(m.x), Elem<T>::to_f(m.y)); }
};
template <> struct GranuleMax<float> {
  float m = -INFINITY;
  __device__ __forceinline__ void add(const uint4& u) {
    m = max3(m, fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  __device__ __forceinline__ float get() const { return m; }
};

// Exponents (to base 2) of a CTA's exponentials, (z - shift) k.  The difference first: one multiply-add would do, but it rounds
// shift k, an error that a large offset of a row makes large, and the largest logit's exponential would not be 1.
struct Exponent {
  float k, shift;
  __device__ __forceinline__ float operator()(float z) const { return (z - shift) * k; }
  // What turns sums relative to a part's largest logit into sums relative to this shift.  (A part without any has sums of zero,
  // or of NaN, and keeps them.)
  __device__ __forceinline__ float factor(float part_m) const {
    return part_m == -INFINITY ? 1.0f : exp2_approx((part_m - shift) * k);
  }
};
template <typename T>
__device__ __forceinline__ void granule_exp(const uint4& u, const Exponent& x, float (&e)[Granule<T>::N]) {
  float f[Granule<T>::N];
  Granule<T>::unpack(u, f);
#pragma unroll
  for (int j = 0; j < Granule<T>::N; j += 2) {
    const float2 d = mul2(add2(make_float2(f[j], f[j + 1]), dup2(-x.shift)), dup2(x.k));
    e[j] = exp2_approx(d.x);
    e[j + 1] = exp2_approx(d.y);
  }
}
template <int N> __device__ __forceinline__ float sum_of(const float (&e)[N]) {
  float2 s = make_float2(e[0], e[1]);
#pragma unroll
  for (int j = 2; j < N; j += 2) s = add2(s, make_float2(e[j], e[j + 1]));
  return s.x + s.y;
}

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
template <int LANES = 32> __device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum of the WARPS (at most 16) numbers at v, in every lane.
template <int WARPS> __device__ __forceinline__ float add_up(const float* v) {
  const int lane = threadIdx.x & 31;
  return warp_add<16>((lane & 15) < WARPS ? v[lane & 15] : 0.0f);
}

// Factors of a row's gradient: dz_j = c1 e1_j + ct et_j - [j = y] g1 - gt P_j.
struct RowFactors {
  float g1, gt;
  // g: the row's factor
  __device__ __forceinline__ RowFactors(const LossArgs& a, float g, bool label, bool teach) {
    g *= a.grad_scale;
    g1 = label ? g * (1.0f - a.weight) : 0.0f;
    gt = teach ? g * a.weight * a.temperature : 0.0f;
  }
};

// What a CTA knows of its part of a row; the parts of a cluster are joined in every CTA.
struct alignas(16) PartOfRow {
  float m, s1, st;      // largest logit; sums of exponentials relative to it (to 0 where it is -inf)
  float dot, mass;      // over the entries in this part, not yet divided by the sum over all entries: p (z - m), p
  float zy, own, pad;   // z_y - m and 1 where the label is in this part
};
struct WholeRow {
  float m, s1, st, dot, zy;
};

// Lanes 0 .. parts - 1 hold a part each (parts <= 8).  k1, kt: the exponents' factors of s1 and st.
template <bool DUAL> __device__ __forceinline__ WholeRow join_parts(const PartOfRow& p, int parts, float k1, float kt, bool teacher) {
  const bool in = (threadIdx.x & 31) < parts, some = in && p.m != -INFINITY;
  float m = warp_max(in ? p.m : -INFINITY);
  if (m == -INFINITY) m = 0.0f;
  const float d = (some ? p.m : 0.0f) - m;
  auto all = [&](float v) { return __shfl_sync(0xffffffffu, warp_add<8>(in ? v : 0.0f), 0); };
  WholeRow w{m, all(p.s1 * Exponent{k1, m}.factor(p.m)), 0.0f, 0.0f, all(p.zy + p.own * d)};
  w.st = DUAL ? all(p.st * Exponent{kt, m}.factor(p.m)) : w.s1;
  if (teacher) w.dot = all(p.dot + p.mass * d);
  return w;
}
__device__ __forceinline__ PartOfRow load_part(uint32_t cluster_addr) {
  PartOfRow p;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(p.m), "=f"(p.s1), "=f"(p.st), "=f"(p.dot) : "r"(cluster_addr) : "memory");
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(p.mass), "=f"(p.zy), "=f"(p.own), "=f"(p.pad) : "r"(cluster_addr + 16) : "memory");
  return p;
}
// Stores a part into another CTA's shared memory; its bytes count on that CTA's barrier.  (A cluster barrier would do as
// well, but its release waits for all of the CTA's stores to global memory, a row's gradient each time.)
__device__ __forceinline__ void send_part(const PartOfRow& p, uint32_t cluster_addr, uint32_t cluster_bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(cluster_addr), "f"(p.m), "f"(p.s1), "f"(p.st), "f"(p.dot), "r"(cluster_bar) : "memory");
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(cluster_addr + 16), "f"(p.mass), "f"(p.zy), "f"(p.own), "f"(p.pad), "r"(cluster_bar) : "memory");
}

// t_sum: sum of exp((t - t_max) / T) over the entries; entropy: the same weighted with (t - t_max) / T.
__device__ __forceinline__ void store_loss(const LossArgs& a, int row, const WholeRow& w, bool label, bool teach, float t_sum,
                                           float entropy) {
  float loss = 0.0f;
  if (w.s1 != 0.0f) {
    if (label) loss = (1.0f - a.weight) * (__logf(w.s1) - w.zy);
    if (teach)
      loss += a.weight * a.temperature * a.temperature *
              ((entropy - w.dot / a.temperature) / t_sum - __logf(t_sum) + __logf(w.st));
  }
  a.loss[row] = loss;
  if (a.stats) *reinterpret_cast<float4*>(a.stats + 4ll * row) = make_float4(w.m, w.s1, w.st, 0.0f);
}

// The gradient's element of entry k, by the first of the entries with its id.  e1, et: exponentials of its logit, g1: the label's
// factor, gp: the teacher's over the sum of its exponentials, `look`: the id may occur more than once.
template <typename T, bool DUAL>
__device__ __forceinline__ void store_entry(T* out, int id, int k, float e1, float et, const int* top_id, const float* top_p, int top,
                                            bool look, float c1, float ct, float g1, float gp, int label) {
  float p = top_p[k];
  if (look) {
    p = 0.0f;
    for (int o = 0; o < top; ++o) {
      if (top_id[o] != id) continue;
      if (o < k) return;
      p += top_p[o];
    }
  }
  if (id != label) g1 = 0.0f;
  // (with DUAL each difference by itself: exactly zero where both distributions have one value only)
  out[id] = Elem<T>::from_f(DUAL ? (c1 * e1 - g1) + (ct * et - gp * p) : c1 * e1 - (g1 + gp * p));
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// ------------------------------------------------------------------ rows held on chip
// Logits are read once and, with WRITE, their gradient is written: what bounds the kernel is those bytes.  A row belongs to a
// cluster of 1 to 8 CTAs of THREADS threads, NG granules a thread.  The next row travels into shared memory (cp.async, slots that
// only their thread reads) while this one is worked on; its exponentials, relative to the thread's own largest logit, stay in
// registers in fp32 until the row's sum is known, so each is computed once: two a logit and softmax would
// keep the exponential unit (16 a cycle and SM) busy three quarters of the time that the bytes take, and two softmaxes of
// different temperature (DUAL) longer than that.  Without DUAL there is one exponential a logit: the temperature
// is 1 or one of the two terms has no weight.
//
// Warps do not meet at barriers for the sums: each sends its own to every CTA of the cluster (st.async, counted by an mbarrier)
// and adds up all of them, so that fast warps run ahead into the next row.
//
// The teacher's entries: thread k of every CTA has entry k, and stores its element of the gradient again after the row's where
// it lies in the CTA's part.  A small hash table of their ids tells whether one occurs twice: only then are all entries
// looked through for their sum.

// CTAs an SM has registers for, by the exponentials a thread keeps.
constexpr int loss_ctas_per_sm(int threads, int values) { return (values > 32 ? 512 : values > 16 ? 768 : 1024) / threads; }

// What a warp knows of its part of a row.
struct alignas(16) WarpPart {
  float m, s1;            // largest logit; sum of exponentials relative to it (to 0 where it is -inf)
  float zy, own;          // z_y - m and 1 where the label is in the warp's part
  float t_max, t_sum;     // over the warp's entries: largest t, sum of exp((t - t_max) / T)
  float entropy, st;      // the same weighted with (t - t_max) / T; the second softmax's sum
  float dot, mass;        // over its entries in this CTA's part, as t_sum: p (z - m), p
  float pad[2];
};
// Stores a part into a CTA's shared memory; its bytes count on that CTA's barrier.  (A cluster barrier would do as
// well, but its release waits for all of the CTA's stores to global memory, a row's gradient each time.)
__device__ __forceinline__ void send16(uint32_t cluster_addr, uint32_t cluster_bar, float a, float b, float c, float d) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(cluster_addr), "f"(a), "f"(b), "f"(c), "f"(d), "r"(cluster_bar) : "memory");
}

constexpr int loss_table_size(int top) {      // slots of the hash table: a power of two, at least twice the entries
  int n = 64;
  while (n < 2 * top) n *= 2;
  return n;
}

template <typename T, bool DUAL, int THREADS, int NG, bool WRITE>
__global__ void __launch_bounds__(THREADS, loss_ctas_per_sm(THREADS, (WRITE ? NG : 1) * Granule<T>::N * (DUAL ? 2 : 1)))
loss_rows_kernel(const LossArgs a, int parts, int per, int table) {
  constexpr int N = Granule<T>::N, kWarps = THREADS / 32, kSlots = THREADS * NG, kKept = WRITE ? NG : 1, kMaxParts = 8;
  extern __shared__ __align__(16) uint4 loss_smem[];
  uint4* raw = loss_smem;                                      // [2][kSlots]
  float* top_p = reinterpret_cast<float*>(raw + 2 * kSlots);   // [top] exp((t - its warp's t_max) / T), then relative to the row's
  float* top_z = top_p + a.top;                                // [top] z
  int* top_id = reinterpret_cast<int*>(top_z + a.top);         // [top]
  int* ids = top_id + a.top;                                   // [2][table] hash tables of id + 1
  __shared__ WarpPart inbox[2][kMaxParts * kWarps];
  __shared__ uint64_t arrived[2];      // all parts of a row are in inbox[.]
  __shared__ int twice[2], abort_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = parts > 1 ? cluster_ctarank() : 0;
  const int stride = gridDim.x / parts, g0 = rank * per, warps = parts * kWarps;
  const float inv_t = 1.0f / a.temperature, kt = inv_t * kLog2e;
  // the one exponential's exponent without DUAL: z, or with a teacher alone z / T
  const float k1 = DUAL || a.weight == 0.0f ? kLog2e : kt;
  const T* z0 = static_cast<const T*>(a.logits);
  const bool teacher = a.top > 0, full = DUAL || teacher;      // full: all of a WarpPart travels, else its first 16 bytes
  const WaitCtx wait{&abort_word, a.status};
  if (tid == 0) {
    abort_word = 0;
    twice[0] = twice[1] = 0;
    // (a launch without clusters has no st.async: its warps store their parts and arrive)
    mbar_init(&arrived[0], parts > 1 ? 1 : kWarps);
    mbar_init(&arrived[1], parts > 1 ? 1 : kWarps);
    fence_barrier_init();
  }
  for (int i = tid; i < 2 * table; i += THREADS) ids[i] = 0;
  if (parts > 1) cluster_sync_all();
  else __syncthreads();
  pdl_wait();

  const uint32_t raw_addr = smem_u32(raw + tid);
  // Granules k < kFull are there for every thread, and none of them is a row's last (see loss_rows_fit): a test for each
  // granule costs half as much as the work on it.
  constexpr int kFull = NG > 2 ? NG - 2 : 0;
  auto prefetch = [&](const T* z, int buf) {
    const RowPieces<T> r(z, a.V);
    const int cnt = min(r.count - g0, per);
    const T* src = z + ((g0 + tid) * N - r.lead);
    const uint32_t dst = raw_addr + buf * (kSlots * 16);
    const int left = (r.lead + r.V - (g0 + tid) * N) * static_cast<int>(sizeof(T));
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      // (the first granule may begin in the row before, but not before the matrix)
      if (k == 0 ? tid < cnt && src >= z0 : k < kFull || tid + k * THREADS < cnt)
        cp_async_16(dst + k * THREADS * 16, src + k * THREADS * N, k < kFull ? 16 : min(left - k * THREADS * 16, 16));
    }
  };

  int row = blockIdx.x / parts, buf = 0, turn = 0;
  const T* z = z0 + row * a.ld;
  T* out = static_cast<T*>(a.dlogits) + row * a.ldd;
  const long long z_step = stride * a.ld, out_step = stride * a.ldd;
  RawLabel label_next{};
  RawEntry entry_next{-1, 0};
  float g_next = 1.0f;
  if (row < a.rows) {
    prefetch(z, 0);
    label_next.load(a, row);
    if (tid < a.top) entry_next.load(a, row, tid);
    if (WRITE && a.grad_loss) g_next = a.grad_loss[row * a.ldg];
  }
  cp_async_commit();
  for (; row < a.rows; row += stride, z += z_step, out += out_step, buf ^= 1, turn += buf == 0) {
    const int label = label_next.get(a);
    const RawEntry entry = entry_next;
    const float g = g_next;
    if (row + stride < a.rows) {
      prefetch(z + z_step, buf ^ 1);
      label_next.load(a, row + stride);
      if (tid < a.top) entry_next.load(a, row + stride, tid);
      if (WRITE && a.grad_loss) g_next = a.grad_loss[(row + stride) * a.ldg];
    }
    cp_async_commit();
    const RowPieces<T> r(z, a.V);
    uint4* mine = raw + buf * kSlots + tid;
    const int cnt = min(r.count - g0, per);
    auto place = [&](int id) {      // number in this part of an element's granule, -1 in another part
      const int gl = static_cast<int>(static_cast<unsigned>(id + r.lead) / N) - g0;
      return id >= 0 && gl >= 0 && gl < per ? gl : -1;
    };
    // entry tid's logit is on its way while the row is worked on
    float z_entry = 0.0f;
    if (tid < a.top && place(entry.id(a)) >= 0) z_entry = Elem<T>::to_f(z[entry.id(a)]);
    cp_async_wait<1>();
    // the row's first and last granule, where others' elements lie in them: numbers in this part, or -1
    const int first = g0 == 0 && r.lead > 0 && cnt > 0 ? 0 : -1;
    const int last = (r.lead + r.V) % N != 0 && r.count - 1 - g0 < cnt ? r.count - 1 - g0 : -1;
    const bool owns_first = first == 0 && tid == 0, owns_last = last >= 0 && last != first && tid == (last & (THREADS - 1));
    if (owns_first) mine[0] = z - r.lead >= z0 ? r.mask_edge(mine[0], 0) : r.load_edge(0);
    if (owns_last) mine[last - tid] = r.mask_edge(mine[last - tid], g0 + last);
    // ---- the thread's largest logit and exponentials
    GranuleMax<T> largest;
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (k < kFull || tid + k * THREADS < cnt) largest.add(mine[k * THREADS]);
    const float m_own = largest.get(), shift = m_own == -INFINITY ? 0.0f : m_own;
    const Exponent x1{k1, shift}, xt{kt, shift};
    float e1[kKept][N], et[DUAL ? kKept : 1][N], s1 = 0.0f, st = 0.0f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int kept = WRITE ? k : 0;
      if (k >= kFull && tid + k * THREADS >= cnt) continue;
      const uint4 u = mine[k * THREADS];
      granule_exp<T>(u, x1, e1[kept]);
      s1 += sum_of<N>(e1[kept]);
      if (DUAL) {
        granule_exp<T>(u, xt, et[kept]);
        st += sum_of<N>(et[kept]);
      }
    }
    // ---- the warp's
    const float m_warp = warp_max(m_own), m_from = m_warp == -INFINITY ? 0.0f : m_warp;
    s1 = warp_add(s1 * Exponent{k1, m_from}.factor(m_own));
    if (DUAL) st = warp_add(st * Exponent{kt, m_from}.factor(m_own));
    const int label_gl = place(label);
    const bool owner = label_gl >= 0 && tid == (label_gl & (THREADS - 1));      // of the label's granule
    float zy = 0.0f;
    if (owner) zy = Elem<T>::to_f(reinterpret_cast<const T*>(mine + (label_gl - tid))[static_cast<unsigned>(label + r.lead) % N]);
    const unsigned label_lane = __ballot_sync(0xffffffffu, owner);
    const float zy_warp = __shfl_sync(0xffffffffu, zy, label_lane ? __ffs(label_lane) - 1 : 0);
    float t_max = -INFINITY, t_sum = 0.0f, entropy = 0.0f, dot = 0.0f, mass = 0.0f;
    if (teacher) {
      for (int k = tid; k < a.top; k += THREADS) {
        RawEntry e = entry;
        float v = z_entry;
        if (k >= THREADS) {
          e.load(a, row, k);
          v = place(e.id(a)) >= 0 ? Elem<T>::to_f(z[e.id(a)]) : 0.0f;
        }
        const int id = e.id(a);
        top_id[k] = id;
        top_p[k] = e.logit(a);
        top_z[k] = v;
        t_max = fmaxf(t_max, top_p[k]);
        if (WRITE && place(id) >= 0) {
          int slot = (id * 0x9e3779b1u) >> 20 & (table - 1);
          while (true) {      // (at most half of the slots are ever taken)
            const int was = atomicCAS(&ids[buf * table + slot], 0, id + 1);
            if (was == 0) break;
            if (was == id + 1) {
              twice[buf] = 1;
              break;
            }
            slot = (slot + 1) & (table - 1);
          }
        }
      }
      t_max = warp_max(t_max);
      const float t_from = t_max == -INFINITY ? 0.0f : t_max;
      for (int k = tid; k < a.top; k += THREADS) {
        const float lt = (top_p[k] - t_from) * inv_t, p = top_id[k] >= 0 ? exp2_approx(lt * kLog2e) : 0.0f;
        top_p[k] = p;
        t_sum += p;
        if (p == 0.0f) continue;
        entropy += p * lt;
        if (place(top_id[k]) < 0) continue;
        dot += p * (top_z[k] - m_from);
        mass += p;
      }
      t_sum = warp_add(t_sum);
      entropy = warp_add(entropy);
      dot = warp_add(dot);
      mass = warp_add(mass);
    }
    // ---- to all CTAs of the cluster, and all of it back
    zy = label_lane ? zy_warp - m_from : 0.0f;
    const float own = label_lane ? 1.0f : 0.0f;
    if (parts > 1) {
      if (tid == 0) mbar_expect_tx(&arrived[buf], warps * (full ? 48 : 16));
      if (lane < parts) {
        const uint32_t to = mapa_u32(smem_u32(&inbox[buf][rank * kWarps + warp]), lane), bar = mapa_u32(smem_u32(&arrived[buf]), lane);
        send16(to, bar, m_warp, s1, zy, own);
        if (full) {
          send16(to + 16, bar, t_max, t_sum, entropy, st);
          send16(to + 32, bar, dot, mass, 0.0f, 0.0f);
        }
      }
    } else if (lane == 0) {
      inbox[buf][warp] = WarpPart{m_warp, s1, zy, own, t_max, t_sum, entropy, st, dot, mass, {0.0f, 0.0f}};
      mbar_arrive(&arrived[buf]);
    }
    bool ok = mbar_wait(&arrived[buf], turn & 1, wait, kErrWaitPeer);
    float m = -INFINITY;
    for (int i = lane; i < warps; i += 32) m = fmaxf(m, inbox[buf][i].m);
    m = warp_max(m);
    if (m == -INFINITY) m = 0.0f;
    s1 = st = 0.0f;
    for (int i = lane; i < warps; i += 32) {
      s1 += inbox[buf][i].s1 * Exponent{k1, m}.factor(inbox[buf][i].m);
      if (DUAL) st += inbox[buf][i].st * Exponent{kt, m}.factor(inbox[buf][i].m);
    }
    s1 = warp_add(s1);
    st = DUAL ? warp_add(st) : s1;
    const float my_t = t_max;
    if (teacher) {      // (every CTA has all entries: its own warps' sums are enough)
      const WarpPart& p = inbox[buf][rank * kWarps + (lane & (kWarps - 1))];
      t_max = warp_max(p.t_max);
      if (t_max == -INFINITY) t_max = 0.0f;
      t_sum = warp_add<kWarps>(p.t_max == -INFINITY ? 0.0f : p.t_sum * exp2_approx((p.t_max - t_max) * kt));
    }
    const bool teach = a.weight != 0.0f && t_sum != 0.0f, zero = !(teach || label >= 0) || s1 == 0.0f;
    if (rank == 0 && warp == 0) {
      zy = entropy = dot = 0.0f;
      for (int i = lane; i < warps; i += 32) {
        const WarpPart& p = inbox[buf][i];
        const float from = p.m == -INFINITY ? 0.0f : p.m;
        zy += p.zy + p.own * (from - m);
        if (teacher && p.t_max != -INFINITY) {
          const float ft = (p.t_max - t_max) * inv_t, scale = exp2_approx(ft * kLog2e);
          if (scale != 0.0f) {
            dot += scale * (p.dot + p.mass * (from - m));
            if (i < kWarps) entropy += scale * (p.entropy + p.t_sum * ft);
          }
        }
      }
      zy = warp_add(zy);
      if (teacher) {
        dot = warp_add(dot);
        entropy = warp_add(entropy);
      }
      if (lane == 0) store_loss(a, row, WholeRow{m, s1, st, dot, zy}, label >= 0, teach, t_sum, entropy);
    }
    if (WRITE) {
      // ---- the gradient
      const RowFactors f(a, g, label >= 0, teach);
      const float c1 = (DUAL ? f.g1 : f.g1 + f.gt) * (1.0f / s1) * Exponent{k1, m}.factor(m_own);
      const float ct = DUAL ? f.gt * (1.0f / st) * Exponent{kt, m}.factor(m_own) : 0.0f;
      const bool wide = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(z)) & 15) == 0;
      if (!ok) {
        // (nothing is known of the row)
      } else if (zero) {
        const float o[N] = {};
        for (int gl = tid; gl < cnt; gl += THREADS) r.store(out, g0 + gl, o, wide && gl != first && gl != last);
      } else {
        auto value = [&](float v1, float vt) { return DUAL ? fmaf(ct, vt, c1 * v1) : c1 * v1; };
        if (wide) {
          uint4* o = reinterpret_cast<uint4*>(out + ((g0 + tid) * N - r.lead));
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const int gl = tid + k * THREADS;
            if ((k >= kFull && (gl >= cnt || gl == last)) || (k == 0 && gl == first)) continue;
            float v[N];
#pragma unroll
            for (int j = 0; j < N; j += 2) {
              float2 d = mul2(make_float2(e1[k][j], e1[k][j + 1]), dup2(c1));
              if (DUAL) d = fma2(make_float2(et[k][j], et[k][j + 1]), dup2(ct), d);
              v[j] = d.x;
              v[j + 1] = d.y;
            }
            o[k * THREADS] = Granule<T>::pack(v);
          }
        } else {
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const int gl = tid + k * THREADS;
            if (gl >= cnt || gl == first || gl == last) continue;
#pragma unroll
            for (int j = 0; j < N; ++j)
              out[(g0 + gl) * N - r.lead + j] = Elem<T>::from_f(value(e1[k][j], DUAL ? et[k][j] : 0.0f));
          }
        }
        if (owns_first || owns_last) {
          for (int which = owns_first ? 0 : 1; which < (owns_last ? 2 : 1); ++which) {
            const uint4 u = which ? mine[last - tid] : mine[0];
            float v1[N], vt[N] = {};
            granule_exp<T>(u, x1, v1);
            if (DUAL) granule_exp<T>(u, xt, vt);
#pragma unroll
            for (int j = 0; j < N; ++j) v1[j] = value(v1[j], vt[j]);
            r.store(out, which ? g0 + last : 0, v1, false);
          }
        }
        if (owner) {      // over what this thread has just stored
          const float v = Elem<T>::to_f(reinterpret_cast<const T*>(mine + (label_gl - tid))[static_cast<unsigned>(label + r.lead) % N]);
          out[label] = Elem<T>::from_f((c1 * exp2_approx(x1(v)) - f.g1) + (DUAL ? ct * exp2_approx(xt(v)) : 0.0f));
        }
      }
      if (teacher) {
        const float scale = my_t == -INFINITY ? 0.0f : exp2_approx((my_t - t_max) * kt);
        for (int k = tid; k < a.top; k += THREADS) top_p[k] *= scale;
        ok = __syncthreads_and(ok);      // the row's stores come before the entries', and the table is complete
        const bool look = twice[buf];
        if (ok && teach && !zero) {
          const Exponent y1{k1, m}, yt{kt, m};
          const float r1 = (DUAL ? f.g1 : f.g1 + f.gt) * (1.0f / s1), rt = DUAL ? f.gt * (1.0f / st) : 0.0f;
          for (int k = tid; k < a.top; k += THREADS) {
            if (place(top_id[k]) >= 0)
              store_entry<T, DUAL>(out, top_id[k], k, exp2_approx(y1(top_z[k])), DUAL ? exp2_approx(yt(top_z[k])) : 0.0f, top_id, top_p,
                                   a.top, look, r1, rt, f.g1, f.gt / t_sum, label);
          }
        }
        if (look) {
          __syncthreads();      // others' entries are still read
          if (tid == 0) twice[buf] = 0;
        }
        // the table of the row after next
        for (int i = tid; i < table; i += THREADS) ids[buf * table + i] = 0;
      }
    }
    if (!ok) break;
  }
  cp_async_wait<0>();
  if (parts > 1) cluster_sync_all();      // nobody leaves while parts may still be sent to it
}

// ------------------------------------------------------------------ rows read twice
// The gradient from a forward pass's statistics (MODE 2), and rows that a cluster cannot hold (1 and 3: the second read is
// served by L2 where it can).  A CTA per part of a row; the parts of a row form a cluster where their sums have to be joined.
template <typename T, bool DUAL, int MODE>
__global__ void __launch_bounds__(512, 2)
loss_stream_kernel(const LossArgs a, int parts, int per) {
  constexpr int N = Granule<T>::N, kWarps = 16, kThreads = 512, kAhead = 4;
  extern __shared__ __align__(16) uint4 loss_smem[];
  float* top_p = reinterpret_cast<float*>(loss_smem);
  float* top_z = top_p + a.top;
  int* top_id = reinterpret_cast<int*>(top_z + a.top);
  __shared__ float red_max[2][kWarps], red_sum[6][kWarps];
  __shared__ PartOfRow part;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % parts, row = blockIdx.x / parts;
  const float inv_t = 1.0f / a.temperature, kt = inv_t * kLog2e;
  const float k1 = DUAL || a.weight == 0.0f ? kLog2e : kt;
  const bool teacher = a.top > 0;
  pdl_wait();
  const RowPieces<T> r(static_cast<const T*>(a.logits) + row * a.ld, a.V);
  const int g0 = static_cast<int>(min(static_cast<long long>(rank) * per, static_cast<long long>(r.count)));
  const int g1 = static_cast<int>(min(static_cast<long long>(g0) + per, static_cast<long long>(r.count)));
  auto in_part = [&](int id) {
    const int g = static_cast<int>((static_cast<long long>(id) + r.lead) / N);
    return id >= 0 && g >= g0 && g < g1;
  };
  RawLabel raw_label{};
  raw_label.load(a, row);
  const int label = raw_label.get(a);
  const bool own = label >= 0 && in_part(label);
  const float zy = own ? Elem<T>::to_f(r.row[label]) : 0.0f;
  float t_max = -INFINITY, m = -INFINITY, s1 = 0.0f, st = 0.0f;
  for (int k = tid; k < a.top; k += kThreads) {
    RawEntry e;
    e.load(a, row, k);
    const int id = e.id(a);
    const float t = e.logit(a);
    top_id[k] = id;
    top_p[k] = t;
    top_z[k] = in_part(id) ? Elem<T>::to_f(r.row[id]) : 0.0f;
    t_max = fmaxf(t_max, t);
  }
  if (MODE & kLossFwd) {
    for (int g = g0 + tid; g < g1; g += kThreads * kAhead) {
      uint4 u[kAhead];
      GranuleMax<T> largest;
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (g + k * kThreads < g1) u[k] = r.load(g + k * kThreads);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (g + k * kThreads < g1) largest.add(u[k]);
      const float top = largest.get();
      if (top > m) {
        s1 *= Exponent{k1, top}.factor(m);
        if (DUAL) st *= Exponent{kt, top}.factor(m);
        m = top;
      }
      const float shift = m == -INFINITY ? 0.0f : m;
      const Exponent x1{k1, shift}, xt{kt, shift};
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (g + k * kThreads >= g1) continue;
        float e[N];
        granule_exp<T>(u[k], x1, e);
        s1 += sum_of<N>(e);
        if (DUAL) {
          granule_exp<T>(u[k], xt, e);
          st += sum_of<N>(e);
        }
      }
    }
  }
  const float m_mine = m;
  m = warp_max(m);
  t_max = warp_max(t_max);
  if (lane == 0) {
    red_max[0][warp] = m;
    red_max[1][warp] = t_max;
  }
  __syncthreads();
  m = warp_max(red_max[0][lane % kWarps]);
  t_max = warp_max(red_max[1][lane % kWarps]);
  if (t_max == -INFINITY) t_max = 0.0f;
  const float shift = m == -INFINITY ? 0.0f : m;
  if (MODE & kLossFwd) {
    s1 *= Exponent{k1, shift}.factor(m_mine);
    if (DUAL) st *= Exponent{kt, shift}.factor(m_mine);
  }
  float t_part = 0.0f, entropy = 0.0f, dot = 0.0f, mass = 0.0f;
  for (int k = tid; k < a.top; k += kThreads) {
    const int id = top_id[k];
    const float lt = (top_p[k] - t_max) * inv_t, p = id >= 0 ? exp2_approx(lt * kLog2e) : 0.0f;
    top_p[k] = p;
    t_part += p;
    if (p == 0.0f) continue;
    entropy += p * lt;
    if (!in_part(id)) continue;
    dot += p * (top_z[k] - shift);
    mass += p;
  }
  if (MODE & kLossFwd) {
    s1 = warp_add(s1);
    if (DUAL) st = warp_add(st);
  }
  if (teacher) {
    t_part = warp_add(t_part);
    entropy = warp_add(entropy);
    dot = warp_add(dot);
    mass = warp_add(mass);
  }
  if (lane == 0) {
    red_sum[0][warp] = s1;
    red_sum[1][warp] = st;
    red_sum[2][warp] = t_part;
    red_sum[3][warp] = entropy;
    red_sum[4][warp] = dot;
    red_sum[5][warp] = mass;
  }
  __syncthreads();      // (and every entry's logit has been read before the row is written)
  const float t_sum = teacher ? add_up<kWarps>(red_sum[2]) : 0.0f;
  const bool teach = a.weight != 0.0f && t_sum != 0.0f;
  WholeRow w;
  if (MODE & kLossFwd) {
    PartOfRow p{m, add_up<kWarps>(red_sum[0]), DUAL ? add_up<kWarps>(red_sum[1]) : 0.0f, add_up<kWarps>(red_sum[4]),
                add_up<kWarps>(red_sum[5]), own ? zy - shift : 0.0f, own ? 1.0f : 0.0f, 0};
    if (parts > 1) {
      if (tid == 0) part = p;
      cluster_sync_all();
      if (lane < parts) p = load_part(mapa_u32(smem_u32(&part), lane));
      w = join_parts<DUAL>(p, parts, k1, kt, teacher);
    } else {
      w = WholeRow{shift, p.s1, DUAL ? p.st : p.s1, p.dot, p.zy};
    }
    entropy = add_up<kWarps>(red_sum[3]);
    if (rank == 0 && tid == 0) store_loss(a, row, w, label >= 0, teach, t_sum, entropy);
    if (parts > 1) cluster_sync_all();      // nobody leaves while its part may still be read
  } else {
    const float4 v = *reinterpret_cast<const float4*>(a.stats + 4ll * row);
    w = WholeRow{v.x, v.y, v.z, 0.0f, 0.0f};
  }
  if (!(MODE & kLossBwd)) return;
  const bool zero = !(teach || label >= 0) || w.s1 == 0.0f;
  const RowFactors f(a, a.grad_loss ? a.grad_loss[row * a.ldg] : 1.0f, label >= 0, teach);
  const Exponent x1{k1, w.m}, xt{kt, w.m};
  const float c1 = (DUAL ? f.g1 : f.g1 + f.gt) * (1.0f / w.s1), ct = DUAL ? f.gt * (1.0f / w.st) : 0.0f;
  T* out = static_cast<T*>(a.dlogits) + row * a.ldd;
  const bool wide = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(r.row)) & 15) == 0;
  for (int g = g0 + tid; g < g1; g += kThreads * kAhead) {
    uint4 u[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (g + k * kThreads < g1 && !zero) u[k] = r.load(g + k * kThreads);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (g + k * kThreads >= g1) continue;
      float e[N] = {}, o[N] = {};
      if (!zero) {
        granule_exp<T>(u[k], x1, e);
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = c1 * e[j];
        if (DUAL) {
          granule_exp<T>(u[k], xt, e);
#pragma unroll
          for (int j = 0; j < N; ++j) o[j] += ct * e[j];
        }
      }
      r.store(out, g + k * kThreads, o, wide && !r.edge(g + k * kThreads));
    }
  }
  __syncthreads();      // the label's and the entries' elements come after the row's
  if (zero) return;
  if (tid == 0 && own)
    out[label] = Elem<T>::from_f((c1 * exp2_approx(x1(zy)) - f.g1) + (DUAL ? ct * exp2_approx(xt(zy)) : 0.0f));
  if (!teach) return;
  __syncthreads();
  for (int k = tid; k < a.top; k += kThreads)
    if (in_part(top_id[k]))
      store_entry<T, DUAL>(out, top_id[k], k, exp2_approx(x1(top_z[k])), DUAL ? exp2_approx(xt(top_z[k])) : 0.0f, top_id, top_p, a.top,
                           true, c1, ct, f.g1, f.gt / t_sum, label);
}

// ------------------------------------------------------------------ launches
// What a kernel needs to be told or asked once per device: leave to use its shared memory, clusters of 1, 2, 4 and 8 that run at once.
struct LossDevice {
  int clusters[4];
  bool ready;
};

template <typename T, bool DUAL, int THREADS, int NG, bool WRITE>
static int loss_rows_launch(const LossArgs& a, int parts, int per, cudaStream_t s) {
  auto kern = loss_rows_kernel<T, DUAL, THREADS, NG, WRITE>;
  constexpr size_t kRaw = 2ull * THREADS * NG * 16, kSmem = kRaw + kMaxTop * 12 + 2 * loss_table_size(kMaxTop) * 4;
  static LossDevice known[16];
  int dev = 0;
  cudaGetDevice(&dev);
  LossDevice& d = known[dev & 15];
  if (!d.ready) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem)) != cudaSuccess) return kErrLaunch;
    for (int i = 0; i < 4; ++i) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      cfg.gridDim = dim3(1u << i);
      cfg.blockDim = dim3(THREADS);
      cfg.dynamicSmemBytes = kSmem;
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << i;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&d.clusters[i], kern, &cfg) != cudaSuccess || d.clusters[i] < 1) return kErrLaunch;
    }
    d.ready = true;
  }
  // As many clusters as run at once, each walking over rows: more would only begin when the first have ended (74 clusters of 4
  // where 71 fit, for instance, doubled the time).
  const int most = d.clusters[parts == 1 ? 0 : parts == 2 ? 1 : parts == 4 ? 2 : 3];
  const int grid = (a.rows < most ? a.rows : most) * parts;
  const int table = WRITE && a.top > 0 ? loss_table_size(a.top) : 0;
  launch_pdl(kern, dim3(grid), dim3(THREADS), kRaw + static_cast<size_t>(a.top) * 12 + 2ull * table * 4, s, parts, a, parts, per, table);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

template <typename T, bool DUAL, int MODE> static int loss_stream_launch(const LossArgs& a, int parts, int per, cudaStream_t s) {
  const long long grid = static_cast<long long>(a.rows) * parts;
  if (grid > 0x7fffffffll) return kErrTooLarge;
  launch_pdl(loss_stream_kernel<T, DUAL, MODE>, dim3(static_cast<unsigned>(grid)), dim3(512), static_cast<size_t>(a.top) * 12, s,
             MODE & kLossFwd ? parts : 1, a, parts, per);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

// The kernel for `per` granules a part at THREADS threads: the parts of a row differ by at most 8 granules (its last part, and the
// granule more that an offset from a 16-byte boundary needs), so that all but the last two granules a thread are full.
template <typename T, bool DUAL, int THREADS, int NG, bool WRITE>
static int loss_rows_fit(const LossArgs& a, int parts, int per, cudaStream_t s) {
  if constexpr (NG > 1) {
    if (per <= THREADS * (NG - 1)) return loss_rows_fit<T, DUAL, THREADS, NG - 1, WRITE>(a, parts, per, s);
  }
  return loss_rows_launch<T, DUAL, THREADS, NG, WRITE>(a, parts, per, s);
}

template <typename T, bool DUAL, bool WRITE> static int loss_choose(const LossArgs& a, cudaStream_t s) {
  constexpr int N = Granule<T>::N, kMost = DUAL ? 4 : 8;      // granules a thread: registers for their exponentials
  // granules of the longest row: rows on different offsets from a 16-byte boundary may need one more
  const bool same = a.rows == 1 || a.ld * static_cast<long long>(sizeof(T)) % 16 == 0;
  const long long lead = same ? (reinterpret_cast<uintptr_t>(a.logits) & 15) / sizeof(T) : N - 1;
  const long long granules = (a.V + lead + N - 1) / N;
  if (granules <= 128 * 4) return loss_rows_fit<T, DUAL, 128, 4, WRITE>(a, 1, static_cast<int>(granules), s);
  int parts = 1;
  while (parts < 8 && granules > parts * 256ll * kMost) parts *= 2;
  while (parts < 8 && a.rows * parts * 2ll <= num_sms() && granules > parts * 512ll) parts *= 2;
  const int per = static_cast<int>((granules + parts - 1) / parts);
  if (per <= 256 * kMost) return loss_rows_fit<T, DUAL, 256, kMost, WRITE>(a, parts, per, s);
  if (per <= 512 * kMost) return loss_rows_fit<T, DUAL, 512, kMost, WRITE>(a, parts, per, s);
  return loss_stream_launch<T, DUAL, kLossFwd | (WRITE ? kLossBwd : 0)>(a, parts, per, s);
}

template <typename T, bool DUAL> static int loss_mode(const LossArgs& a, int mode, cudaStream_t s) {
  if (mode == kLossFwd) return loss_choose<T, DUAL, false>(a, s);
  if (mode == (kLossFwd | kLossBwd)) return loss_choose<T, DUAL, true>(a, s);
  const int per = 2048;
  const long long granules = (a.V + 2ll * Granule<T>::N - 2) / Granule<T>::N;
  return loss_stream_launch<T, DUAL, kLossBwd>(a, static_cast<int>(granules > per ? (granules + per - 1) / per : 1), per, s);
}

template <typename T> static int loss_launch(const LossArgs& a, int mode, cudaStream_t s) {
  if (a.weight > 0.0f && a.weight < 1.0f && a.top > 0 && a.labels && a.temperature != 1.0f) return loss_mode<T, true>(a, mode, s);
  return loss_mode<T, false>(a, mode, s);
}
}  // namespace tp
