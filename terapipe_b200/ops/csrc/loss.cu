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
};

__device__ __forceinline__ float load_float(const void* p, long long i, int dtype) {
  if (dtype == 2) return static_cast<const float*>(p)[i];
  if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

enum { kLossFwd = 1, kLossBwd = 2 };   // bits of MODE

// Reductions over the CTA; every thread gets the result.  `red` holds 33 floats.
template <bool MAX> __device__ __forceinline__ float cta_reduce(float v, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float t = MAX ? -INFINITY : 0.0f;
  for (int w = 0; w < nw; ++w) t = MAX ? fmaxf(t, red[w]) : t + red[w];
  return t;
}

// One CTA per row.
template <typename T, int MODE>
__global__ void __launch_bounds__(512)
loss_kernel(const LossArgs a) {
  extern __shared__ float top_smem[];           // [top] p, [top] z, [top] id
  __shared__ float red[33];
  float* top_p = top_smem;
  float* top_z = top_p + a.top;
  int* top_id = reinterpret_cast<int*>(top_z + a.top);
  pdl_wait();
  const int row = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  const float inv_t = 1.0f / a.temperature;
  long long label = -1;
  if (a.labels && a.weight != 1.0f) {
    label = load_id(a.labels, a.label_at(row), a.labels64);
    if (label == a.ignore || label < 0 || label >= a.V) label = -1;
  }
  // the teacher's distribution
  float t_max = -INFINITY;
  for (int k = tid; k < a.top; k += threads) {
    const long long id = load_id(a.tid, a.tid_at(row) + k, a.tid64);
    const bool in = id >= 0 && id < a.V;
    const float t = in ? load_float(a.tlog, a.tlog_at(row) + k, a.tlog_dtype) : -INFINITY;
    top_id[k] = in ? static_cast<int>(id) : -1;
    top_p[k] = t;
    top_z[k] = in ? Elem<T>::to_f(z[id]) : 0.0f;
    t_max = fmaxf(t_max, t);
  }
  float t_sum = 0.0f;
  if (a.top > 0) {
    t_max = cta_reduce<true>(t_max, red);
    if (t_max == -INFINITY) t_max = 0.0f;
    for (int k = tid; k < a.top; k += threads)
      if (top_id[k] >= 0) t_sum += __expf((top_p[k] - t_max) * inv_t);
    t_sum = cta_reduce<false>(t_sum, red);
  }
  const bool teach = a.weight != 0.0f && a.top > 0 && t_sum != 0.0f, active = teach || label >= 0;
  const float z_label = label >= 0 ? Elem<T>::to_f(z[label]) : 0.0f;
  float m, s1, st;
  if (MODE & kLossFwd) {
    m = -INFINITY;
    for (int j = tid; j < a.V; j += threads) m = fmaxf(m, Elem<T>::to_f(z[j]));
    m = cta_reduce<true>(m, red);
    if (m == -INFINITY) m = 0.0f;
    s1 = 0.0f, st = 0.0f;
    for (int j = tid; j < a.V; j += threads) {
      const float d = Elem<T>::to_f(z[j]) - m;
      s1 += __expf(d);
      st += __expf(d * inv_t);
    }
    s1 = cta_reduce<false>(s1, red);
    st = cta_reduce<false>(st, red);
    float kl = 0.0f;
    for (int k = tid; k < a.top; k += threads) {
      if (top_id[k] < 0) continue;
      const float lt = (top_p[k] - t_max) * inv_t, p = __expf(lt) / t_sum;
      if (p > 0.0f) kl += p * ((lt - __logf(t_sum)) - ((top_z[k] - m) * inv_t - __logf(st)));
    }
    kl = a.top > 0 ? cta_reduce<false>(kl, red) : 0.0f;
    if (tid == 0) {
      float loss = 0.0f;
      if (s1 != 0.0f) {
        if (label >= 0) loss = (1.0f - a.weight) * (__logf(s1) - (z_label - m));
        if (teach) loss += a.weight * a.temperature * a.temperature * kl;
      }
      a.loss[row] = loss;
      if (a.stats) {
        a.stats[4ll * row] = m;
        a.stats[4ll * row + 1] = s1;
        a.stats[4ll * row + 2] = st;
      }
    }
  } else {
    m = a.stats[4ll * row];
    s1 = a.stats[4ll * row + 1];
    st = a.stats[4ll * row + 2];
  }
  if (MODE & kLossBwd) {
    T* dz = static_cast<T*>(a.dlogits) + row * a.ldd;
    const bool zero = !active || s1 == 0.0f;
    const float g = a.grad_scale * (a.grad_loss ? a.grad_loss[row * a.ldg] : 1.0f);
    const float g1 = label >= 0 ? g * (1.0f - a.weight) : 0.0f, gt = teach ? g * a.weight * a.temperature : 0.0f;
    const float c1 = g1 / s1, ct = gt / st;
    for (int j = tid; j < a.V; j += threads) {
      const float d = Elem<T>::to_f(z[j]) - m;
      dz[j] = Elem<T>::from_f(zero ? 0.0f : c1 * __expf(d) + ct * __expf(d * inv_t));
    }
    __syncthreads();      // the label's and the teacher's elements come last
    if (!zero) {
      for (int k = tid; k <= a.top; k += threads) {
        const int id = k < a.top ? top_id[k] : static_cast<int>(label);
        if (id < 0) continue;
        float p = 0.0f;
        bool first = true;
        for (int o = 0; o < a.top; ++o) {
          if (top_id[o] != id) continue;
          if (o < k) first = false;
          p += teach ? __expf((top_p[o] - t_max) * inv_t) / t_sum : 0.0f;
        }
        if (!first) continue;
        const float d = (k < a.top ? top_z[k] : z_label) - m;
        // (each difference by itself: exactly zero where both distributions have one value only)
        dz[id] = Elem<T>::from_f((c1 * __expf(d) - (id == label ? g1 : 0.0f)) + (ct * __expf(d * inv_t) - gt * p));
      }
    }
  }
}

template <typename T> static int loss_launch(const LossArgs& a, int mode, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(a.top) * 12;
  const dim3 grid(a.rows), block(512);
  if (mode == kLossFwd) launch_pdl(loss_kernel<T, kLossFwd>, grid, block, smem, s, 1, a);
  else if (mode == kLossBwd) launch_pdl(loss_kernel<T, kLossBwd>, grid, block, smem, s, 1, a);
  else launch_pdl(loss_kernel<T, kLossFwd | kLossBwd>, grid, block, smem, s, 1, a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}
}  // namespace tp

using namespace tp;

// mode: 1 loss and stats, 2 gradient from stats, 3 loss and gradient.  dtype, tlog_dtype: 0 fp16, 1 bf16, 2 fp32.  Outer
// index i of an array lies at (i / cols) * s0 + (i % cols) * s1.  dlogits may be logits.
extern "C" int tp_loss(int mode, int dtype, const void* logits, long long ld, int rows, int V, const void* labels,
                       int labels64, int label_cols, long long label_s0, long long label_s1, long long ignore,
                       const void* tid, int tid64, int tid_cols, long long tid_s0, long long tid_s1, const void* tlog,
                       int tlog_dtype, int tlog_cols, long long tlog_s0, long long tlog_s1, int top, float temperature,
                       float weight, float* loss, float* stats, void* dlogits, long long ldd, const float* grad_loss,
                       long long ldg, float grad_scale, void* stream) {
  if (mode < 1 || mode > 3 || dtype < 0 || dtype > 2 || tlog_dtype < 0 || tlog_dtype > 2 || rows < 0 || V < 0 || top < 0 ||
      label_cols < 1 || tid_cols < 1 || tlog_cols < 1 || !(temperature > 0.0f) || (top > 0 && (!tid || !tlog)))
    return kErrBadArgument;
  if (top > kMaxTop) return kErrTooLarge;
  if (rows == 0) return kOk;
  if (((mode & kLossFwd) && !loss) || (mode == kLossBwd && !stats) || ((mode & kLossBwd) && V > 0 && !dlogits))
    return kErrBadArgument;
  LossArgs a{logits, ld, rows, V, labels, OuterIndex{label_s0, label_s1, label_cols}, ignore, labels64, tid, tlog,
             OuterIndex{tid_s0, tid_s1, tid_cols}, OuterIndex{tlog_s0, tlog_s1, tlog_cols}, top, tid64, tlog_dtype,
             temperature, weight, loss, stats, dlogits, ldd, grad_loss, ldg, grad_scale};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return loss_launch<__half>(a, mode, s);
  if (dtype == 1) return loss_launch<__nv_bfloat16>(a, mode, s);
  return loss_launch<float>(a, mode, s);
}
