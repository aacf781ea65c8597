// Penalties, bias and grammar mask on next-token logits, and the gradient of the processed logits.
//
//   seen(v)  = v occurs among the row's first len history tokens
//   count(v) = occurrences at positions [prompt_len, len)  (what the model has said so far)
//   y = seen ? (x > 0 ? x / r : x r) : x;   y -= f count + p [count > 0];   y += bias;   not allowed: -inf
//   dx = g * (seen ? (x > 0 ? 1 / r : r) : 1), 0 where not allowed
//
// Bound by reading x (g) and writing y (dx) once.  A CTA takes 32 KB of a row: its loads are issued first and wait in
// registers while the CTA counts the row's history tokens that fall into its part of the vocabulary in shared memory
// (integer atomics: the order does not matter).  A larger part reads the history less often (it comes from L2 once per
// part), a smaller one gives a single row more CTAs: 32 KB keeps both below a tenth of the time at 1536 tokens.
// The backward needs x only for its sign at seen tokens and reads it there alone.
#include <type_traits>

#include "common.cuh"

namespace vo {
namespace {

constexpr int kThreads = 256;
constexpr int kPartBytes = 32768;  // of a row, one CTA

struct LogitArgs {
  const void *x, *g;
  void* y;
  int64_t ldx, ldg, ldy;
  const void* hist;      // [N, L] int64 or int32
  int64_t ldh;
  int hist64, L;
  const int *lens, *prompt_lens;
  const int* rows;       // [R] history row of each logits row; null: the row itself
  int N;                 // history rows
  const float *rep, *pres, *freq;  // [R]
  float rep0, pres0, freq0;        // where the pointers are null
  const float* bias;     // [R or 1, V]
  int64_t ldb;
  const uint32_t* allowed;  // [R or 1, ceil(V / 32)]
  int64_t lda;
  int V;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return bf2f(v); }
template <typename T>
__device__ __forceinline__ T of_f(float v);
template <>
__device__ __forceinline__ float of_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 of_f<__nv_bfloat16>(float v) { return f2bf(v); }

// one history token in the counters: bit 31 for the prompt, plus one for the response (0: not seen)
constexpr uint32_t kSeen = 0x80000000u;

// ALIGNED: rows of x, y (and g, bias) are on 16-byte boundaries, a thread takes 16 bytes at a time; otherwise single
// elements, consecutive threads consecutive ones
template <typename T, bool BWD, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) logits_kernel(const LogitArgs a) {
  constexpr int VEC = 16 / sizeof(T), PART = kPartBytes / sizeof(T), NV = PART / VEC / kThreads;
  extern __shared__ __align__(16) uint32_t cnt[];  // [PART], only with a history
  const int64_t r = blockIdx.y;
  const int v0 = blockIdx.x * PART, nv = min(PART, a.V - v0);
  const T* x = static_cast<const T*>(a.x) + r * a.ldx + v0;
  const T* src = BWD ? static_cast<const T*>(a.g) + r * a.ldg + v0 : x;
  union Pack {
    uint4 u;
    T t[VEC];
  } d[NV];
  // element j of this thread's group k
  auto at = [&](int k, int j) { return ALIGNED ? (threadIdx.x + k * kThreads) * VEC + j : (k * VEC + j) * kThreads + threadIdx.x; };
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (ALIGNED && at(k, 0) + VEC <= nv) {
      d[k].u = __ldcs(reinterpret_cast<const uint4*>(src + at(k, 0)));
    } else {
      d[k].u = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (at(k, j) < nv) d[k].t[j] = src[at(k, j)];
    }
  }
  const bool counted = a.hist != nullptr;
  if (counted) {
    for (int i = threadIdx.x; i < PART / 4; i += kThreads) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int64_t hr = a.rows ? a.rows[r] : r;
    if (VO_DCHECK(hr >= 0 && hr < a.N)) {
      const int len = max(0, min(a.lens ? a.lens[r] : a.L, a.L));
      const int pl = a.prompt_lens ? a.prompt_lens[r] : 0;
      auto count = [&](int64_t tok, int i) {
        const int64_t c = tok - v0;
        if (tok < 0 || c < 0 || c >= nv) return;
        if (i >= pl) atomicAdd(&cnt[c], 1u);
        else atomicOr(&cnt[c], kSeen);
      };
      if (a.hist64) {
        const int64_t* h = static_cast<const int64_t*>(a.hist) + hr * a.ldh;
#pragma unroll 4
        for (int i = threadIdx.x; i < len; i += kThreads) count(__ldg(reinterpret_cast<const long long*>(h) + i), i);
      } else {
        const int* h = static_cast<const int*>(a.hist) + hr * a.ldh;
#pragma unroll 4
        for (int i = threadIdx.x; i < len; i += kThreads) count(__ldg(h + i), i);
      }
    }
    __syncthreads();
  }
  const float rep = a.rep ? a.rep[r] : a.rep0, pres = a.pres ? a.pres[r] : a.pres0, freq = a.freq ? a.freq[r] : a.freq0;
  const float irep = 1.f / rep;
  T* y = static_cast<T*>(a.y) + r * a.ldy + v0;
  const float* bias = !BWD && a.bias ? a.bias + r * a.ldb + v0 : nullptr;
  const uint32_t* ok = a.allowed ? a.allowed + r * a.lda + v0 / 32 : nullptr;
  auto penalise = [&](float z, uint32_t c, int i) {  // c != 0
    if (BWD) return z * (to_f(x[i]) > 0.f ? irep : rep);
    z = z > 0.f ? z / rep : z * rep;
    const uint32_t n = c & ~kSeen;
    return n ? z - fmaf(freq, (float)n, pres) : z;
  };
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i0 = at(k, 0);
    if (i0 >= nv) break;
    if (ALIGNED && i0 + VEC <= nv) {
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = to_f(d[k].t[j]);
      if (counted) {
#pragma unroll
        for (int j4 = 0; j4 < VEC; j4 += 4) {
          const uint4 c4 = *reinterpret_cast<const uint4*>(cnt + i0 + j4);
          if ((c4.x | c4.y | c4.z | c4.w) == 0) continue;
          const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c[j]) f[j4 + j] = penalise(f[j4 + j], c[j], i0 + j4 + j);
        }
      }
      if (bias) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
          const float4 b = __ldg(reinterpret_cast<const float4*>(bias + i0 + j));
          f[j] += b.x, f[j + 1] += b.y, f[j + 2] += b.z, f[j + 3] += b.w;
        }
      }
      if (ok) {
        const uint32_t w = ok[i0 >> 5] >> (i0 & 31);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!((w >> j) & 1u)) f[j] = BWD ? 0.f : -INFINITY;
      }
      Pack o;
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.t[j] = of_f<T>(f[j]);
      __stcs(reinterpret_cast<uint4*>(y + i0), o.u);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int i = at(k, j);
        if (i >= nv) break;
        float f = to_f(d[k].t[j]);
        if (counted && cnt[i]) f = penalise(f, cnt[i], i);
        if (bias) f += bias[i];
        if (ok && !((ok[i >> 5] >> (i & 31)) & 1u)) f = BWD ? 0.f : -INFINITY;
        y[i] = of_f<T>(f);
      }
    }
  }
}

template <typename T, bool BWD, bool ALIGNED>
void launch(const LogitArgs& a, dim3 grid) {
  constexpr int kSmem = kPartBytes / sizeof(T) * 4;
  static const cudaError_t set =
      cudaFuncSetAttribute(logits_kernel<T, BWD, ALIGNED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  VO_CUDA_OK(set);
  logits_kernel<T, BWD, ALIGNED><<<grid, kThreads, a.hist ? kSmem : 0, stream()>>>(a);
  VO_CUDA_OK(cudaGetLastError());
  count_launch();
}

const float* row_param(const c10::optional<torch::Tensor>& t, const char* name, int64_t R, const torch::Tensor& x) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK_VALUE(t->scalar_type() == torch::kFloat32 && t->dim() == 1 && t->size(0) == R && t->is_contiguous() &&
                        t->device() == x.device(),
                    name, ": a number or contiguous float32 [rows] on the logits' device");
  return t->data_ptr<float>();
}

const int* row_ints(const c10::optional<torch::Tensor>& t, const char* name, int64_t R, const torch::Tensor& x) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK_VALUE(t->scalar_type() == torch::kInt32 && t->dim() == 1 && t->size(0) == R && t->is_contiguous() &&
                        t->device() == x.device(),
                    name, ": contiguous int32 [rows] on the logits' device");
  return t->data_ptr<int>();
}

}  // namespace

// x [R, V] fp32 or bf16 (last dim contiguous); g: the gradient of the processed logits (backward) or none.
torch::Tensor process_logits(torch::Tensor x, c10::optional<torch::Tensor> g, c10::optional<torch::Tensor> history,
                             c10::optional<torch::Tensor> lens, c10::optional<torch::Tensor> prompt_lens,
                             c10::optional<torch::Tensor> rows, c10::optional<torch::Tensor> rep, double rep0,
                             c10::optional<torch::Tensor> pres, double pres0, c10::optional<torch::Tensor> freq, double freq0,
                             c10::optional<torch::Tensor> bias, c10::optional<torch::Tensor> allowed) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() == 2 && (x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16),
                    "logits: float32 or bfloat16 [rows, vocab] on a GPU");
  const int64_t R = x.size(0), V = x.size(1);
  TORCH_CHECK_VALUE(V < (1ll << 31), "vocab out of range");
  if (x.stride(1) != 1) x = x.contiguous();
  LogitArgs a{};
  a.V = (int)V;
  if (history.has_value() && history->defined()) {
    const auto& h = *history;
    TORCH_CHECK_VALUE(h.dim() == 2 && (h.scalar_type() == torch::kInt64 || h.scalar_type() == torch::kInt32) &&
                          (h.stride(1) == 1 || h.size(1) <= 1) && h.device() == x.device() && h.size(1) < (1ll << 31) &&
                          h.size(0) < (1ll << 31),
                      "history: int64 or int32 [sequences, tokens], tokens contiguous, on the logits' device");
    a.rows = row_ints(rows, "rows", R, x);
    TORCH_CHECK_VALUE(a.rows || h.size(0) == R, "history: one row per logits row (or pass rows)");
    a.hist = h.numel() ? h.data_ptr() : nullptr;
    a.ldh = h.stride(0);
    a.hist64 = h.scalar_type() == torch::kInt64;
    a.L = (int)h.size(1);
    a.N = (int)h.size(0);
    a.lens = row_ints(lens, "lens", R, x);
    a.prompt_lens = row_ints(prompt_lens, "prompt_lens", R, x);
  }
  a.rep = row_param(rep, "repetition", R, x);
  a.pres = row_param(pres, "presence", R, x);
  a.freq = row_param(freq, "frequency", R, x);
  a.rep0 = (float)rep0;
  a.pres0 = (float)pres0;
  a.freq0 = (float)freq0;
  if (bias.has_value() && bias->defined()) {
    const auto& t = *bias;
    TORCH_CHECK_VALUE(t.scalar_type() == torch::kFloat32 && t.device() == x.device() && t.dim() >= 1 && t.dim() <= 2 &&
                          t.size(-1) == V && t.stride(-1) == 1 && (t.dim() == 1 || t.size(0) == R || t.size(0) == 1),
                      "bias: float32 [vocab] or [rows, vocab] on the logits' device");
    a.bias = t.data_ptr<float>();
    a.ldb = t.dim() == 2 && t.size(0) == R ? t.stride(0) : 0;
  }
  if (allowed.has_value() && allowed->defined()) {
    const auto& t = *allowed;
    TORCH_CHECK_VALUE(t.scalar_type() == torch::kInt32 && t.device() == x.device() && t.dim() == 2 &&
                          t.size(1) == (V + 31) / 32 && t.stride(1) == 1 && (t.size(0) == R || t.size(0) == 1),
                      "allowed: int32 bitmask [rows or 1, ceil(vocab / 32)] on the logits' device");
    a.allowed = reinterpret_cast<const uint32_t*>(t.data_ptr<int>());
    a.lda = t.size(0) == R ? t.stride(0) : 0;
  }
  c10::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty({R, V}, x.options());
  if (y.numel() == 0) return y;
  const bool bwd = g.has_value() && g->defined();
  torch::Tensor gt;
  if (bwd) {
    TORCH_CHECK_VALUE(g->sizes() == x.sizes() && g->scalar_type() == x.scalar_type() && g->device() == x.device(),
                      "gradient: like the logits");
    gt = g->stride(1) == 1 ? *g : g->contiguous();
    a.g = gt.data_ptr();
    a.ldg = gt.stride(0);
  }
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  a.y = y.data_ptr();
  a.ldy = V;
  TORCH_CHECK_VALUE(R <= 65535 * 1024ll, "too many rows");
  const int64_t es = x.element_size();
  const int64_t parts = (V * es + kPartBytes - 1) / kPartBytes;
  const auto aligned = [&](const void* p, int64_t ld, int64_t size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0; };
  const bool vec = aligned(a.x, a.ldx, es) && aligned(a.y, a.ldy, es) && (!bwd || aligned(a.g, a.ldg, es)) &&
                   (!a.bias || aligned(a.bias, a.ldb, 4));
  // grid.y holds 65535 rows at most: more rows in further launches, each on its rows' slices
  for (int64_t r0 = 0; r0 < R; r0 += 65535) {
    LogitArgs b = a;
    b.x = static_cast<const char*>(a.x) + r0 * a.ldx * es;
    b.y = static_cast<char*>(a.y) + r0 * a.ldy * es;
    if (bwd) b.g = static_cast<const char*>(a.g) + r0 * a.ldg * es;
    if (a.rows) b.rows = a.rows + r0;
    else if (a.hist) {
      b.hist = static_cast<const char*>(a.hist) + r0 * a.ldh * (a.hist64 ? 8 : 4);
      b.N = a.N - (int)r0;
    }
    for (const int** p : {&b.lens, &b.prompt_lens})
      if (*p) *p += r0;
    for (const float** p : {&b.rep, &b.pres, &b.freq})
      if (*p) *p += r0;
    if (b.bias) b.bias += r0 * a.ldb;
    if (b.allowed) b.allowed += r0 * a.lda;
    const dim3 grid((unsigned)parts, (unsigned)std::min<int64_t>(65535, R - r0));
    auto run = [&](auto t, auto back) {
      using T = decltype(t);
      constexpr bool B = decltype(back)::value;
      vec ? launch<T, B, true>(b, grid) : launch<T, B, false>(b, grid);
    };
    if (x.scalar_type() == torch::kFloat32) bwd ? run(float(), std::true_type{}) : run(float(), std::false_type{});
    else bwd ? run(__nv_bfloat16(), std::true_type{}) : run(__nv_bfloat16(), std::false_type{});
  }
  return y;
}

}  // namespace vo
