// Penalties, bias and grammar mask on next-token logits, and the gradient of the processed logits.
//
//   seen(v)  = v occurs among the row's first len history tokens
//   count(v) = occurrences at positions [prompt_len, len)  (what the model has said so far)
//   y = seen ? (x > 0 ? x / r : x r) : x;   y -= f count + p [count > 0];   y += bias;   not allowed: -inf
//   dx = g * (seen ? (x > 0 ? 1 / r : r) : 1), 0 where not allowed
//
// Bound by reading x (g) and writing y (dx) once.  CTAs walk through 32 KB parts of the rows, each a contiguous run of
// them, in two steps.  All entries: bias and mask, 16 bytes at a time, the next part on its way in registers meanwhile.
// Then the few entries that the history penalises, one thread a token, computed from x and written over; testing every
// entry for a penalty instead took four times the instructions and was bound by them.
// A row's distinct tokens and their counts come from a hash table in shared memory, filled once per row (integer atomics:
// the order does not matter) and sorted by part, so that a part starts the loads of its tokens' entries before its stream.
// Histories longer than kStaged tokens (and vocabularies of more than kMaxParts parts) are counted part by part in
// direct-addressed counters instead, read from L2 each time.
// Measured (B200): 64 x 151936 fp32 with a mask 23.6 us (12.2 at the copy rate; the table is filled ahead of the penalised
// entries), 512 x 151936 bf16 70 us, its gradient 76 us (a plain copy 51).  Tokens counted per part: 261 us for the two.
// The backward needs x only for its sign at those tokens and reads it there alone.
#include <type_traits>

#include "common.cuh"
#include "per_device.h"

namespace vo {
namespace {

constexpr int kThreads = 512;
constexpr int kPartBytes = 32768;  // of a row
constexpr int kStaged = 4096;      // history tokens of a row at most for the hash table: 96 KB, two CTAs per SM
constexpr int kMaxParts = 256;     // parts of a row at most for the sort

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
  int parts;         // of a row
  int64_t total;     // parts of all rows
  int per;           // CTAs of a row, 0: a CTA takes parts of several rows
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

// two consecutive entries of a 32-bit word, or one
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float* f) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* f) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    const bf16x8 v = pack8(f);
    return *reinterpret_cast<const uint4*>(&v);
  }
}

// places of the hash table for a history of L tokens: a power of two, half of them empty at least
__host__ __device__ __forceinline__ int table_size(int L) {
  int h = 64;
  while (h < 2 * L) h *= 2;
  return h;
}

// ALIGNED: rows of x, y (and g, bias) are on 16-byte boundaries, a thread takes 16 bytes at a time; otherwise single
// entries, consecutive threads consecutive ones.  LONG: counters per part instead of the hash table per row.
template <typename T, bool BWD, bool ALIGNED, bool LONG>
__global__ void __launch_bounds__(kThreads, 2) logits_kernel(const LogitArgs a) {
  constexpr int VEC = 16 / sizeof(T), PART = kPartBytes / sizeof(T), NV = PART / VEC / kThreads;
  // LONG: counters [PART].  Otherwise keys and counts of the table, tokens and counts by part.  Only with a history
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ int first[kMaxParts + 1], fill[kMaxParts];  // tokens of a part: [first, next first)
  uint32_t* cnt = smem;
  const int H = LONG ? 0 : table_size(a.L);
  int* keys = reinterpret_cast<int*>(smem);
  uint32_t* vals = smem + H;
  int* list = reinterpret_cast<int*>(smem + 2 * H);
  uint32_t* list_n = smem + 2 * H + a.L;
  const int tid = threadIdx.x;
  // fewer rows than CTAs: a.per CTAs share a row, so that each fills one table; otherwise one line of all parts
  const int64_t lines = a.per ? blockIdx.x / a.per : 0, line = a.per ? a.parts : a.total;
  const int in = a.per ? blockIdx.x % a.per : blockIdx.x, of = a.per ? a.per : gridDim.x;
  const int64_t w0 = lines * line + line * in / of, w1 = lines * line + line * (in + 1) / of;
  // entry j of this thread's group k
  auto at = [&](int k, int j) { return ALIGNED ? (tid + k * kThreads) * VEC + j : (k * VEC + j) * kThreads + tid; };
  union Pack {
    uint4 u;
    T t[VEC];
  };
  const T* xs = static_cast<const T*>(a.x);
  const T* ss = BWD ? static_cast<const T*>(a.g) : xs;
  const int64_t lds = BWD ? a.ldg : a.ldx;
  auto load = [&](int64_t r, int v0, Pack(&d)[NV]) {
    const int nv = min(PART, a.V - v0);
    const T* src = ss + r * lds + v0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      d[k].u = make_uint4(0, 0, 0, 0);
      if (ALIGNED && at(k, 0) + VEC <= nv) {
        d[k].u = __ldg(reinterpret_cast<const uint4*>(src + at(k, 0)));
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (at(k, j) < nv) d[k].t[j] = src[at(k, j)];
      }
    }
  };
  // mask words of this thread's groups
  auto load_mask = [&](int64_t r, int v0, uint32_t(&m)[NV]) {
    if (!ALIGNED || !a.allowed) return;
    const int nv = min(PART, a.V - v0);
    const uint32_t* ok = a.allowed + r * a.lda + v0 / 32;
#pragma unroll
    for (int k = 0; k < NV; ++k) m[k] = at(k, 0) < nv ? __ldg(ok + (at(k, 0) >> 5)) : 0;
  };
  int64_t r = w0 / a.parts;
  int part = (int)(w0 % a.parts);
  Pack d[NV];
  uint32_t mw[NV];
  if (w0 < w1) {
    load(r, part * PART, d);
    load_mask(r, part * PART, mw);
  }
  const bool counted = a.hist != nullptr;
  if (LONG)
    for (int i = tid; i < PART / 4; i += kThreads) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
  struct Tok {
    int at, n, c;  // the part's tokens in the list, this thread's one
    T z, x;        // its entries as loaded: a conversion would wait for them
  };
  auto fetch = [&](int64_t r, int part, Tok& t) {
    t.at = first[part];
    t.n = first[part + 1] - t.at;
    if (tid < t.n) {
      t.c = list[t.at + tid];
      t.z = ss[r * lds + part * PART + t.c];
      if (BWD) t.x = xs[r * a.ldx + part * PART + t.c];
    }
  };
  Tok t0;
  t0.n = 0;
  int64_t row = -1;  // whose history and parameters are loaded
  int len = 0, pl = 0;
  const void* hist = nullptr;
  float rep = 1.f, irep = 1.f, pres = 0.f, freq = 0.f;
  for (int64_t w = w0; w < w1; ++w) {
    const int v0 = part * PART, nv = min(PART, a.V - v0);
    auto token = [&](int i) -> int64_t {  // -1: no entry of the vocabulary
      const int64_t t = a.hist64 ? (int64_t)__ldg(static_cast<const long long*>(hist) + i) : (int64_t)__ldg(static_cast<const int*>(hist) + i);
      return t >= 0 && t < a.V ? t : -1;
    };
    const bool new_row = counted && row != r;
    if (new_row) {
      row = r;
      rep = a.rep ? a.rep[r] : a.rep0;
      pres = a.pres ? a.pres[r] : a.pres0;
      freq = a.freq ? a.freq[r] : a.freq0;
      irep = 1.f / rep;
      const int64_t hr = a.rows ? a.rows[r] : r;
      const bool known = VO_DCHECK(hr >= 0 && hr < a.N);
      len = known ? max(0, min(a.lens ? a.lens[r] : a.L, a.L)) : 0;
      pl = a.prompt_lens ? a.prompt_lens[r] : 0;
      hist = known ? static_cast<const char*>(a.hist) + hr * a.ldh * (a.hist64 ? 8 : 4) : nullptr;
    }
    const T *x = xs + r * a.ldx + v0, *src = ss + r * lds + v0;
    T* y = static_cast<T*>(a.y) + r * a.ldy + v0;
    const float* bias = !BWD && a.bias ? a.bias + r * a.ldb + v0 : nullptr;
    const uint32_t* ok = a.allowed ? a.allowed + r * a.lda + v0 / 32 : nullptr;
    constexpr float kOut = BWD ? 0.f : -INFINITY;  // where the mask forbids
    auto each = [&](auto f) {  // LONG: f(place in the part, position) for the tokens that fall into it
#pragma unroll 4
      for (int i = tid; i < len; i += kThreads) {
        const int64_t c = token(i) - v0;
        if (c >= 0 && c < nv) f((int)c, i);
      }
    };
    int64_t r_next = r;
    int part_next = part + 1;
    if (part_next == a.parts) part_next = 0, ++r_next;
    Pack dn[NV];
    uint32_t mn[NV];
    if (w + 1 < w1) {
      load(r_next, part_next * PART, dn);
      load_mask(r_next, part_next * PART, mn);
    }
    Tok t1;
    const bool same = !LONG && counted && r_next == r && w + 1 < w1;  // the next part's tokens come from this table
    if (same && !new_row) fetch(r, part_next, t1);
    if (LONG) {
      __syncthreads();  // counters are clear
      each([&](int c, int i) {
        if (i >= pl) atomicAdd(&cnt[c], 1u);
        else atomicOr(&cnt[c], kSeen);
      });
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i0 = at(k, 0);
      if (ALIGNED && i0 + VEC <= nv) {
        if (bias || ok) {
          float f[VEC];
          unpack16<T>(d[k].u, f);
          if (bias) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
              const float4 b = __ldg(reinterpret_cast<const float4*>(bias + i0 + j));
              f[j] += b.x, f[j + 1] += b.y, f[j + 2] += b.z, f[j + 3] += b.w;
            }
          }
          if (ok) {
            const uint32_t m = mw[k] >> (i0 & 31);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = (m >> j) & 1u ? f[j] : kOut;
          }
          d[k].u = pack16<T>(f);
        }
        *reinterpret_cast<uint4*>(y + i0) = d[k].u;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int i = at(k, j);
          if (i >= nv) break;
          float f = to_f(d[k].t[j]);
          if (bias) f += bias[i];
          if (ok && !((ok[i >> 5] >> (i & 31)) & 1u)) f = kOut;
          y[i] = of_f<T>(f);
        }
      }
    }
    if constexpr (!LONG) {
      if (new_row) {  // behind the first part's stream, which does not need it
        // of the parts that this CTA takes of the row
        const int64_t left = w1 - w;
        const int vlo = v0, vhi = left >= a.parts - part ? a.V : (part + (int)left) * PART;
        __syncthreads();  // the row before is done with its tokens
        const uint32_t none = 0xffffffffu;
        for (int i = tid; i < H / 4; i += kThreads) {
          reinterpret_cast<uint4*>(keys)[i] = make_uint4(none, none, none, none);
          reinterpret_cast<uint4*>(vals)[i] = make_uint4(0, 0, 0, 0);
        }
        for (int i = tid; i <= a.parts; i += kThreads) first[i] = 0;
        __syncthreads();
        constexpr int AT_ONCE = 4;  // token loads in flight
        for (int i0 = tid; i0 < len; i0 += AT_ONCE * kThreads) {
          int t[AT_ONCE];
#pragma unroll
          for (int q = 0; q < AT_ONCE; ++q) t[q] = i0 + q * kThreads < len ? (int)token(i0 + q * kThreads) : -1;
#pragma unroll
          for (int q = 0; q < AT_ONCE; ++q) {
            if (t[q] < vlo || t[q] >= vhi) continue;
            uint32_t h = ((uint32_t)t[q] * 2654435761u) >> 7;  // multiplicative hash
            int k;
            while ((k = atomicCAS(&keys[h &= H - 1], -1, t[q])) != -1 && k != t[q]) ++h;
            if (i0 + q * kThreads >= pl) atomicAdd(&vals[h], 1u);
            else atomicOr(&vals[h], kSeen);
            if (k == -1) atomicAdd(&first[t[q] / PART + 1], 1);
          }
        }
        __syncthreads();
        if (tid < 32) {  // running sums over the parts
          int sum = 0;
          for (int p0 = 0; p0 < a.parts; p0 += 32) {
            int v = p0 + tid < a.parts ? first[p0 + tid + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int u = __shfl_up_sync(0xffffffffu, v, o);
              if (tid >= o) v += u;
            }
            if (p0 + tid < a.parts) first[p0 + tid + 1] = sum + v;
            sum += __shfl_sync(0xffffffffu, v, 31);
          }
          __syncwarp();
          for (int p = tid; p < a.parts; p += 32) fill[p] = first[p];
        }
        __syncthreads();
        for (int i = tid; i < H; i += kThreads) {
          const int t = keys[i];
          if (t < 0) continue;
          const int n = atomicAdd(&fill[t / PART], 1);
          list[n] = t % PART;
          list_n[n] = vals[i];
        }
        __syncthreads();
        fetch(r, part, t0);
        if (same) fetch(r, part_next, t1);
      }
    }
    if (counted) {
      __syncthreads();  // entries are written (LONG: tokens are counted)
      auto penalise = [&](int c, float z, float xv, uint32_t n) {
        if (BWD) {
          z *= xv > 0.f ? irep : rep;
        } else {
          z = z > 0.f ? z / rep : z * rep;
          n &= ~kSeen;
          if (n) z -= fmaf(freq, (float)n, pres);
          if (bias) z += bias[c];
        }
        if (ok && !((ok[c >> 5] >> (c & 31)) & 1u)) z = kOut;
        y[c] = of_f<T>(z);
      };
      if constexpr (LONG) {
        each([&](int c, int) { penalise(c, to_f(src[c]), to_f(x[c]), cnt[c]); });
        __syncthreads();
        each([&](int c, int) { cnt[c] = 0; });
      } else {
        if (tid < t0.n) penalise(t0.c, to_f(t0.z), BWD ? to_f(t0.x) : 0.f, list_n[t0.at + tid]);
        for (int i = tid + kThreads; i < t0.n; i += kThreads) {
          const int c = list[t0.at + i];
          penalise(c, to_f(src[c]), BWD ? to_f(x[c]) : 0.f, list_n[t0.at + i]);
        }
        t0 = t1;
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) d[k] = dn[k], mw[k] = mn[k];
    r = r_next;
    part = part_next;
  }
}

template <typename T, bool BWD, bool ALIGNED, bool LONG>
void launch(const LogitArgs& a) {
  constexpr int kMost = LONG ? kPartBytes / (int)sizeof(T) * 4 : (2 * 2 * kStaged + 2 * kStaged) * 4;
  static PerDevice once;
  VO_CUDA_OK(once([] { return cudaFuncSetAttribute(logits_kernel<T, BWD, ALIGNED, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost); }));
  const int smem = !a.hist ? 0 : LONG ? kMost : (2 * table_size(a.L) + 2 * a.L) * 4;
  const int most = 2 * num_sms();
  const int64_t R = a.total / a.parts;
  LogitArgs b = a;
  b.per = R <= most ? (int)std::min<int64_t>(a.parts, most / R) : 0;
  const int grid = b.per ? (int)R * b.per : most;
  logits_kernel<T, BWD, ALIGNED, LONG><<<grid, kThreads, smem, stream()>>>(b);
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
  const int64_t es = x.element_size();
  a.parts = (int)((V * es + kPartBytes - 1) / kPartBytes);
  a.total = R * a.parts;
  const auto aligned = [&](const void* p, int64_t ld, int64_t size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0; };
  const bool vec = aligned(a.x, a.ldx, es) && aligned(a.y, a.ldy, es) && (!bwd || aligned(a.g, a.ldg, es)) &&
                   (!a.bias || aligned(a.bias, a.ldb, 4));
  auto run = [&](auto t, auto back) {
    using T = decltype(t);
    constexpr bool B = decltype(back)::value;
    if (a.hist && (a.L > kStaged || a.parts > kMaxParts)) vec ? launch<T, B, true, true>(a) : launch<T, B, false, true>(a);
    else vec ? launch<T, B, true, false>(a) : launch<T, B, false, false>(a);
  };
  if (x.scalar_type() == torch::kFloat32) bwd ? run(float(), std::true_type{}) : run(float(), std::false_type{});
  else bwd ? run(__nv_bfloat16(), std::true_type{}) : run(__nv_bfloat16(), std::false_type{});
  return y;
}

}  // namespace vo
