// 8-bit paged KV cache: quantising append, page copies, and attention on the CUDA cores.
//
// A pool holds e4m3 numbers [pages, Hk, block, hd] and one fp32 scale per (page, KV head), a power of two:
// the smallest 2^e (e >= -100) with amax <= 448 * 2^e.  Dividing by a power of two is exact, so a value is
// rounded once when it is written, and bringing a partly filled page to a larger scale moves exponents only
// (a value rounds again only where it becomes subnormal in e4m3).  A row holds the value code * scale.
#include <string>

#include "common.cuh"
#include "paged8.cuh"
#include "paged8_tc.h"

namespace vo {
namespace {

using p8::kMinExp;

// ------------------------------------------------------------------------------------------------- append
constexpr int kAppendMax = 256;  // threads at most
constexpr int kHeld = 8;         // 16-byte pieces that a thread keeps in registers

struct AppendArgs {
  const __nv_bfloat16 *k, *v;       // [B, Hk, S, hd], last dim contiguous
  int64_t ksb, ksh, kss, vsb, vsh, vss;
  uint8_t *kp, *vp;                 // [pages, Hk, block, hd]
  float *ks, *vs;                   // [pages, Hk]
  const int *table, *start, *counts;
  int width, pages, B, Hk, S, hd, block, offset, touched;
};

// largest magnitude among 8 values as bf16 bits (of |x|: they order like the numbers), per half word
__device__ __forceinline__ uint32_t amax_bits(const uint4& u, uint32_t m) {
  m = __vmaxu2(m, u.x & 0x7fff7fffu);
  m = __vmaxu2(m, u.y & 0x7fff7fffu);
  m = __vmaxu2(m, u.z & 0x7fff7fffu);
  return __vmaxu2(m, u.w & 0x7fff7fffu);
}
// the same over finite values only
__device__ __forceinline__ uint32_t amax_finite(const uint4& u, uint32_t m) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = w[i] & 0x7fff7fffu;
    m = __vmaxu2(m, a & ~__vcmpgeu2(a, 0x7f807f80u));
  }
  return m;
}

// One CTA per (sequence, touched page, KV head, K or V).  Bound by reading the new rows and writing their codes: the rows
// are loaded once, all loads in flight, and kept in registers over the page's maximum (a page of more than
// kAppendMax * kHeld pieces, 32 KB, is read a second time, from L2).
// Measured (B200, 4 KV heads of 128): 64 x 1 token 4.4 us (launch), 24 ragged sequences up to 333 tokens 8.2 us (dependent
// loads), 64 x 1024 tokens 42.6 us = 4.7 TB/s, 64 x 4096 tokens 141 us = 5.7 TB/s.
__global__ void __launch_bounds__(kAppendMax) append_kernel(const AppendArgs a) {
  __shared__ uint32_t red[kAppendMax / 32];
  const int b = blockIdx.x / a.touched, t = blockIdx.x % a.touched, h = blockIdx.y, nt = blockDim.x, tid = threadIdx.x;
  const bool is_v = blockIdx.z != 0;
  const int p0 = a.start[b] + a.offset;
  const int n = a.counts ? max(0, min(a.counts[b], a.S)) : a.S;
  if (!VO_DCHECK(p0 >= 0) || n == 0) return;
  const int page = p0 / a.block + t;
  const int64_t base = (int64_t)page * a.block;
  const int lo = (int)max((int64_t)p0, base) - p0;                       // first new row of this page
  const int hi = (int)min((int64_t)p0 + n, base + a.block) - p0;         // one past the last
  if (lo >= hi) return;
  if (!VO_DCHECK(page < a.width)) return;                                // past the table: dropped
  const int id = a.table[(int64_t)b * a.width + page];
  const __nv_bfloat16* x = is_v ? a.v + b * a.vsb + h * a.vsh + lo * a.vss : a.k + b * a.ksb + h * a.ksh + lo * a.kss;
  const int64_t xs = is_v ? a.vss : a.kss;
  const int upr = a.hd / 8, units = (hi - lo) * upr;
  auto piece = [&](int u) { return __ldg(reinterpret_cast<const uint4*>(x + (u / upr) * xs + (u % upr) * 8)); };
  uint4 held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = tid + i * nt < units ? piece(tid + i * nt) : make_uint4(0, 0, 0, 0);
  if (!VO_DCHECK(id >= 0 && id < a.pages)) return;
  const int r0 = (int)(p0 + lo - base);                                  // rows already in the page
  uint8_t* dst = (is_v ? a.vp : a.kp) + ((int64_t)id * a.Hk + h) * a.block * a.hd;
  float* sp = (is_v ? a.vs : a.ks) + (int64_t)id * a.Hk + h;
  const float was = r0 > 0 ? *sp : 0.f;
  auto page_max = [&](auto f) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) m = f(held[i], m);
    for (int u = tid + kHeld * nt; u < units; u += nt) m = f(piece(u), m);
    m = max(m & 0xffffu, m >> 16);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    m = red[0];
    for (int i = 1; i < nt / 32; ++i) m = max(m, red[i]);
    return m;
  };
  uint32_t m = page_max([](const uint4& u, uint32_t v) { return amax_bits(u, v); });
  if (m >= 0x7f80u) {  // an infinity or NaN among the rows: they do not count
    __syncthreads();
    m = page_max([](const uint4& u, uint32_t v) { return amax_finite(u, v); });
  }
  float now = p8::scale_of(__uint_as_float(m << 16));
  if (r0 > 0) {
    now = fmaxf(was, now);
    if (now != was) {
      const float ratio = was / now;
      for (int u = tid; u < r0 * upr; u += nt) {
        uint2* w = reinterpret_cast<uint2*>(dst + (int64_t)u * 8);
        float f[8];
        p8::unpack_e4m3x8(*w, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= ratio;
        *w = p8::pack_e4m3x8(f);
      }
    }
  }
  if (tid == 0) *sp = now;  // every thread read the old scale before the barrier above
  const float inv = 1.f / now;
  auto put = [&](int u, const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16) * inv, f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * inv;
    *reinterpret_cast<uint2*>(dst + (int64_t)r0 * a.hd + (int64_t)u * 8) = p8::pack_e4m3x8(f);  // rows follow one another in a page
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (tid + i * nt < units) put(tid + i * nt, held[i]);
  for (int u = tid + kHeld * nt; u < units; u += nt) put(u, piece(u));
}

// ------------------------------------------------------------------------------------------------- page copies
constexpr int kMaxPools = 8;
struct CopyArgs {
  uint8_t* base[kMaxPools];
  int64_t page_bytes[kMaxPools];  // bytes of one page of one layer
  int64_t layer_bytes[kMaxPools];
  int vec[kMaxPools];             // bytes per access: 16, 4 or 1
  const int *src, *dst;
  int pages;
};

// One CTA per (pair, layer, pool), bound by memory.  Measured (B200, 4 KV heads of 128): 400 pages of 128 rows x 8 layers 145 us =
// 5.8 TB/s, 7 pages of 16 rows x 48 layers 5.0 us (launch).  Four loads of a thread in flight: 136 and 6.1 us, so plain.
template <typename T>
__device__ __forceinline__ void copy_as(uint8_t* d, const uint8_t* s, int64_t n) {
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) reinterpret_cast<T*>(d)[i] = reinterpret_cast<const T*>(s)[i];
}

__global__ void __launch_bounds__(256) copy_pages_kernel(const CopyArgs a) {
  const int i = blockIdx.x, layer = blockIdx.y, p = blockIdx.z;
  const int s = a.src[i], d = a.dst[i];
  if (!VO_DCHECK(s >= 0 && s < a.pages && d >= 0 && d < a.pages)) return;  // outside the pool: skipped
  uint8_t* base = a.base[p] + layer * a.layer_bytes[p];
  const uint8_t* from = base + s * a.page_bytes[p];
  uint8_t* to = base + d * a.page_bytes[p];
  if (a.vec[p] == 16) copy_as<uint4>(to, from, a.page_bytes[p] / 16);
  else if (a.vec[p] == 4) copy_as<uint32_t>(to, from, a.page_bytes[p] / 4);
  else copy_as<uint8_t>(to, from, a.page_bytes[p]);
}

// ------------------------------------------------------------------------------------------------- attention
// Any head_dim that is a multiple of 16 up to 256, any page size: one CTA per (sequence, query token, query
// head), its four warps take 32-key groups in turn.  Scores: lane = key, the lane reads its whole row; P V:
// lane = head-dim columns, probabilities broadcast by shuffles.  Every warp keeps its own running maximum,
// sum and output, merged in shared memory at the end.  Bound by each query head reading the rows again and by the lane's
// row-by-row loads.  Measured (B200): 16 sequences x 2048 rows, 4 KV and 16 query heads of 96, pages of 16: 293 us.
constexpr int kMaxHd = 256;

__global__ void __launch_bounds__(128) attend_any_kernel(const p8::AttendArgs a) {
  __shared__ float qs[kMaxHd];
  __shared__ float os[4][kMaxHd];
  __shared__ float ml[4][2];
  const int hd = a.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t id = blockIdx.x;
  const int hq = (int)(id % a.Hq);
  id /= a.Hq;
  const int s = (int)(id % a.S), b = (int)(id / a.S);
  const int kh = hq / a.rep;
  __nv_bfloat16* out = a.out + (((int64_t)b * a.S + s) * a.Hq + hq) * hd;
  const int len = p8::row_limit(a, b, s);
  if (len <= 0) {
    for (int i = threadIdx.x; i < hd; i += 128) out[i] = f2bf(0.f);
    return;
  }
  const __nv_bfloat16* q = a.q + b * a.qsb + hq * a.qsh + s * a.qss;
  for (int i = threadIdx.x; i < hd; i += 128) qs[i] = bf2f(q[i]) * a.scale_log2;
  __syncthreads();
  float m = -INFINITY, l = 0.f;
  float acc[kMaxHd / 32];
#pragma unroll
  for (int j = 0; j < kMaxHd / 32; ++j) acc[j] = 0.f;
  for (int t0 = warp * 32; t0 < len; t0 += 128) {
    const int t = t0 + lane;
    int page = -1;
    if (t < len) page = a.table[(int64_t)b * a.width + t / a.block];
    const bool ok = t < len && VO_DCHECK(page >= 0 && page < a.pages);  // out-of-pool pages read as zeros
    float sc = t < len ? 0.f : -INFINITY, vsc = 0.f;
    int64_t row = 0;
    if (ok) {
      row = (((int64_t)page * a.Hk + kh) * a.block + t % a.block) * hd;
      vsc = a.vs[(int64_t)page * a.Hk + kh];
      float d = 0.f;
      for (int c = 0; c < hd; c += 8) {
        float f[8];
        p8::unpack_e4m3x8(*reinterpret_cast<const uint2*>(a.kp + row + c), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) d = fmaf(qs[c + i], f[i], d);
      }
      sc = d * a.ks[(int64_t)page * a.Hk + kh];
    }
    const float mn = fmaxf(m, warp_max(sc));
    // mn stays -inf only while every score so far is -inf or NaN: NaN then spreads through p
    const float al = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float p = sc == -INFINITY ? 0.f : exp2f(sc - (mn == -INFINITY ? 0.f : mn));
    l = l * al + warp_sum(p);
    m = mn;
#pragma unroll
    for (int j = 0; j < kMaxHd / 32; ++j) acc[j] *= al;
    const int nk = min(32, len - t0);
    for (int k = 0; k < nk; ++k) {
      const float pk = __shfl_sync(0xffffffffu, p, k), vk = __shfl_sync(0xffffffffu, vsc, k);
      const int64_t rk = __shfl_sync(0xffffffffu, row, k);
      if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, k)) continue;
#pragma unroll
      for (int j = 0; j < kMaxHd / 32; ++j) {
        const int d = lane + 32 * j;
        if (d < hd) acc[j] = fmaf(pk, p8::e4m3_to_float(a.vp[rk + d]) * vk, acc[j]);
      }
    }
  }
  if (lane == 0) {
    ml[warp][0] = m;
    ml[warp][1] = l;
  }
#pragma unroll
  for (int j = 0; j < kMaxHd / 32; ++j)
    if (lane + 32 * j < hd) os[warp][lane + 32 * j] = acc[j];
  __syncthreads();
  const float top = fmaxf(fmaxf(ml[0][0], ml[1][0]), fmaxf(ml[2][0], ml[3][0]));
  float w[4], total = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = top == -INFINITY ? 1.f : exp2f(ml[i][0] - top);
    total += w[i] * ml[i][1];
  }
  for (int i = threadIdx.x; i < hd; i += 128) {
    const float o = w[0] * os[0][i] + w[1] * os[1][i] + w[2] * os[2][i] + w[3] * os[3][i];
    out[i] = f2bf(total == 0.f ? 0.f : o / total);
  }
}

const uint8_t* bytes_of(const torch::Tensor& t) { return reinterpret_cast<const uint8_t*>(t.data_ptr()); }
const __nv_bfloat16* bf_of(const torch::Tensor& t) { return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr()); }

// 8-value vector loads of a [.., .., .., hd] bf16 tensor: last dim contiguous, every row on a 16-byte boundary
bool rows_ok(const torch::Tensor& t) {
  return t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// the tensor itself, or a copy that satisfies rows_ok (a contiguous one may still start off a 16-byte boundary; dimensions of
// one element keep their strides, which are not used)
torch::Tensor vector_rows(torch::Tensor t) {
  if (rows_ok(t)) return t;
  t = t.contiguous();
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

void check_i32(const torch::Tensor& t, const char* name, int64_t n, const torch::Tensor& like) {
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kInt32 && t.dim() == 1 && t.size(0) == n && t.is_contiguous() &&
                        t.device() == like.device(),
                    name, ": contiguous int32 [", std::to_string(n), "] on the pools' device");
}

void check_pools(const torch::Tensor& kp, const torch::Tensor& vp, const torch::Tensor& ks, const torch::Tensor& vs,
                 const torch::Tensor& table, int64_t B) {
  TORCH_CHECK_VALUE(kp.dim() == 4 && kp.scalar_type() == torch::kFloat8_e4m3fn && kp.is_contiguous() && kp.is_cuda(),
                    "k_pool: contiguous float8_e4m3fn [pages, kv_heads, block, head_dim]");
  TORCH_CHECK_VALUE(vp.sizes() == kp.sizes() && vp.scalar_type() == kp.scalar_type() && vp.is_contiguous() &&
                        vp.device() == kp.device(),
                    "v_pool: like k_pool");
  const int64_t hd = kp.size(3);
  TORCH_CHECK_VALUE(hd % 16 == 0 && hd >= 16 && hd <= kMaxHd, "head_dim: a multiple of 16 up to ", std::to_string(kMaxHd), ", got ", std::to_string(hd));
  TORCH_CHECK_VALUE(kp.size(0) >= 1 && kp.size(1) >= 1 && kp.size(2) >= 1 && kp.size(0) < (1 << 30) && kp.size(2) < (1 << 24),
                    "empty or oversized pool");
  TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(kp.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(vp.data_ptr()) % 16 == 0,
                    "pools start on 16-byte boundaries");
  for (const auto* s : {&ks, &vs})
    TORCH_CHECK_VALUE(s->dim() == 2 && s->size(0) == kp.size(0) && s->size(1) == kp.size(1) &&
                          s->scalar_type() == torch::kFloat32 && s->is_contiguous() && s->device() == kp.device(),
                      "scales: contiguous float32 [pages, kv_heads]");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == B && table.scalar_type() == torch::kInt32 &&
                        table.is_contiguous() && table.device() == kp.device(),
                    "block_table: contiguous int32 [batch, max_pages]");
}

}  // namespace

// k / v [B, Hk, S, hd] bf16 -> rows [start[b] + offset, + counts[b]) of the sequences' pages.
void paged8_append(torch::Tensor k, torch::Tensor v, torch::Tensor kp, torch::Tensor vp, torch::Tensor ks, torch::Tensor vs,
                   torch::Tensor table, torch::Tensor start, c10::optional<torch::Tensor> counts, int64_t offset) {
  TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes(), "k, v: [batch, kv_heads, tokens, head_dim]");
  TORCH_CHECK_VALUE(k.scalar_type() == torch::kBFloat16 && v.scalar_type() == torch::kBFloat16 && k.is_cuda() &&
                        v.device() == k.device() && kp.device() == k.device(),
                    "k, v: bfloat16 on the pools' device");
  const int64_t B = k.size(0), Hk = k.size(1), S = k.size(2), hd = k.size(3);
  check_pools(kp, vp, ks, vs, table, B);
  TORCH_CHECK_VALUE(kp.size(1) == Hk && kp.size(3) == hd, "k, v: kv_heads and head_dim of the pools");
  check_i32(start, "start", B, kp);
  const int* cnt = nullptr;
  if (counts.has_value() && counts->defined()) {
    check_i32(*counts, "counts", B, kp);
    cnt = counts->data_ptr<int>();
  }
  TORCH_CHECK_VALUE(S < (1 << 30) && Hk <= 65535 && offset >= 0 && offset < (1 << 30), "tokens, kv_heads or offset out of range");
  if (B == 0 || S == 0) return;
  c10::cuda::CUDAGuard g(k.device());
  k = vector_rows(k);
  v = vector_rows(v);
  const int block = (int)kp.size(2);
  const int touched = (int)((S + block - 2) / block + 1);
  TORCH_CHECK_VALUE(B * touched < (1ll << 31), "batch x pages out of range");
  AppendArgs a{bf_of(k), bf_of(v), k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2),
               const_cast<uint8_t*>(bytes_of(kp)), const_cast<uint8_t*>(bytes_of(vp)), ks.data_ptr<float>(), vs.data_ptr<float>(),
               table.data_ptr<int>(), start.data_ptr<int>(), cnt, (int)table.size(1), (int)kp.size(0), (int)B, (int)Hk, (int)S,
               (int)hd, block, (int)offset, touched};
  // as many threads as keep the new rows of a page in registers, a warp at least
  const int64_t most = std::min<int64_t>(S, block) * (hd / 8);
  int threads = 32;
  while (threads < kAppendMax && most > threads * kHeld) threads *= 2;
  append_kernel<<<dim3((unsigned)(B * touched), (unsigned)Hk, 2), threads, 0, stream()>>>(a);
  VO_CUDA_OK(cudaGetLastError());
  count_launch();
}

// pools [layers, pages, ...]: page dst[i] of every layer becomes a copy of page src[i]; one launch.
void copy_pages(std::vector<torch::Tensor> pools, torch::Tensor src, torch::Tensor dst) {
  TORCH_CHECK_VALUE(!pools.empty() && pools.size() <= kMaxPools, "copy_pages: 1 to ", std::to_string(kMaxPools), " pools");
  CopyArgs a{};
  const torch::Tensor& p0 = pools[0];
  TORCH_CHECK_VALUE(p0.is_cuda() && p0.dim() >= 2 && p0.size(1) < (1ll << 31), "copy_pages: pools [layers, pages, ...] on a GPU");
  for (size_t i = 0; i < pools.size(); ++i) {
    const torch::Tensor& p = pools[i];
    TORCH_CHECK_VALUE(p.dim() >= 2 && p.size(0) == p0.size(0) && p.size(1) == p0.size(1) && p.is_contiguous() &&
                          p.device() == p0.device(),
                      "copy_pages: contiguous pools [layers, pages, ...] with the same layers and pages");
    a.base[i] = const_cast<uint8_t*>(bytes_of(p));
    a.page_bytes[i] = p.stride(1) * p.element_size();
    a.layer_bytes[i] = p.stride(0) * p.element_size();
    const uint64_t al = reinterpret_cast<uint64_t>(a.base[i]) | (uint64_t)a.page_bytes[i] | (uint64_t)a.layer_bytes[i];
    a.vec[i] = al % 16 == 0 ? 16 : al % 4 == 0 ? 4 : 1;
  }
  check_i32(src, "src", src.numel(), p0);
  check_i32(dst, "dst", src.numel(), p0);
  const int64_t n = src.numel(), layers = p0.size(0);
  if (n == 0 || layers == 0 || p0.numel() == 0) return;
  TORCH_CHECK_VALUE(n < (1ll << 31) && layers <= 65535, "copy_pages: too many pairs or layers");
  c10::cuda::CUDAGuard g(p0.device());
  a.src = src.data_ptr<int>();
  a.dst = dst.data_ptr<int>();
  a.pages = (int)p0.size(1);
  copy_pages_kernel<<<dim3((unsigned)n, (unsigned)layers, (unsigned)pools.size()), 256, 0, stream()>>>(a);
  VO_CUDA_OK(cudaGetLastError());
  count_launch();
}

int64_t paged8_error(bool reset) {
  const int few = paged8_decode_error(reset), many = paged8_chunk_error(reset);
  return few ? few : many;
}

// q [B, Hq, S, hd] bf16 -> [B, S, Hq, hd]: query token i of sequence b stands at position
// lens[b] + len_add - q_lens[b] + i and attends to the cached rows up to its own; rows past q_lens[b] and
// rows without a key are zero.
torch::Tensor paged8_attend(torch::Tensor q, torch::Tensor kp, torch::Tensor vp, torch::Tensor ks, torch::Tensor vs,
                            torch::Tensor table, torch::Tensor lens, c10::optional<torch::Tensor> q_lens, double scale,
                            int64_t len_add) {
  TORCH_CHECK_VALUE(q.dim() == 4 && q.scalar_type() == torch::kBFloat16 && q.is_cuda() && q.device() == kp.device(),
                    "q: bfloat16 [batch, q_heads, tokens, head_dim] on the pools' device");
  const int64_t B = q.size(0), Hq = q.size(1), S = q.size(2), hd = q.size(3);
  check_pools(kp, vp, ks, vs, table, B);
  const int64_t Hk = kp.size(1);
  TORCH_CHECK_VALUE(kp.size(3) == hd && Hq >= 1 && Hq % Hk == 0, "q: head_dim of the pools, q_heads a multiple of kv_heads");
  check_i32(lens, "lens", B, kp);
  const int* ql = nullptr;
  if (q_lens.has_value() && q_lens->defined()) {
    check_i32(*q_lens, "q_lens", B, kp);
    ql = q_lens->data_ptr<int>();
  }
  TORCH_CHECK_VALUE(len_add >= 0 && len_add < (1 << 30) && S < (1 << 30), "tokens or length offset out of range");
  c10::cuda::CUDAGuard g(q.device());
  auto out = torch::empty({B, S, Hq, hd}, q.options());
  if (out.numel() == 0) return out;
  q = vector_rows(q);
  TORCH_CHECK_VALUE(B * S * Hq < (1ll << 31), "batch x tokens x heads out of range");
  p8::AttendArgs a{bf_of(q), q.stride(0), q.stride(1), q.stride(2), bytes_of(kp), bytes_of(vp), ks.data_ptr<float>(),
                   vs.data_ptr<float>(), table.data_ptr<int>(), lens.data_ptr<int>(), ql,
                   reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), (int)table.size(1), (int)kp.size(0), (int)kp.size(2), (int)B,
                   (int)Hq, (int)Hk, (int)(Hq / Hk), (int)S, (int)hd, (int)len_add, (float)(scale * 1.4426950408889634)};
  // Few rows: bound by the cache's bytes, the kernel with keys as the products' M.  Many: bound by arithmetic, rows as M.
  // Head widths and page sizes outside both: the CUDA-core kernel.
  const bool few = paged8_decode_ok(a);
  if (few || paged8_chunk_ok(a)) {
    const int sms = num_sms();
    auto ws = torch::empty({few ? paged8_decode_workspace(a, sms) : paged8_chunk_workspace(a, sms)}, q.options().dtype(torch::kUInt8));
    int launches = 0;
    const int rc = (few ? paged8_decode_launch : paged8_chunk_launch)(a, ws.data_ptr(), sms, stream(), &launches);
    TORCH_CHECK(rc == 0, "8-bit attention launch failed: ", std::to_string(rc));
    count_launch(launches);
    return out;
  }
  attend_any_kernel<<<(unsigned)(B * S * Hq), 128, 0, stream()>>>(a);
  VO_CUDA_OK(cudaGetLastError());
  count_launch();
  return out;
}

}  // namespace vo
