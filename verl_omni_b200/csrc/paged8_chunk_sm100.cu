// Attention over the 8-bit paged KV cache for many query rows (chunks of a prompt, verification of several tokens, wide
// head groups), on tcgen05.
//
// Here the bound is arithmetic: the exponentials and the two products of rows x keys.  Query rows (token, head of the KV
// group) are the M of both products, 256 rows a CTA in two tiles of 128; keys and values become f16 once per 256 rows:
// every e4m3 number is an f16 number, and the page scales enter as code * scale / (largest scale of the CTA's key range)
// (powers of two: exact down to 2^-24 of it; other scales to 11 bits).  Probabilities are f16 too (11 bits), kept in tensor
// memory over the scores they come from; queries are brought to [2^7, 2^9) by a power of two per row, exact for bf16.
// Running maximum with a lazy rescale of the output (only when it grows by more than 2^8), fp32 sums.  Probabilities are
// held times 2^7, up to 2^15 with the laziness: they keep 11 bits down to 2^-21 of the maximum and 8 down to 2^-24, below in
// steps of 2^-31.
// Work: as in the kernel for few rows, the 128-key tiles of all (sequence, KV head, 256 rows) items form one line split
// evenly over one CTA per SM; causal items are as long as their last row's reach; cut items are merged in key order.
// Warps 0-3 and 4-7: softmax and output of row tile 0 and 1 (thread = row); 8-11 and 12-14: K and V pages -> f16 tiles in
// shared memory (the codes come by TMA, a tile ahead); 15: tensor-memory allocation, MMA issue.
// Measured (B200): 4 x 512 tokens on 8000 rows, 32 query and 4 KV heads of 128: 366 us, 710 TFLOP/s.  What bounds it is the
// chain of a tile (scores, softmax, second product): leaving out the stores of the conversion, the exponentials or half of
// either product gained 3 to 9 % each.  64-key tiles with the scores a tile ahead: 513 us.
// The loops are kept short (few unrolled copies): five roles run at once, and with everything unrolled the warps mostly
// waited for instructions.
#include <type_traits>

#include "dcheck.cuh"
#include "paged8.cuh"
#include "paged8_tc.h"
#include "per_device.h"
#include "tc8.cuh"

namespace vo {
namespace p8chk {

using namespace tc8;
using p8::AttendArgs;

constexpr int TK = 128, TR = 128, ROWS = 2 * TR;
constexpr int NTHREADS = 512;         // 16 warps of 128 registers
constexpr int NLK = 128, NLV = 96;    // threads that load and convert K, V
constexpr int KST = 1, VST = 2;       // f16 K and V tiles: a K tile is free for the next one once its scores are computed
// Buffers of per-item values between the loaders and the softmax.  Items without rows in row tile 1 come one at a time (the
// last row tile of a head; all items have a tile) or row tile 1 has none at all, so a softmax is at most two items behind
// the MMA warp, and that two tiles behind the loaders: a buffer is neither refilled nor its phase passed over before then.
constexpr int kSegs = 6;
constexpr float kLazy = 8.f;          // log2 growth of the maximum that is left in the probabilities
constexpr float kUp = 7.f;            // and log2 of what one at the maximum is held as: f16 reaches 2^16

__device__ int g_error = 0;

template <int HD>
struct Cfg {
  static constexpr int TILE = TK * HD * 2;  // f16 K, V or Q tile: HD / 64 groups of 64 columns, 128 rows of 128 bytes
  static constexpr int K_OFF = 2 * TILE;
  static constexpr int V_OFF = K_OFF + KST * TILE;
  static constexpr int RAW = TK * HD;
  static constexpr int RAW_OFF = V_OFF + VST * TILE;
  static constexpr int NAN_OFF = RAW_OFF + 2 * RAW;  // [kSegs][HD] first key with a NaN value per column
  static constexpr int REF_OFF = NAN_OFF + kSegs * HD * 4;  // [kSegs][2] largest scales, then 4 + 4 partial maxima
  static constexpr int QUP_OFF = REF_OFF + kSegs * 8 + 32;  // [ROWS] row factors of the queries
  static constexpr int BAR_OFF = QUP_OFF + ROWS * 4;
  static constexpr int NBARS = 2 * KST + 2 * VST + 8 + 2 * kSegs + 2;
  static constexpr int START_OFF = BAR_OFF + NBARS * 8;  // tmem slot, abort flag, start item, scan sums
  static constexpr int BYTES = START_OFF + 24 + 8 * 16 + 1024;
};

// What the merge needs of border c (between CTA c - 1 and CTA c): parts > 0 where it is the first border inside an item.
struct Border {
  int b, kh, rt, parts;  // the item, the CTAs that hold parts of it
};

struct Params {
  AttendArgs a;
  int RT;          // row tiles (256) of a (sequence, KV head)
  float* part_o;   // [G][2][ROWS][HD]
  float* part_ml;  // [G][2][ROWS][2]
  Border* border;  // [G]
};

// tiles of row tile rt of sequence b: up to the last key that its last query token sees (one masked tile where none is)
__device__ __forceinline__ int tiles_of(const AttendArgs& a, int len, int nq, int rt) {
  const int last = min((int)(((int64_t)rt * ROWS + ROWS - 1) / a.rep), nq - 1);
  if ((int64_t)rt * ROWS >= (int64_t)nq * a.rep) return 1;
  const int lim = len - nq + last + 1;
  return lim > 0 ? (lim - 1) / TK + 1 : 1;
}

struct Walk {
  int b, kh, rt, tile, nt, len, nq;
};
__device__ __forceinline__ void enter_seq(Walk& w, const AttendArgs& a) {
  const bool in = w.b < a.B;
  w.len = in ? p8::seq_len(a, w.b) : 0;
  w.nq = in ? p8::seq_q(a, w.b) : 0;
}
__device__ __forceinline__ void next_item(Walk& w, const Params& p) {
  w.tile = 0;
  if (++w.rt == p.RT) {
    w.rt = 0;
    if (++w.kh == p.a.Hk) {
      w.kh = 0;
      ++w.b;
      enter_seq(w, p.a);
    }
  }
  w.nt = tiles_of(p.a, w.len, w.nq, w.rt);
}
__device__ __forceinline__ int row_lim(const AttendArgs& a, const Walk& w, int64_t row) {
  const int s = (int)(row / a.rep);
  return s < w.nq ? max(0, w.len - w.nq + s + 1) : 0;
}

// 16 bytes, or zeros without an access
__device__ __forceinline__ uint4 load16(const void* p, bool ok) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((int)ok));
  return v;
}
template <bool V>
__device__ __forceinline__ void loader_sync() {
  if (V) asm volatile("bar.sync 2, 96;" ::: "memory");
  else asm volatile("bar.sync 1, 128;" ::: "memory");
}
__device__ __forceinline__ float inv_pow2(float x) { return __int_as_float((254 << 23) - __float_as_int(x)); }
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// kind::f16 instruction descriptor with f16 operands, fp32 accumulation
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, int a_mn, int b_mn) { return idesc(M, N, a_mn, b_mn); }
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
// two fp32 lanes of one instruction: r = a s + c, s += a
__device__ __forceinline__ void ffma2(float a0, float a1, float s, float c, float& r0, float& r1) {
  asm("{\n\t.reg .b64 x, y, z, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
      "fma.rn.f32x2 r, x, y, z;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r0), "=f"(r1)
      : "f"(a0), "f"(a1), "f"(s), "f"(c));
}
__device__ __forceinline__ void fadd2(float& s0, float& s1, float a0, float a1) {
  asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "+f"(s0), "+f"(s1)
      : "f"(a0), "f"(a1));
}

template <int HD>
__global__ void __launch_bounds__(NTHREADS, 1)
    chunk8_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ Params p) {
  using C = Cfg<HD>;
  constexpr uint32_t TMEM_COLS = 512, S_COL = 0, O_COL = 256;
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  uint64_t* k_full = bars;              // [KST] f16 K tile written (NLK)
  uint64_t* k_empty = k_full + KST;     // [KST] its products done (commit)
  uint64_t* v_full = k_empty + KST;     // [VST] the same of V (NLV)
  uint64_t* v_empty = v_full + VST;     // [VST]
  uint64_t* s_full = v_empty + VST;     // [2] scores of a row tile (commit)
  uint64_t* p_full = s_full + 2;        // [2] probabilities written (4 warps)
  uint64_t* o_final = p_full + 2;       // [2] last product of an item done (commit)
  uint64_t* q_full = o_final + 2;       // [2] queries written (128)
  uint64_t* ref_full = q_full + 2;      // [kSegs] largest scales of an item known (NLK + NLV)
  uint64_t* nan_full = ref_full + kSegs;  // [kSegs] all its tiles loaded (NLV)
  uint64_t* raw_fulls = nan_full + kSegs;  // [2] codes of K, V landed (1 + tx)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::START_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* start = reinterpret_cast<int*>(tmem_slot + 2);                      // b, kh, rt, tile
  long long* sums = reinterpret_cast<long long*>(sm + C::START_OFF + 24);  // [16]
  int* nan_at = reinterpret_cast<int*>(sm + C::NAN_OFF);
  float* refs = reinterpret_cast<float*>(sm + C::REF_OFF);
  float* q_up = reinterpret_cast<float*>(sm + C::QUP_OFF);
  const AttendArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int64_t R = (int64_t)a.S * a.rep;

  if (tid == 0) {
    for (int i = 0; i < KST; ++i) mbar_init(&k_full[i], NLK), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < VST; ++i) mbar_init(&v_full[i], NLV), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4), mbar_init(&o_final[i], 1), mbar_init(&q_full[i], 128);
    for (int i = 0; i < kSegs; ++i) mbar_init(&ref_full[i], NLK + NLV), mbar_init(&nan_full[i], NLV);
    for (int i = 0; i < 2; ++i) mbar_init(&raw_fulls[i], 1);
    *abort_flag = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 15) tmem_alloc(tmem_slot, TMEM_COLS);
  // everything above is on the chip: it may run before the kernels in front have ended
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- this CTA's share of the line of tiles
  auto seq_tiles = [&](int b) {
    const int len = p8::seq_len(a, b), nq = p8::seq_q(a, b);
    long long n = 0;
    for (int rt = 0; rt < p.RT; ++rt) n += tiles_of(a, len, nq, rt);
    return n;
  };
  long long mine = 0;
  const int per = (a.B + NTHREADS - 1) / NTHREADS;
  for (int b = tid * per; b < min(a.B, (tid + 1) * per); ++b) mine += seq_tiles(b);
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < NTHREADS / 32; ++i) {
    if (i < warp) before += sums[i];
    total += sums[i];
  }
  total *= a.Hk;
  const int used = (int)min((long long)gridDim.x, total);  // CTAs with work: one tile each at least
  const bool idle = (int)blockIdx.x >= used;
  const long long g0 = idle ? total : total * blockIdx.x / used, g1 = idle ? total : total * (blockIdx.x + 1) / used;
  long long lo = (before + upto - mine) * a.Hk;
  if (idle && tid == 0) p.border[blockIdx.x] = Border{0, 0, 0, 0};
  if (g0 >= lo && g0 < lo + mine * a.Hk) {
    for (int b = tid * per;; ++b) {
      const long long n = seq_tiles(b);
      if (g0 < lo + n * a.Hk) {
        const int kh = (int)((g0 - lo) / n), len = p8::seq_len(a, b), nq = p8::seq_q(a, b);
        lo += n * kh;
        int rt = 0, nt = tiles_of(a, len, nq, 0);
        while (g0 >= lo + nt) {
          lo += nt;
          nt = tiles_of(a, len, nq, ++rt);
        }
        start[0] = b;
        start[1] = kh;
        start[2] = rt;
        start[3] = (int)(g0 - lo);
        // the item's tiles [lo, lo + nt); tile g lies in CTA ((g + 1) used - 1) / total
        const int from = (int)(((lo + 1) * used - 1) / total), to = (int)(((lo + nt) * used - 1) / total);
        p.border[blockIdx.x] = Border{b, kh, rt, lo < g0 && from == (int)blockIdx.x - 1 ? to - from + 1 : 0};
        break;
      }
      lo += n * a.Hk;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  // the merge kernel's CTAs may take free places now; they wait for this grid's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int ntot = (int)(g1 - g0);
  Walk w;  // a CTA without tiles walks nothing
  w.b = idle ? a.B : start[0];
  w.kh = start[1];
  w.rt = start[2];
  w.tile = start[3];
  enter_seq(w, a);
  w.nt = tiles_of(a, w.len, w.nq, w.rt);

  // ------------------------------------------------------------------ pages -> f16 tiles (K or V)
  auto loader = [&](auto is_v) {
    constexpr bool V = decltype(is_v)::value;
    constexpr int NT = V ? NLV : NLK, ST = V ? VST : KST;
    constexpr int NC = HD / 16;            // 16-byte pieces of a row
    constexpr int RP = NT / NC;            // rows of a pass
    constexpr int NI = (TK + RP - 1) / RP;  // passes: row i * RP + lt / NC (V: the last one partly empty)
    const int lt = tid - (V ? 256 + NLK : 256), lw = lt >> 5;
    const int r_in = lt / NC, c = lt % NC;
    const int blk = min(a.block, TK), nblk = TK / blk;
    const float* sc = V ? a.vs : a.ks;
    const CUtensorMap* map = V ? &mv : &mk;
    uint64_t *raw_full = &raw_fulls[V ? 1 : 0], *full = V ? v_full : k_full, *empty = V ? v_empty : k_empty;
    const uint8_t* codes = sm + C::RAW_OFF + (V ? C::RAW : 0);
    uint8_t* tiles = sm + (V ? C::V_OFF : C::K_OFF);
    // the tile that is loaded next, by lane: rows [8 l, 8 l + 8) for lanes l and l + 16
    int id_n = -1, off_n = 0, kh_n = 0;  // page, first row inside it, KV head
    auto fetch = [&](const Walk& x) {
      const int t = x.tile * TK + (lane & 15) * 8;
      kh_n = x.kh;
      id_n = t < x.len ? __ldg(a.table + (int64_t)x.b * a.width + t / a.block) : -1;
      off_n = t % a.block;
    };
    constexpr float kNoPage = -1.f;
    auto scale_of_page = [&](int kh, int id) { return id >= 0 && id < a.pages ? __ldg(sc + (int64_t)id * a.Hk + kh) : kNoPage; };
    int started = 0;  // tiles whose copies were started
    // starts its copies (the role's first warp, lane = page) and reads its scale.  Nothing is started where
    // the tile before was given up (landed false): its copies may still be on their way to the same place
    auto start_tile = [&](bool landed) {
      const int base = id_n >= 0 && id_n < a.pages ? (id_n * a.Hk + kh_n) * a.block + off_n : -1;
      if (lw == 0 && __all_sync(0xffffffffu, landed)) {
        const int row = __shfl_sync(0xffffffffu, base, (lane * blk >> 3) & 15);
        const bool load = lane < nblk && row >= 0;
        const unsigned n = __popc(__ballot_sync(0xffffffffu, load));
        if (lane == 0) mbar_expect_tx(raw_full, n * blk * HD);
        __syncwarp();
        if (load) tma_load_2d(smem_u32(codes) + lane * blk * HD, map, raw_full, 0, row);
        ++started;
      }
      return scale_of_page(kh_n, id_n);
    };
    // code * scale / ref in f16, 64-column groups of swizzled 128-byte rows; rows from n on and rows without a page (a
    // negative factor; one that is zero in f16 still leaves NaN) are zero.  The two halves of a piece are written in the other order in the odd groups, so that a row's eight lanes
    // hit different banks.  nan: first keys with a NaN per column are noted and the value left out.
    auto convert = [&](uint8_t* dst, int n, float factor, int* nan, int t0) {
      const __half2 mine_f = __float2half2_rn(factor);
      const int grp = c >> 2, i0 = (c & 3) * 2;
      const bool odd = grp & 1;
      uint8_t* base = dst + grp * (TK * 128);
      constexpr int NB = 4;  // pieces in flight
#pragma unroll 1
      for (int b0 = 0; b0 < NI; b0 += NB) {
        uint32_t fs[NB];
        uint4 d[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int r = (b0 + i) * RP + r_in;
          fs[i] = __shfl_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&mine_f), (r >> 3) & 15);
          d[i] = *reinterpret_cast<const uint4*>(codes + min(r, TK - 1) * HD + c * 16);
          if (r >= min(n, TK) || (fs[i] & 0x8000u)) d[i] = make_uint4(0, 0, 0, 0);
        }
        if (V && nan != nullptr) {
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            uint32_t* u = reinterpret_cast<uint32_t*>(&d[i]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if ((((u[q] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) == 0) continue;
              for (int by = 0; by < 4; ++by)
                if (((u[q] >> (8 * by)) & 0x7f) == 0x7f) {
                  atomicMin(&nan[c * 16 + q * 4 + by], t0 + (b0 + i) * RP + r_in);
                  u[q] &= ~(0xffu << (8 * by));
                }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int r = (b0 + i) * RP + r_in;
          const uint32_t u[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
          const __half2 f = *reinterpret_cast<const __half2*>(&fs[i]);
          uint32_t h[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2((uint16_t)(j & 1 ? u[j >> 1] >> 16 : u[j >> 1] & 0xffff), __NV_E4M3);
            const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&x), f);
            h[j] = *reinterpret_cast<const uint32_t*>(&y);
          }
          const uint4 h0 = make_uint4(h[0], h[1], h[2], h[3]), h1 = make_uint4(h[4], h[5], h[6], h[7]);
          if (r < TK) {
            *reinterpret_cast<uint4*>(base + swz<128>(r, odd ? i0 + 1 : i0)) = odd ? h1 : h0;
            *reinterpret_cast<uint4*>(base + swz<128>(r, odd ? i0 : i0 + 1)) = odd ? h0 : h1;
          }
        }
      }
      fence_async_smem();
    };
    int seg = 0, left = 0, common = 0, buf = 0;
    float inv_ref = 1.f, s0 = 0.f;
    if (ntot > 0) {
      fetch(w);
      s0 = start_tile(true);
    }
    for (int i = 0; i < ntot; ++i) {
      if (left == 0) {
        // largest scale over this item's part: the f16 numbers are relative to it
        left = min(w.nt - w.tile, ntot - i);
        buf = seg % kSegs;
        const int p0 = w.tile * TK / a.block, p1 = (min(w.len, (w.tile + left) * TK) + a.block - 1) / a.block;
        float m = 0.f;
        for (int x = p0 + lt; x < p1; x += NT) m = fmaxf(m, scale_of_page(w.kh, __ldg(a.table + (int64_t)w.b * a.width + x)));
        m = warp_fmax(m);
        float* pm = refs + 2 * kSegs + (V ? 4 : 0);
        loader_sync<V>();  // the maxima of the item before have been read
        if (lane == 0) pm[lw] = m;
        loader_sync<V>();
        m = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], V ? 0.f : pm[3]));
        m = m > 0.f ? m : 1.f;
        inv_ref = 1.f / m;
        common = max(1, w.len - w.nq + (int)((int64_t)w.rt * ROWS / a.rep) + 1);  // keys below: seen by every row that sees any
        // buffers seg % kSegs were last read by the softmax several items ago: this wait is past that
        mbar_wait(&empty[i % ST], ((i / ST) & 1) ^ 1, abort_flag, &g_error, V ? 26 : 21);
        if (V)
          for (int x = lt; x < HD; x += NT) nan_at[buf * HD + x] = 0x7fffffff;
        if (lt == 0) refs[buf * 2 + (V ? 1 : 0)] = m;
        loader_sync<V>();
        mbar_arrive(&ref_full[buf]);
        ++seg;
      }
      const int t0 = w.tile * TK, n = V ? w.len - t0 : TK;  // K: rows past the length too, their scores are masked
      if (--left == 0) next_item(w, p);
      else ++w.tile;
      if (i + 1 < ntot) fetch(w);
      const bool landed = mbar_wait(raw_full, i & 1, abort_flag, &g_error, V ? 25 : 24);
      mbar_wait(&empty[i % ST], ((i / ST) & 1) ^ 1, abort_flag, &g_error, V ? 23 : 22);
      // V: where some row sees only part of the tile, a NaN value must not reach it through 0 * NaN
      convert(tiles + (i % ST) * C::TILE, n, s0 * inv_ref, V && t0 + TK > common ? nan_at + buf * HD : nullptr, t0);
      mbar_arrive(&full[i % ST]);
      loader_sync<V>();  // every loader has read the codes: their place is refilled
      if (i + 1 < ntot) s0 = start_tile(landed);
      if (V && left == 0) mbar_arrive(&nan_full[buf]);
    }
    if (*abort_flag && lt == 0 && started > 0) mbar_drain(raw_full, (started - 1) & 1);  // copies in flight land before the CTA leaves
  };
  if (warp >= 8 && warp < 12) {
    loader(std::false_type{});
  } else if (warp >= 12 && warp < 15) {
    loader(std::true_type{});
  } else if (warp == 15) {
    // ------------------------------------------------------------------ MMA issuer
    {
      const int e = lane == 0;
      constexpr uint32_t id_s = idesc_f16(128, 128, 0, 0), id_o = idesc_f16(128, HD, 0, 1);
      const uint32_t base = smem_u32(sm), tm = (uint32_t)uniform((int)tmem);
      const int ntot_u = uniform(ntot);
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      auto track = [&](uint64_t* b, uint32_t par) {
        commit(b, e);
        last_bar = b;
        last_par = par;
      };
      uint32_t ns = 0, nq = 0;  // parities of a row tile's score tiles and items, bit = row tile
      const uint64_t q_desc = desc<128>(base, 16, 1024), k_desc = desc<128>(base + C::K_OFF, 16, 1024),
                     v_desc = desc<128>(base + C::V_OFF, TK * 128, 1024);
      auto issue_s = [&](int t, int i) {
        const uint64_t q = q_desc + ((t * C::TILE) >> 4), k = k_desc + (((i % KST) * C::TILE) >> 4);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          constexpr uint32_t kGroup = TK * 128 >> 4;  // descriptors count 16-byte units
          const uint32_t off = (kk >> 2) * kGroup + (kk & 3) * 2;
          mma_f16_ss(tm + S_COL + t * 128, q + off, k + off, id_s, kk > 0, e);
        }
        track(&s_full[t], (ns >> t) & 1);
        ns ^= 1u << t;
      };
      auto issue_pv = [&](int t, int i, bool first) {
        const uint64_t v = v_desc + (((i % VST) * C::TILE) >> 4);
#pragma unroll
        for (int kk = 0; kk < TK / 16; ++kk)
          mma_f16_ts(tm + O_COL + t * HD, tm + S_COL + t * 128 + kk * 8, v + kk * (2048 >> 4), id_o, !first || kk > 0, e);
      };
      bool ok = true;
      int i = 0;
      while (ok && i < ntot_u) {
        const int n = uniform(min(w.nt - w.tile, ntot_u - i));
        const int nt = uniform((int64_t)w.rt * ROWS + TR < R ? 2 : 1);  // row tiles with rows
        ok = mbar_wait_warp(&k_full[i % KST], (i / KST) & 1, abort_flag, &g_error, 33);
#pragma unroll 1
        for (int t = 0; ok && t < nt; ++t) {
          ok = mbar_wait_warp(&q_full[t], (nq >> t) & 1, abort_flag, &g_error, 31);
          if (!ok) break;
          fence_after();
          issue_s(t, i);
        }
        if (!ok) break;
        track(&k_empty[i % KST], (i / KST) & 1);
        for (int j = 0; ok && j < n; ++j, ++i) {
          const bool more = j + 1 < n;
          ok = mbar_wait_warp(&v_full[i % VST], (i / VST) & 1, abort_flag, &g_error, 34);
#pragma unroll 1
          for (int t = 0; ok && t < nt; ++t) {
            ok = mbar_wait_warp(&p_full[t], ((ns >> t) & 1) ^ 1, abort_flag, &g_error, 35);  // of the score tile issued last
            if (!ok) break;
            fence_after();
            issue_pv(t, i, j == 0);
            if (t + 1 == nt) track(&v_empty[i % VST], (i / VST) & 1);
            if (more) {
              if (t == 0) ok = mbar_wait_warp(&k_full[(i + 1) % KST], ((i + 1) / KST) & 1, abort_flag, &g_error, 36);
              if (!ok) break;
              fence_after();
              issue_s(t, i + 1);
              if (t + 1 == nt) track(&k_empty[(i + 1) % KST], ((i + 1) / KST) & 1);
            } else {
              track(&o_final[t], (nq >> t) & 1);
            }
          }
        }
        nq ^= nt == 2 ? 3u : 1u;
        next_item(w, p);
      }
      if (last_bar) mbar_drain(last_bar, last_par);
    }
    __syncwarp();
  } else if (warp < 8) {
    // ------------------------------------------------------------------ softmax and output of one row tile
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t S_t = tmem + S_COL + t * 128 + lane_off, O_t = tmem + O_COL + t * HD + lane_off;
    const float sgn = a.scale_log2 < 0.f ? -1.f : 1.f;
    int it = 0, seg = 0, ns = 0, nitem = 0;
    auto load_queries = [&](const Walk& x) {
      // queries in f16, times 2^-e per row: the warp's 32 rows, HD / 8 lanes a row
      constexpr int LPR = HD / 8, RPI = 32 / LPR;
      const int c = lane % LPR;
      const int r0 = x.rt * ROWS + t * TR + (warp & 3) * 32 + lane / LPR;
#pragma unroll 1
      for (int b0 = 0; b0 < LPR; b0 += 4) {
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = r0 + (b0 + i) * RPI;
          const bool has = r < R;
          const int s = has ? r / a.rep : 0, h = x.kh * a.rep + (has ? r % a.rep : 0);
          u[i] = load16(a.q + x.b * a.qsb + h * a.qsh + s * a.qss + c * 8, has);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rl = (warp & 3) * 32 + lane / LPR + (b0 + i) * RPI;  // row of the tile
          const uint32_t q4[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
          // the bits of |q| order like the numbers; infinities and NaN lie above all finite ones
          uint32_t mb = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) mb = __vmaxu2(mb, q4[k] & 0x7fff7fffu);
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) mb = __vmaxu2(mb, __shfl_xor_sync(0xffffffffu, mb, o));
          mb = max(mb & 0xffffu, mb >> 16);
          const bool finite = mb < 0x7f80u;
          const float up = !finite || mb == 0 ? 1.f : p8::scale_of(__uint_as_float(mb << 16)), inv = sgn * inv_pow2(up);
          uint32_t h[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            h[k] = finite ? pack_f16(__uint_as_float(q4[k] << 16) * inv, __uint_as_float(q4[k] & 0xffff0000u) * inv) : 0u;
          *reinterpret_cast<uint4*>(sm + t * C::TILE + (c >> 3) * (TK * 128) + swz<128>(rl, c & 7)) = make_uint4(h[0], h[1], h[2], h[3]);
          // an infinity or NaN in the query: its scores are NaN
          if (c == 0) q_up[t * TR + rl] = finite ? up : __int_as_float(0x7fffffff);
        }
      }
      fence_async_smem();
      mbar_arrive(&q_full[t]);
      __syncwarp();
    };
    // items without rows in this tile: nothing is issued for it
    auto skip = [&] {
      while (it < ntot && (int64_t)w.rt * ROWS + t * TR >= R) {
        it += min(w.nt - w.tile, ntot - it);
        ++seg;
        next_item(w, p);
      }
    };
    skip();
    if (it < ntot) load_queries(w);
    while (it < ntot) {
      const int n = min(w.nt - w.tile, ntot - it), item = seg, buf = item % kSegs;
      const Walk cur = w;
      const int64_t rr = (int64_t)w.rt * ROWS + t * TR + row;  // row among the (token, head) rows of the KV head
      it += n;
      ++seg;
      next_item(w, p);
      const int lim_row = rr < R ? row_lim(a, cur, rr) : 0;
      mbar_wait(&ref_full[buf], (item / kSegs) & 1, abort_flag, &g_error, 41);
      float sl2 = sgn * a.scale_log2 * q_up[t * TR + row] * refs[buf * 2];
      if (sl2 == 0.f || lim_row == 0) sl2 = 1e-37f;  // keeps masked scores at -inf
      const float vref = refs[buf * 2 + 1];
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j, ++ns) {
        const int t0 = (cur.tile + j) * TK;
        const int lim = max(0, min(TK, lim_row - t0));  // this row sees keys [t0, t0 + lim) of the tile
        mbar_wait(&s_full[t], ns & 1, abort_flag, &g_error, 42);
        __syncwarp();
        fence_after();
        float mx = -INFINITY;
        auto scores = [&](int g, uint32_t(&x)[32], uint32_t(&y)[32]) {  // 64 of them, -inf where the row does not see the key
          ld_nowait(S_t + g * 64, x);
          ld_nowait(S_t + g * 64 + 32, y);
          wait_ld();
          if (lim < (g + 1) * 64) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              x[i] = g * 64 + i < lim ? x[i] : 0xff800000u;
              y[i] = g * 64 + 32 + i < lim ? y[i] : 0xff800000u;
            }
          }
        };
#pragma unroll 1
        for (int g = 0; g < 2; ++g) {
          uint32_t x[32], y[32];
          scores(g, x, y);
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, fmaxf(__uint_as_float(x[i]), __uint_as_float(y[i])));
        }
        const float m_blk = mx * sl2;
        float alpha = 1.f;
        const bool move = m_blk > m + kLazy || (m == -INFINITY && m_blk > -INFINITY);
        if (move) {
          alpha = m == -INFINITY ? 0.f : ex2(m - m_blk);
          m = m_blk;
        }
        if (j > 0 && __any_sync(0xffffffffu, move)) {
          // O_t is quiescent: the product before these scores is complete, the next one waits for this warp
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            ld_nowait(O_t + c * 32, o);
            wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            st32(O_t + c * 32, o);
          }
        }
        const float nmb = m == -INFINITY ? 0.f : kUp - m;
        float rs0 = 0.f, rs1 = 0.f;
#pragma unroll 1
        for (int g = 0; g < 2; ++g) {  // probabilities of 64 keys, f16 pairs over scores that have been read
          uint32_t x[32], y[32];
          scores(g, x, y);
          auto emit = [&](uint32_t(&v)[32], uint32_t at) {
            uint32_t h[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x0, x1;
              ffma2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]), sl2, nmb, x0, x1);
              const float e0 = ex2(x0), e1 = ex2(x1);
              fadd2(rs0, rs1, e0, e1);
              h[i] = pack_f16(e0, e1);
            }
            st16(at, h);
          };
          emit(x, S_t + g * 32);
          emit(y, S_t + g * 32 + 16);
        }
        wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        l = l * alpha + (rs0 + rs1);
      }
      skip();
      if (it < ntot) load_queries(w);  // this item's scores are all computed; its last products run meanwhile
      mbar_wait(&o_final[t], nitem & 1, abort_flag, &g_error, 43);
      mbar_wait(&nan_full[buf], (item / kSegs) & 1, abort_flag, &g_error, 44);
      ++nitem;
      __syncwarp();
      fence_after();
      const bool from_start = cur.tile == 0, whole = from_start && n == cur.nt;
      const float mul = whole ? (l == 0.f ? 0.f : vref / l) : vref;
      const int64_t slot = ((int64_t)blockIdx.x * 2 + (from_start ? 1 : 0)) * ROWS + t * TR + row;
      const int64_t orow = ((int64_t)cur.b * a.S + rr / a.rep) * a.Hq + cur.kh * a.rep + rr % a.rep;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        ld_nowait(O_t + c * 32, o);
        wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float f = __uint_as_float(o[i]) * mul;
          if (whole && l == 0.f) f = 0.f;  // a row without keys (a NaN among the tile's values would stay NaN)
          if (nan_at[buf * HD + c * 32 + i] < lim_row) f = __int_as_float(0x7fffffff);
          o[i] = __float_as_uint(f);
        }
        if (rr < R) {
          if (whole) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint32_t h[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 b2 = __floats2bfloat162_rn(__uint_as_float(o[g * 8 + 2 * i]), __uint_as_float(o[g * 8 + 2 * i + 1]));
                h[i] = *reinterpret_cast<const uint32_t*>(&b2);
              }
              *reinterpret_cast<uint4*>(a.out + orow * HD + c * 32 + g * 8) = make_uint4(h[0], h[1], h[2], h[3]);
            }
          } else {
#pragma unroll
            for (int g = 0; g < 8; ++g)
              *reinterpret_cast<uint4*>(p.part_o + slot * HD + c * 32 + g * 4) = make_uint4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
          }
        }
      }
      if (!whole && rr < R) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m, l);
      fence_before();
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 15) {
    __syncwarp();
    tmem_free(tmem, TMEM_COLS);
  }
}

// Merges the partials of items that CTA borders cut; blocks (c, 8 rows), a warp per row, in the order of the keys.
template <int HD>
__global__ void __launch_bounds__(256) merge8_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const AttendArgs& a = p.a;
  const int c = blockIdx.x + 1, lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
  const Border me = p.border[c];
  if (me.parts == 0) return;
  const int64_t rr = (int64_t)me.rt * ROWS + r;
  if (rr >= (int64_t)a.S * a.rep) return;
  constexpr int V = HD / 32;
  float m = -INFINITY;
  auto row_of = [&](int i) -> int64_t { return i == c - 1 ? ((int64_t)i * 2 + 1) * ROWS + r : (int64_t)i * 2 * ROWS + r; };
  const int last = c - 1 + me.parts;
  for (int i = c - 1; i < last; ++i) m = fmaxf(m, p.part_ml[row_of(i) * 2]);
  float l = 0.f, o[V];
#pragma unroll
  for (int k = 0; k < V; ++k) o[k] = 0.f;
  for (int i = c - 1; i < last; ++i) {
    const int64_t x = row_of(i);
    const float w = m == -INFINITY ? 1.f : ex2(p.part_ml[x * 2] - m);
    l += p.part_ml[x * 2 + 1] * w;
#pragma unroll
    for (int k = 0; k < V; ++k) o[k] += p.part_o[x * HD + lane * V + k] * w;
  }
  const int64_t orow = ((int64_t)me.b * a.S + rr / a.rep) * a.Hq + me.kh * a.rep + rr % a.rep;
#pragma unroll
  for (int k = 0; k < V; ++k) a.out[orow * HD + lane * V + k] = __float2bfloat16_rn(l == 0.f ? 0.f : o[k] / l);
}

template <int HD>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int G, cudaStream_t stream, int* launches) {
  static PerDevice once;
  cudaError_t e = once([] { return cudaFuncSetAttribute(chunk8_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::BYTES); });
  if (e != cudaSuccess) return (int)e;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cfg.stream = stream;
  cfg.gridDim = dim3(G);
  cfg.blockDim = dim3(NTHREADS);
  cfg.dynamicSmemBytes = Cfg<HD>::BYTES;
  e = cudaLaunchKernelEx(&cfg, chunk8_kernel<HD>, mk, mv, p);
  if (e != cudaSuccess) return (int)e;
  ++*launches;
  if (G == 1) return 0;
  cfg.gridDim = dim3(G - 1, ROWS / 8);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, merge8_kernel<HD>, p);
  if (e != cudaSuccess) return (int)e;
  ++*launches;
  return 0;
}

int64_t row_tiles(const AttendArgs& a) { return ((int64_t)a.S * a.rep + ROWS - 1) / ROWS; }
int ctas(const AttendArgs& a, int sms) {
  const int64_t reach = ((int64_t)a.width * a.block + TK - 1) / TK;
  const int64_t most = (int64_t)a.B * a.Hk * row_tiles(a) * (reach < 1 ? 1 : reach);
  return (int)(most < sms ? most : sms);
}

}  // namespace p8chk

bool paged8_chunk_ok(const p8::AttendArgs& a) {
  return (a.hd == 64 || a.hd == 128) && paged8_pages_ok(a) && (int64_t)a.S * a.rep < (1ll << 30);
}

int64_t paged8_chunk_workspace(const p8::AttendArgs& a, int sms) {
  const int64_t G = p8chk::ctas(a, sms);
  return G * 2 * p8chk::ROWS * (a.hd + 2) * 4 + G * (int64_t)sizeof(p8chk::Border);
}

int paged8_chunk_launch(const p8::AttendArgs& a, void* workspace, int sms, cudaStream_t stream, int* launches) {
  using namespace p8chk;
  CUtensorMap mk, mv;
  const int64_t rows = (int64_t)a.pages * a.Hk * a.block;
  const int box = a.block < TK ? a.block : TK;
  int e = map_rows(&mk, a.kp, rows, a.hd, box, false);
  if (e) return e;
  e = map_rows(&mv, a.vp, rows, a.hd, box, false);
  if (e) return e;
  const int G = ctas(a, sms);
  Params p;
  p.a = a;
  p.RT = (int)row_tiles(a);
  p.part_o = static_cast<float*>(workspace);  // 16-byte rows first
  p.part_ml = p.part_o + (int64_t)G * 2 * ROWS * a.hd;
  p.border = reinterpret_cast<Border*>(p.part_ml + (int64_t)G * 2 * ROWS * 2);
  return a.hd == 128 ? launch<128>(mk, mv, p, G, stream, launches) : launch<64>(mk, mv, p, G, stream, launches);
}

int paged8_chunk_error(bool reset) {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, p8chk::g_error, sizeof(int)) != cudaSuccess) return -1;
  if (reset && h) {
    const int z = 0;
    cudaMemcpyToSymbol(p8chk::g_error, &z, sizeof(int));
  }
  return h;
}

}  // namespace vo
