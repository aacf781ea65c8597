// Attention over the 8-bit paged KV cache for few query rows (query tokens x heads of a KV group <= 16), on tcgen05.
//
//   o = softmax(scale q k^T) v,  k = code * k_scale[page],  v = code * v_scale[page]  (scales: powers of two)
//
// The bound is the cache's bytes: 2 * head_dim bytes per row and KV head, read once for all query heads of the group.
// The e4m3 codes go from global memory to the tensor core as they are: a 128-key tile of K and V is staged by TMA, and
// both products take it from shared memory (S^T = K Q^T: keys as M, rows as N; O^T = V^T P^T: dims as M).  The other
// operand keeps its precision as a sum of two e4m3 numbers: q = 2^e (q_hi + q_lo) holds every bit of a bf16 query whose
// elements lie within 2^13 of the row's largest (a rounding of 2^-21 of the largest below), p likewise to 8 bits; both parts
// are columns of one product (N = 2 x rows: the tile is read once for both) and are added when they are read.  The low part
// is at most 1/16 of the high one: q_lo is held times 16 and p_lo (p <= 256) times 32, so that a weight keeps its 8 bits down
// to 2^-13 of its reference, with steps of 2^-22 below.  The reference is the row's running maximum, or near the tile's own
// where that lies more than 2^4 lower: behind one key far above all others the tiles without it lose nothing.  Page scales stay
// outside: k_scale multiplies the thread's (key's) scores, the v scales of a tile enter as p * v_scale / max(v_scale) and the
// maximum as a factor of the folded output.
//
// Work: the tiles of all (sequence, KV head) items form one line that the CTAs split evenly (two CTAs per SM, as many as
// there are tiles at most), so ragged lengths balance and a long single sequence fills the GPU.  An item inside one CTA
// is finished there; one cut by a border leaves (maximum, sum, output) partials that the combine kernel merges in
// the order of the keys, so results do not depend on timing.
// Measured (B200, 8 query heads per KV head): 64 sequences x 4096 rows, 4 KV heads of 128, pages of 128: 56.4 us, the same with
// one key far above the others; its bytes alone take 41 us.  16 heads per KV head: 90 us; 2 tokens x 8 heads: 125 us.  Time grows by
// 7.0 TB/s with the rows over about 20 us (fill, item changes, merge).  Before small weights were kept 54.6 us; against that K and
// V in one ring took 57, a second softmax group taking every other tile 65 us.
// Warps 0-3: softmax (thread = key) and output (thread = head-dim column); 4: TMA producer, page ids read two tiles and
// scales one tile ahead; 5: tensor-memory allocation, MMA issue (scores one tile ahead of the softmax).
#include "dcheck.cuh"
#include "paged8.cuh"
#include "paged8_tc.h"
#include "per_device.h"
#include "tc8.cuh"

namespace vo {
namespace p8dec {

using namespace tc8;
using p8::AttendArgs;

constexpr int TK = 128;        // keys per tile
constexpr int MAXR = 16;       // query rows of an item at most
constexpr int NTHREADS = 192;
constexpr int kMaxBlocksPerTile = 16;  // pages of 8 rows
constexpr float kQLow = 16.f;          // what the high part of a query leaves (16 at most) is held times 2^4
constexpr float kPOne = 256.f;         // probabilities are held times 2^8 (e4m3 reaches 448)
constexpr float kPLow = 32.f;          // and what the high part leaves (8 at most) times 2^5
constexpr float kFar = 4.f;            // log2 distance from the running maximum to a tile's that is left in the probabilities

__device__ int g_error = 0;

template <int HD, int NR>
struct Cfg {
  static constexpr int NP = NR < 8 ? 8 : NR;            // rows of a part
  static constexpr int NB = 2 * NP;                     // MMA N: high parts, then low parts
  static constexpr int KV = TK * HD;                    // bytes of K or V of a tile
  // K and V tiles in rings of their own, 96 KB, two CTAs per SM: a K tile is free as soon as its scores are computed, a V
  // tile is held over the softmax
  static constexpr int SK = HD == 128 ? 2 : 4, SV = HD == 128 ? 4 : 8;
  static constexpr int V_OFF = SK * KV;
  static constexpr int Q_OFF = V_OFF + SV * KV;         // NB rows of HD bytes
  static constexpr int P_OFF = Q_OFF + NB * HD;         // two buffers of NB rows of TK bytes
  static constexpr int SC_OFF = P_OFF + 2 * NB * TK;    // per V tile: k and v scale of each page
  static constexpr int TV_OFF = SC_OFF + SV * 2 * kMaxBlocksPerTile * 4;       // per V tile: largest v scale, whether a page is missing, 2^8 / the former
  static constexpr int RED_OFF = TV_OFF + SV * 16;                             // [2][4][MAXR] warp maxima
  static constexpr int QS_OFF = RED_OFF + 2 * 4 * MAXR * 4;                    // [2][MAXR] row factors
  static constexpr int FOLD_OFF = QS_OFF + 2 * MAXR * 4;                       // [4][2][2][MAXR] a warp's row factors of the fold
  static constexpr int BAR_OFF = FOLD_OFF + 4 * 2 * 2 * MAXR * 4;
  static constexpr int NBARS = 2 * SK + 2 * SV + 11;
  static constexpr int START_OFF = BAR_OFF + NBARS * 8;  // tmem slot, abort flag, start item, scan sums
  static constexpr int BYTES = START_OFF + 96 + 1024;
};

// What the merge needs of border c (between CTA c - 1 and CTA c): parts > 0 where it is the first border inside an item.
struct Border {
  int item, parts;  // the item, the CTAs that hold parts of it
};

struct Params {
  AttendArgs a;
  float* part_o;   // [G][2][NR][HD]
  float* part_ml;  // [G][2][NR][2]
  Border* border;  // [G]
};

struct Walk {
  int b, kh, tile, nt, len;
};
__device__ __forceinline__ int tiles_of(int len) { return len > 0 ? (len - 1) / TK + 1 : 1; }  // an empty sequence: one masked tile
__device__ __forceinline__ void enter(Walk& w, const AttendArgs& a) {
  w.len = w.b < a.B ? p8::seq_len(a, w.b) : 0;
  w.nt = tiles_of(w.len);
}
__device__ __forceinline__ void next_item(Walk& w, const AttendArgs& a) {
  w.tile = 0;
  if (++w.kh == a.Hk) {
    w.kh = 0;
    ++w.b;
    enter(w, a);
  }
}

__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ float inv_pow2(float x) { return __int_as_float((254 << 23) - __float_as_int(x)); }

template <int HD, int NR, bool CAUSAL>
__global__ void __launch_bounds__(NTHREADS, 2)
    decode8_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const __grid_constant__ Params p) {
  using C = Cfg<HD, NR>;
  constexpr int SK = C::SK, SV = C::SV, NP = C::NP, NB = C::NB;
  constexpr uint32_t S_COL = 0, O_COL = 2 * NB, TMEM_COLS = 4 * NB;
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  uint64_t* k_full = bars;               // [SK] K tile landed (1 + tx)
  uint64_t* k_empty = k_full + SK;       // [SK] its scores computed (commit)
  uint64_t* v_full = k_empty + SK;       // [SV] V tile landed, scales written (1 + tx)
  uint64_t* v_empty = v_full + SV;       // [SV] its products done (commit)
  uint64_t* s_full = v_empty + SV;       // [2] scores in tensor memory (commit)
  uint64_t* s_empty = s_full + 2;        // [2] scores read (128)
  uint64_t* p_full = s_empty + 2;        // [2] probabilities written (128)
  uint64_t* o_full = p_full + 2;         // [2] tile output in tensor memory (commit)
  uint64_t* o_empty = o_full + 2;        // [2] tile output read (128)
  uint64_t* q_full = o_empty + 2;        // queries of the next item written (128)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::START_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* start = reinterpret_cast<int*>(tmem_slot + 2);                      // b, kh, tile of the first tile
  long long* sums = reinterpret_cast<long long*>(sm + C::START_OFF + 24);  // [6] per-warp tile counts
  float* scl = reinterpret_cast<float*>(sm + C::SC_OFF);
  float* tile_v = reinterpret_cast<float*>(sm + C::TV_OFF);
  float* red = reinterpret_cast<float*>(sm + C::RED_OFF);
  float* qsc = reinterpret_cast<float*>(sm + C::QS_OFF);
  const AttendArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;

  if (tid == 0) {
    for (int i = 0; i < SK; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < SV; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 128);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 128);
    }
    mbar_init(q_full, 128);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  }
  if (warp == 5) tmem_alloc(tmem_slot, TMEM_COLS);
  if (warp < 4)  // rows past the queries and heads stay zero for the whole kernel
    for (int u = tid; u < (C::SC_OFF - C::Q_OFF) / 16; u += 128) reinterpret_cast<uint4*>(sm + C::Q_OFF)[u] = make_uint4(0, 0, 0, 0);
  // everything above is on the chip: it may run before the kernels in front have ended
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- this CTA's share [g0, g1) of the line of tiles, and the item that holds g0
  long long mine = 0;
  const int per = (a.B + NTHREADS - 1) / NTHREADS;
  for (int b = tid * per; b < min(a.B, (tid + 1) * per); ++b) mine += tiles_of(p8::seq_len(a, b));
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
  if (idle && tid == 0) p.border[blockIdx.x] = Border{0, 0};
  if (g0 >= lo && g0 < lo + mine * a.Hk) {
    for (int b = tid * per;; ++b) {
      const int nt = tiles_of(p8::seq_len(a, b));
      if (g0 < lo + (long long)nt * a.Hk) {
        const int kh = (int)((g0 - lo) / nt);
        start[0] = b;
        start[1] = kh;
        start[2] = (int)((g0 - lo) % nt);
        // the item's tiles [begin, end); tile g lies in CTA ((g + 1) used - 1) / total
        const long long begin = lo + (long long)kh * nt, end = begin + nt;
        const int from = (int)(((begin + 1) * used - 1) / total), to = (int)((end * used - 1) / total);
        p.border[blockIdx.x] = Border{b * a.Hk + kh, begin < g0 && from == (int)blockIdx.x - 1 ? to - from + 1 : 0};
        break;
      }
      lo += (long long)nt * a.Hk;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  // the combine kernel's CTAs may take free places now; they wait for this grid's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int ntot = (int)(g1 - g0);
  Walk w;  // a CTA without tiles walks nothing
  w.b = idle ? a.B : start[0];
  w.kh = start[1];
  w.tile = start[2];
  enter(w, a);

  if (warp == 4) {
    // ------------------------------------------------------------------ TMA producer
    const int blk = min(a.block, TK), nblk = TK / blk;
    struct Pre {
      int id, kh, row;  // page of this lane (-2: no keys there), KV head, first row inside the page
    };
    auto fetch = [&](Pre& f) {
      const int t0 = w.tile * TK, t = t0 + lane * blk;
      f.id = lane < nblk && t < w.len ? __ldg(a.table + (int64_t)w.b * a.width + t / a.block) : -2;
      f.kh = w.kh;
      f.row = a.block > TK ? t0 % a.block : 0;
      if (++w.tile == w.nt) next_item(w, a);
    };
    auto in_pool = [&](const Pre& f) { return f.id >= 0 && f.id < a.pages; };
    auto scales = [&](const Pre& f) {
      const int64_t i = (int64_t)f.id * a.Hk + f.kh;
      return in_pool(f) ? make_float2(__ldg(a.ks + i), __ldg(a.vs + i)) : make_float2(-1.f, 0.f);
    };
    // the copies of one tile into ring place st of `full`, lane = page
    auto issue = [&](const Pre& f, const CUtensorMap* m, uint64_t* full, uint32_t dst) {
      const bool load = in_pool(f);
      const unsigned n = __popc(__ballot_sync(0xffffffffu, load));
      if (lane == 0) mbar_expect_tx(full, n * (uint32_t)blk * HD);
      __syncwarp();
      if (load) tma_load_2d(dst + lane * blk * HD, m, full, 0, (f.id * a.Hk + f.kh) * a.block + f.row);
    };
    const uint32_t base = smem_u32(sm);
    Pre f0{-2, 0, 0}, f1{-2, 0, 0};
    if (ntot > 0) fetch(f0);
    if (ntot > 1) fetch(f1);
    float2 s0 = scales(f0);
    if (ntot > 0) issue(f0, &mk, &k_full[0], base);
    int issued = 0, k_issued = min(ntot, 1);
    for (int i = 0; i < ntot; ++i) {
      Pre f2{-2, 0, 0};
      if (i + 2 < ntot) fetch(f2);
      const float2 s1 = scales(f1);
      if (i + 1 < ntot) {  // K a tile ahead of V: its place is free early
        const int st = (i + 1) % SK;
        bool ok = true;
        if (lane == 0) ok = mbar_wait(&k_empty[st], (((i + 1) / SK) & 1) ^ 1, abort_flag, &g_error, 1);
        if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) break;
        issue(f1, &mk, &k_full[st], base + st * C::KV);
        k_issued = i + 2;
      }
      const int st = i % SV;
      bool ok = true;
      if (lane == 0) ok = mbar_wait(&v_empty[st], ((i / SV) & 1) ^ 1, abort_flag, &g_error, 11);
      if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) break;
      if (lane < nblk) {
        scl[(st * 2) * kMaxBlocksPerTile + lane] = s0.x;  // negative: no such page, its rows read as zeros
        scl[(st * 2 + 1) * kMaxBlocksPerTile + lane] = s0.y;
      }
      (void)VO_DCHECK(in_pool(f0) || f0.id == -2);  // checked builds record a page id outside the pool
      const float vmax = warp_fmax(s0.y);  // 0 without a page
      const bool missing = __any_sync(0xffffffffu, lane < nblk && !in_pool(f0));
      if (lane == 0) *reinterpret_cast<float4*>(tile_v + st * 4) = make_float4(vmax, missing ? 1.f : 0.f, vmax > 0.f ? kPOne / vmax : 0.f, 0.f);
      __syncwarp();
      issue(f0, &mv, &v_full[st], base + C::V_OFF + st * C::KV);
      issued = i + 1;
      f0 = f1;
      f1 = f2;
      s0 = s1;
    }
    if (lane == 0 && *abort_flag) {  // the copies in flight land before the CTA leaves
      for (int i = max(0, issued - SV); i < issued; ++i) mbar_drain(&v_full[i % SV], (i / SV) & 1);
      for (int i = max(0, k_issued - SK); i < k_issued; ++i) mbar_drain(&k_full[i % SK], (i / SK) & 1);
    }
    __syncwarp();
  } else if (warp == 5) {
    // ------------------------------------------------------------------ MMA issuer
    {
      const int e = lane == 0;
      constexpr uint32_t id_s = idesc(128, NB, 0, 0);  // K (K-major) x Q (K-major)
      constexpr uint32_t id_o = idesc(128, NB, 1, 0);  // V (read MN-major) x P (K-major)
      const uint32_t base = smem_u32(sm), tm = (uint32_t)uniform((int)tmem);
      const int ntot_u = uniform(ntot);
      uint64_t* last_bar = nullptr;  // the latest commit: its completion covers every product issued
      uint32_t last_par = 0;
      int left = 0, seg = 0;
      auto issue_s = [&](int i) {
        if (left == 0) {  // first tile of an item: its queries
          left = uniform(min(w.nt - w.tile, ntot_u - i));
          if (!mbar_wait_warp(q_full, seg & 1, abort_flag, &g_error, 2)) return false;
          ++seg;
          next_item(w, a);
        }
        --left;
        const int sb = i & 1, st = i % SK;
        if (!mbar_wait_warp(&k_full[st], (i / SK) & 1, abort_flag, &g_error, 3) ||
            !mbar_wait_warp(&s_empty[sb], ((i >> 1) & 1) ^ 1, abort_flag, &g_error, 4))
          return false;
        fence_after();
        const uint32_t ka = base + st * C::KV, qa = base + C::Q_OFF;
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk)
          mma_ss(tm + S_COL + sb * NB, desc<HD>(ka + kk * 32, 16, 8 * HD), desc<HD>(qa + kk * 32, 16, 8 * HD), id_s, kk > 0, e);
        commit(&s_full[sb], e);
        commit(&k_empty[st], e);
        last_bar = &k_empty[st];
        last_par = (i / SK) & 1;
        return true;
      };
      auto issue_pv = [&](int i) {
        const int sb = i & 1, st = i % SV;
        if (!mbar_wait_warp(&v_full[st], (i / SV) & 1, abort_flag, &g_error, 12) ||
            !mbar_wait_warp(&p_full[sb], (i >> 1) & 1, abort_flag, &g_error, 5) ||
            !mbar_wait_warp(&o_empty[sb], ((i >> 1) & 1) ^ 1, abort_flag, &g_error, 6))
          return false;
        fence_after();
        const uint32_t va = base + C::V_OFF + st * C::KV, pa = base + C::P_OFF + sb * NB * TK;
        // head_dim 64: the second half of the 128 lanes repeats the first (stride 0 between 64-dim groups), unused
#pragma unroll
        for (int kk = 0; kk < TK / 32; ++kk)
          mma_ss(tm + O_COL + sb * NB, desc<HD>(va + kk * 32 * HD, 0, 8 * HD), desc<128>(pa + kk * 32, 16, 1024), id_o, kk > 0, e);
        commit(&o_full[sb], e);
        commit(&v_empty[st], e);
        last_bar = &v_empty[st];
        last_par = (i / SV) & 1;
        return true;
      };
      bool ok = ntot_u > 0 && issue_s(0);
      for (int i = 0; i < ntot_u && ok; ++i) {
        if (i + 1 < ntot_u) ok = issue_s(i + 1);
        if (ok) ok = issue_pv(i);
      }
      if (last_bar) mbar_drain(last_bar, last_par);  // before tensor memory is released
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax and output (warps 0-3)
    const int R = a.S * a.rep;  // query rows of an item, <= NR
    // queries of item (b, kh): thread = 8 consecutive elements of a row; row factor 2^e * scale goes to the scores
    constexpr int LPR = HD / 8, QN = (NR * LPR + 127) / 128;  // lanes of a row, rows of a thread
    uint4 qr[QN];
    auto fetch_q = [&](int b, int kh) {
#pragma unroll
      for (int i = 0; i < QN; ++i) {
        const int r = tid / LPR + i * (128 / LPR);
        qr[i] = make_uint4(0, 0, 0, 0);
        if (r < R) {
          const int s = r / a.rep, h = kh * a.rep + r % a.rep;
          qr[i] = __ldg(reinterpret_cast<const uint4*>(a.q + b * a.qsb + h * a.qsh + s * a.qss + (tid % LPR) * 8));
        }
      }
    };
    auto load_q = [&](int buf) {
#pragma unroll
      for (int i = 0; i < QN; ++i) {
        const int r = tid / LPR + i * (128 / LPR), c = tid % LPR;
        if (r >= NR) break;  // whole warps
        float f[8];
        const uint4 u = qr[i];
        const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
        float m = 0.f;
        bool finite = true;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f[2 * k] = __uint_as_float(uw[k] << 16);
          f[2 * k + 1] = __uint_as_float(uw[k] & 0xffff0000u);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          m = fmaxf(m, fabsf(f[k]));
          finite = finite && fabsf(f[k]) <= 3.4028234e38f;
        }
        if (!finite) m = INFINITY;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const bool bad = m == INFINITY;  // a row with an infinity or NaN: its scores are NaN
        const float up = m == 0.f || bad ? 1.f : p8::scale_of(m), inv = inv_pow2(up);
        float lo8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = bad ? 0.f : f[i] * inv;
        const uint2 hi = p8::pack_e4m3x8(f);
        p8::unpack_e4m3x8(hi, lo8);
#pragma unroll
        for (int i = 0; i < 8; ++i) lo8[i] = (f[i] - lo8[i]) * kQLow;
        uint8_t* q = sm + C::Q_OFF + swz<HD>(r, c >> 1) + (c & 1) * 8;
        *reinterpret_cast<uint2*>(q) = hi;
        *reinterpret_cast<uint2*>(q + NP * HD) = p8::pack_e4m3x8(lo8);
        if (c == 0) qsc[buf * MAXR + r] = bad ? __int_as_float(0x7fffffff) : a.scale_log2 * up;
      }
      fence_async_smem();
      mbar_arrive(q_full);
    };
    const uint32_t trow = tmem + ((uint32_t)(warp * 32) << 16);
    const int blk = min(a.block, TK), my_blk = tid / blk;
    // row factors of a tile's fold, by its parity, a copy per warp (they are the same in all threads, and registers are short): what
    // is there already shrinks by alpha where the maximum grew, the tile's output by down where its reference lies below it
    float* alpha = reinterpret_cast<float*>(sm + C::FOLD_OFF) + warp * 4 * MAXR;
    float* down = alpha + 2 * MAXR;
    int seg = 0, it = 0;
    if (ntot > 0) {
      fetch_q(w.b, w.kh);
      load_q(0);
    }
    while (it < ntot) {
      const int nseg = min(w.nt - w.tile, ntot - it), nq = p8::seq_q(a, w.b);
      const bool from_start = w.tile == 0, whole = from_start && nseg == w.nt;
      float m[NR], lpart[NR], acc[NR], qf[NR];
      int lim[CAUSAL ? NR : 1];
      float vfac = 0.f;  // of the tile that is folded next
      bool rescale = false, far = false;  // and whether it has row factors
      int nan_at = 0x7fffffff;  // first key whose value in this thread's column is NaN (tiles that a row sees partly)
      compute_sync();           // row factors of this item are written
#pragma unroll
      for (int h = 0; h < NR; ++h) {
        m[h] = -INFINITY;
        lpart[h] = acc[h] = 0.f;
        qf[h] = qsc[(seg & 1) * MAXR + h];
        if (CAUSAL) {
          const int s = h / a.rep;
          lim[h] = h < R && s < nq ? max(0, w.len - nq + s + 1) : 0;
        }
      }
      if (!CAUSAL) lim[0] = nq > 0 ? w.len : 0;
      // keys below it are seen by every row that sees any
      const int common = nq == 0 ? 0 : CAUSAL ? max(1, w.len - nq + 1) : w.len;
      auto fold = [&](int i) {  // thread = head-dim column: acc = acc * alpha_i + O_i
        const int sb = i & 1;
        mbar_wait(&o_full[sb], (i >> 1) & 1, abort_flag, &g_error, 7);
        __syncwarp();
        fence_after();
        uint32_t r[NB];
        ld_nowait(trow + O_COL + sb * NB, r);
        wait_ld();
        fence_before();
        mbar_arrive(&o_empty[sb]);
        if (rescale) {
#pragma unroll
          for (int h = 0; h < NR; ++h) acc[h] *= alpha[sb * MAXR + h];
        }
        if (far) {
#pragma unroll
          for (int h = 0; h < NR; ++h) {
            const float f = down[sb * MAXR + h];
            r[h] = __float_as_uint(__uint_as_float(r[h]) * f), r[NP + h] = __float_as_uint(__uint_as_float(r[NP + h]) * f);
          }
        }
#pragma unroll
        for (int h = 0; h < NR; ++h) acc[h] = fmaf(fmaf(__uint_as_float(r[NP + h]), 1.f / kPLow, __uint_as_float(r[h])), vfac, acc[h]);
      };
      const Walk cur = w;
      next_item(w, a);
      for (int j = 0; j < nseg; ++j) {
        const int i = it + j, sb = i & 1, st = i % SV, t0 = (cur.tile + j) * TK, t = t0 + tid;
        const bool last_q = j + 1 == nseg && it + nseg < ntot;
        if (last_q) fetch_q(w.b, w.kh);  // the next item's queries
        mbar_wait(&v_full[st], (i / SV) & 1, abort_flag, &g_error, 8);
        mbar_wait(&s_full[sb], (i >> 1) & 1, abort_flag, &g_error, 9);
        __syncwarp();
        fence_after();
        uint32_t r[NB];
        ld_nowait(trow + S_COL + sb * NB, r);
        const float ksc = scl[(st * 2) * kMaxBlocksPerTile + my_blk];
        float vsc = scl[(st * 2 + 1) * kMaxBlocksPerTile + my_blk];
        const float4 tv = *reinterpret_cast<const float4*>(tile_v + st * 4);
        // a whole tile: every row sees all of its keys, all its pages exist
        const bool full = t0 + TK <= common && tv.y == 0.f;
        wait_ld();
        fence_before();
        mbar_arrive(&s_empty[sb]);
        float s[NR];
#pragma unroll
        for (int h = 0; h < NR; ++h) s[h] = fmaf(__uint_as_float(r[NP + h]), 1.f / kQLow, __uint_as_float(r[h])) * (ksc * qf[h]);
        bool there = true;
        if (!full) {
          there = t < cur.len && !(ksc < 0.f);
          if (!there) vsc = 0.f;
#pragma unroll
          for (int h = 0; h < NR; ++h) {
            const bool seen = CAUSAL ? t < lim[h] : t < lim[0];
            s[h] = !seen ? -INFINITY : ksc < 0.f ? 0.f : s[h];
          }
        }
        float4* rd = reinterpret_cast<float4*>(red + sb * 4 * MAXR);  // [warp][row]
#pragma unroll
        for (int h = 0; h < NR; h += 4) {
          const float4 v = make_float4(warp_fmax(s[h]), warp_fmax(s[h + 1]), warp_fmax(s[h + 2]), warp_fmax(s[h + 3]));
          if (lane == 0) rd[warp * (MAXR / 4) + h / 4] = v;
        }
        compute_sync();
        const float vr = vsc * tv.z;
        float mx[NR];
        bool grown = false;
#pragma unroll
        for (int h = 0; h < NR; h += 4) {
          float4 x = rd[h / 4];
#pragma unroll
          for (int w4 = 1; w4 < 4; ++w4) {
            const float4 y = rd[w4 * (MAXR / 4) + h / 4];
            x.x = fmaxf(x.x, y.x), x.y = fmaxf(x.y, y.y), x.z = fmaxf(x.z, y.z), x.w = fmaxf(x.w, y.w);
          }
          mx[h] = x.x, mx[h + 1] = x.y, mx[h + 2] = x.z, mx[h + 3] = x.w;
        }
#pragma unroll
        for (int h = 0; h < NR; ++h) grown = grown || mx[h] > m[h];
        if (grown) {  // the same in all threads; rare once a sequence is under way
#pragma unroll
          for (int h = 0; h < NR; ++h) {
            const float mn = fmaxf(m[h], mx[h]), al = mn == -INFINITY ? 1.f : ex2(m[h] - mn);
            lpart[h] *= al;
            m[h] = mn;
            if (lane == 0) alpha[sb * MAXR + h] = al;
          }
        }
        uint8_t* pb = sm + C::P_OFF + sb * NB * TK;
        const int prow = tid & 15, pcol = tid >> 4;
        // p to 8 bits: the nearest e4m3 number and the nearest one to what is left (f16 between: 11 bits)
        auto emit = [&](int h, float p0, float p1) {
          const __half2 p16 = __floats2half2_rn(p0, p1);
          const __nv_fp8x2_storage_t hi = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&p16), __NV_SATFINITE, __NV_E4M3);
          const __half2_raw back = __nv_cvt_fp8x2_to_halfraw2(hi, __NV_E4M3);
          const __half2 rest = __hmul2(__hsub2(p16, *reinterpret_cast<const __half2*>(&back)), __float2half2_rn(kPLow));
          const __nv_fp8x2_storage_t lo2 = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&rest), __NV_SATFINITE, __NV_E4M3);
          uint8_t* d0 = pb + swz<128>(h, pcol) + prow;
          uint8_t* d1 = pb + swz<128>(h + 1, pcol) + prow;
          d0[0] = (uint8_t)hi;
          d1[0] = (uint8_t)(hi >> 8);
          d0[NP * TK] = (uint8_t)lo2;
          d1[NP * TK] = (uint8_t)(lo2 >> 8);
        };
        bool far_now = false;  // the same in all threads, too
#pragma unroll
        for (int h = 0; h < NR; ++h) far_now = far_now || m[h] - mx[h] > kFar;
#pragma unroll
        for (int h = 0; h < NR; ++h) {
          // in a full tile m is finite, or the scores are NaN
          s[h] = full || s[h] != -INFINITY ? ex2(s[h] - m[h]) : 0.f;
          lpart[h] += s[h];
        }
        if (far_now) {
#pragma unroll
          for (int h = 0; h < NR; ++h) {
            const float gap = m[h] - mx[h];  // no key of the tile seen: infinite, no weight either; none so far: NaN
            const float f = p8::pow2(gap > kFar ? -(int)fminf(gap, 126.f) : 0);
            s[h] *= inv_pow2(f);
            if (lane == 0) down[sb * MAXR + h] = f;
          }
        }
#pragma unroll
        for (int h = 0; h < NR; h += 2) emit(h, s[h] * vr, s[h + 1] * vr);
        if (!full) {
          uint8_t* vt = sm + C::V_OFF + st * C::KV;
          if (!there) {  // rows that hold nothing: zero, so that 0 * garbage stays 0
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) reinterpret_cast<uint4*>(vt + tid * HD)[c] = make_uint4(0, 0, 0, 0);
          }
          if (CAUSAL && tv.y != 0.f) compute_sync();  // zeroed before they are looked through below
          if (CAUSAL && tid < HD) {
            // some row may see only part of this tile: a NaN value must not reach it through 0 * NaN
            for (int k = 0; k < min(TK, cur.len - t0); ++k) {
              uint8_t* v = vt + swz<HD>(k, tid >> 4) + (tid & 15);
              if ((*v & 0x7f) == 0x7f) {
                *v = 0;
                nan_at = min(nan_at, t0 + k);
              }
            }
          }
        }
        fence_async_smem();
        mbar_arrive(&p_full[sb]);
        if (last_q) load_q((seg & 1) ^ 1);  // scores of this item are all read
        if (j > 0) fold(i - 1);
        rescale = grown;
        far = far_now;
        vfac = tv.x * (1.f / kPOne);
      }
      fold(it + nseg - 1);
      // sums over the keys' threads
      compute_sync();
#pragma unroll
      for (int h = 0; h < NR; ++h) {
        float v = lpart[h];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) red[h * 4 + warp] = v;  // [row][warp] here
      }
      compute_sync();
      const int64_t slot = ((int64_t)blockIdx.x * 2 + (from_start ? 1 : 0)) * NR;
#pragma unroll
      for (int h = 0; h < NR; ++h) {
        if (h >= R) break;
        const float4 x = *reinterpret_cast<const float4*>(red + h * 4);
        float l = (x.x + x.y) + (x.z + x.w), o = acc[h];
        if (CAUSAL && lim[h] > nan_at) o = __int_as_float(0x7fffffff);
        if (CAUSAL && lim[h] == 0) m[h] = -INFINITY, l = 0.f, o = 0.f;  // a row that sees nothing
        if (tid < HD) {
          if (whole) {
            const int64_t row = ((int64_t)cur.b * a.S + h / a.rep) * a.Hq + cur.kh * a.rep + h % a.rep;
            a.out[row * HD + tid] = __float2bfloat16_rn(l == 0.f ? 0.f : o / l);
          } else {
            p.part_o[(slot + h) * HD + tid] = o;
          }
        }
        if (!whole && tid == h) {
          p.part_ml[(slot + h) * 2] = m[h];
          p.part_ml[(slot + h) * 2 + 1] = l;
        }
      }
      compute_sync();  // the sums are read before the next item's maxima overwrite them
      it += nseg;
      ++seg;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 5) tmem_free(tmem, TMEM_COLS);
}

// Merges the partials of an item that CTA borders cut: block c acts where border c is the first inside its item.  Part 0
// is slot 1 of the CTA before, the others slot 0 of CTAs c, c + 1, ...; a warp takes a row (NR = 4: two warps, every other
// part each; NR = 16: two rows one after the other), lane = HD / 32 columns, weights of 32 parts at once in the lanes.
// The order of the sums is that of the keys.
template <int HD, int NR>
__global__ void __launch_bounds__(256) combine8_kernel(const AttendArgs a, const float* __restrict__ part_o,
                                                       const float* __restrict__ part_ml, const Border* __restrict__ border) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int V = HD / 32, WPR = NR < 8 ? 2 : 1;  // columns of a lane, warps of a row
  __shared__ float so[8][HD], sml[8][2];
  const int c = blockIdx.x + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = a.S * a.rep;
  const Border me = border[c];
  if (me.parts == 0) return;
  const int parts = me.parts, sub = warp % WPR;
#pragma unroll 1
  for (int r = warp / WPR; r < NR; r += 8 / WPR) {
    auto row_of = [&](int i) -> int64_t { return i == 0 ? ((int64_t)(c - 1) * 2 + 1) * NR + r : (int64_t)(c + i - 1) * 2 * NR + r; };
    float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
    for (int k = 0; k < V; ++k) o[k] = 0.f;
    for (int i0 = sub; i0 < parts; i0 += 32 * WPR) {
      const int i = i0 + lane * WPR;
      const float2 ml = r < R && i < parts ? *reinterpret_cast<const float2*>(part_ml + row_of(i) * 2) : make_float2(-INFINITY, 0.f);
      const float mn = fmaxf(m, warp_fmax(ml.x));
      const float al = mn == -INFINITY ? 1.f : ex2(m - mn), w = mn == -INFINITY ? 1.f : ex2(ml.x - mn);
      float lw = ml.y * w;
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, s);
      l = l * al + lw;
      m = mn;
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] *= al;
      const int n = min(32, (parts - i0 + WPR - 1) / WPR);
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const float wj = __shfl_sync(0xffffffffu, w, j);
        const float* x = part_o + row_of(i0 + j * WPR) * HD + lane * V;
        if (r < R) {
          if constexpr (V == 4) {
            const float4 v = *reinterpret_cast<const float4*>(x);
            o[0] += v.x * wj, o[1] += v.y * wj, o[2] += v.z * wj, o[3] += v.w * wj;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(x);
            o[0] += v.x * wj, o[1] += v.y * wj;
          }
        }
      }
    }
    if constexpr (WPR == 2) {
      if (lane == 0) sml[warp][0] = m, sml[warp][1] = l;
#pragma unroll
      for (int k = 0; k < V; ++k) so[warp][lane * V + k] = o[k];
      __syncthreads();
      if (sub == 0) {
        const float m1 = sml[warp + 1][0], mn = fmaxf(m, m1);
        const float w0 = mn == -INFINITY ? 1.f : ex2(m - mn), w1 = mn == -INFINITY ? 1.f : ex2(m1 - mn);
        l = l * w0 + sml[warp + 1][1] * w1;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = o[k] * w0 + so[warp + 1][lane * V + k] * w1;
      }
    }
    if (sub == 0 && r < R) {
      const int b = me.item / a.Hk, kh = me.item % a.Hk;
      const int64_t row = ((int64_t)b * a.S + r / a.rep) * a.Hq + kh * a.rep + r % a.rep;
#pragma unroll
      for (int k = 0; k < V; ++k) a.out[row * HD + lane * V + k] = __float2bfloat16_rn(l == 0.f ? 0.f : o[k] / l);
    }
  }
}

template <int HD, int NR, bool CAUSAL>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int G, cudaStream_t stream, int* launches) {
  static PerDevice once;
  cudaError_t e = once([] {
    return cudaFuncSetAttribute(decode8_kernel<HD, NR, CAUSAL>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD, NR>::BYTES);
  });
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
  cfg.dynamicSmemBytes = Cfg<HD, NR>::BYTES;
  e = cudaLaunchKernelEx(&cfg, decode8_kernel<HD, NR, CAUSAL>, mk, mv, p);
  if (e != cudaSuccess) return (int)e;
  ++*launches;
  if (G == 1) return 0;
  cfg.gridDim = dim3(G - 1);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, combine8_kernel<HD, NR>, p.a, (const float*)p.part_o, (const float*)p.part_ml, (const Border*)p.border);
  if (e != cudaSuccess) return (int)e;
  ++*launches;
  return 0;
}

template <int HD>
int pick(const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, int G, int NR, cudaStream_t stream, int* launches) {
  const bool causal = p.a.S > 1;
#define VO_D8(N) \
  if (NR == N) return causal ? launch<HD, N, true>(mk, mv, p, G, stream, launches) : launch<HD, N, false>(mk, mv, p, G, stream, launches);
  VO_D8(4) VO_D8(8) VO_D8(16)
#undef VO_D8
  return -1;
}

// row slots of a CTA: the query rows rounded up to 4, 8 or 16
int rows_of(int64_t r) { return r <= 4 ? 4 : r <= 8 ? 8 : 16; }

// CTAs: two per SM, one tile each at least (by the table's reach: the lengths are on the device)
int ctas(const AttendArgs& a, int sms) {
  const int64_t reach = ((int64_t)a.width * a.block + TK - 1) / TK;
  const int64_t most = (int64_t)a.B * a.Hk * (reach < 1 ? 1 : reach);
  return (int)(most < 2 * sms ? most : 2 * sms);
}

}  // namespace p8dec

bool paged8_decode_ok(const p8::AttendArgs& a) {
  if (a.hd != 64 && a.hd != 128) return false;
  if ((int64_t)a.S * a.rep > p8dec::MAXR) return false;
  return paged8_pages_ok(a);
}

int64_t paged8_decode_workspace(const p8::AttendArgs& a, int sms) {
  const int64_t G = p8dec::ctas(a, sms), NR = p8dec::rows_of((int64_t)a.S * a.rep);
  return G * 2 * NR * (a.hd + 2) * 4 + G * (int64_t)sizeof(p8dec::Border);
}

int paged8_decode_launch(const p8::AttendArgs& a, void* workspace, int sms, cudaStream_t stream, int* launches) {
  using namespace p8dec;
  CUtensorMap mk, mv;
  const int64_t rows = (int64_t)a.pages * a.Hk * a.block;
  const int box = a.block < TK ? a.block : TK;
  int e = map_rows(&mk, a.kp, rows, a.hd, box, true);
  if (e) return e;
  e = map_rows(&mv, a.vp, rows, a.hd, box, true);
  if (e) return e;
  const int G = ctas(a, sms), NR = rows_of((int64_t)a.S * a.rep);
  Params p;
  p.a = a;
  p.part_o = static_cast<float*>(workspace);  // 16-byte rows first
  p.part_ml = p.part_o + (int64_t)G * 2 * NR * a.hd;
  p.border = reinterpret_cast<Border*>(p.part_ml + (int64_t)G * 2 * NR * 2);
  return a.hd == 128 ? pick<128>(mk, mv, p, G, NR, stream, launches) : pick<64>(mk, mv, p, G, NR, stream, launches);
}

int paged8_decode_error(bool reset) {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, p8dec::g_error, sizeof(int)) != cudaSuccess) return -1;
  if (reset && h) {
    const int z = 0;
    cudaMemcpyToSymbol(p8dec::g_error, &z, sizeof(int));
  }
  return h;
}

}  // namespace vo
