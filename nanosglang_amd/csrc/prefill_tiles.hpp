// The prefill kernel (prefill_attention.hip: 32 query rows a wave on
// v_mfma_f32_32x32x16_bf16, 64-token steps through an LDS ring) for what that one
// does not do:
//   KV8   the 8-bit pool (fp8_kv.hpp).  A thread loads 16-byte runs of codes
//         and their row's scale bytes a step ahead and turns the present ones
//         into bf16 in the same LDS tiles on the way, exactly, one instruction
//         per two values, once for all of the workgroup's rows.
//   PART  an item is a share [kvb, kve) of its tile's KV range and leaves partial
//         rows (O unnormalised, m, l) of D + 4 floats for a merge, 32 NW rows per
//         item and KV head.
//
// Softmax may subtract any base from a row's scores, so a row keeps the maximum
// of its item's first step (a row that sees nothing of it sees nothing of the
// item): the steps after it need no maximum, no rescaling of the accumulators
// and no wait for either.  Later scores above the base make probabilities above
// one, which bf16 and the fp32 sums hold with the same relative error up to
// 2^127; a workgroup one of whose rows passed 2^60 finds its rows' maxima in a
// pass over K and goes through its steps once more.  Dropping the running maximum
// (16 max3, a swap, 64 multiplies or, around a branch, as many register moves of
// the accumulators per step) measured at 4 x 1000-token chunks over 2048 - 8192,
// 32 / 8 heads of 128, a kernel alone, from 413 to 386 us.  Pass after pass 307 us now,
// 0.93 PFLOP/s of the causal products: matrix cores 39 % busy, vector ALU 40 %,
// LDS 30 %, their phases a third overlapped.
#pragma once

#include "attention.hpp"
#include "fp8_kv.hpp"

namespace nsg {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 64;  // KV tokens per ring step

// One LDS DMA copy of 16 bytes per lane (lane l lands at lds + 16 l), in asm:
// through the builtin the compiler's wait-count pass would wait for every
// copy in flight before each LDS read; the ring's own waits order them.
__device__ __forceinline__ void dma16(uint32_t lds, const void* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(src)
               : "memory", "m0");
}

__device__ __forceinline__ float max_xor32(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_xor32(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// V's chunk swizzle: the 32 lanes that one pass of a transposed read serves take
// four chunks of four neighbouring rows, which fall on 16 different 16-byte bank
// groups (with the swizzle of prefill_attention.hip on 8: 104,000 of 278,000 LDS
// cycles a CU were conflicts in the chunks below, 35,000 of 210,000 with this one, and
// they took 320 us instead of 307).
template <int D>
__device__ __forceinline__ int swz_vt(int t) {
  if constexpr (D == 64) return 4 * ((t >> 1) & 1) + 2 * ((t >> 2) & 1);  // two rows a line
  return 4 * (t & 3) + 2 * ((t >> 2) & 1);
}

// The order of N products, each of which takes READS reads from LDS, in what was
// scheduled since the last barrier: the reads of AHEAD products first, then a
// product and the reads of a later one in turn, so that a read's latency passes
// under AHEAD products (4 x 1000-token chunks over 2048 - 8192, 32 / 8 heads of 128:
// 331 us with each product behind its own reads, 318 with four ahead, 320 with six; V as it was
// swizzled then).
template <int N, int READS, int AHEAD, int I = 0>
__device__ __forceinline__ void feed() {
  constexpr int kMfma = 0x8, kLdsRead = 0x100;
  if constexpr (I == 0) __builtin_amdgcn_sched_group_barrier(kLdsRead, READS * AHEAD, 0);
  __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
  if constexpr (I + AHEAD < N) __builtin_amdgcn_sched_group_barrier(kLdsRead, READS, 0);
  if constexpr (I + 1 < N) feed<N, READS, AHEAD, I + 1>();
}

// Ring slots.  Two wave groups (head dim 128, 8 waves): four, a slot is read
// over four phases.  Otherwise two of head dim 128 (68 KB, two workgroups a CU)
// or three of 64 (52 KB, three a CU); the 8-bit pool's next step waits in
// registers, so two do.
template <int D, int NW, bool KV8>
constexpr int tile_ring() {
  if (NW == 8) return 4;
  if (KV8) return 2;
  return D == 64 ? 3 : 2;
}

template <int D, int NW, bool KV8, bool PART>
__global__ __launch_bounds__(NW * 64, D == 64 ? 3 : 2) void attn_tile_kernel(AttnParams p) {
  constexpr int KC = D / 16;              // k chunks of S^T = K Q^T
  constexpr int DT = D / 32;              // d tiles of O^T
  constexpr int CPR = D / 8;              // 16-byte chunks per token row of a tile
  constexpr int TILE = kStep * D;         // bf16 per K (or V) tile
  constexpr int TPI = 64 / CPR;           // token rows per 1 KB copy
  constexpr int NR = kStep / TPI / NW;    // row blocks a wave copies per step (K and V each)
  constexpr int NI = 2 * NR;              // copies per wave per step
  constexpr int NBUF = tile_ring<D, NW, KV8>();
  constexpr bool PP = NW == 8;            // (head dim 128 only) two wave groups half a step apart
  static_assert(NR >= 1 && (NBUF - 1) * NI <= 63, "vmcnt counts to 63");
  __shared__ __attribute__((aligned(1024))) bf16 ring[NBUF][2][TILE];
  __shared__ int s_pages[kMaxItemPages];
  __shared__ int s_redo;  // some row's base was too low

  const int wi = blockIdx.y;
  const int h = blockIdx.x;
  const int* wk = p.work + (size_t)wi * NSG_ATTN_WORK_INTS;
  const int qs = wk[0], qn = wk[1], lim0 = wk[2], pb = wk[3], kve = wk[5];
  const int kvb = PART ? wk[4] : 0;
  if (qn == 0) return;
  const int P = 1 << p.log2P;
  const int G = p.G;
  const int nrows = qn * G;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31;
  const int g = lane >> 5;

  // page ids of the item
  const int page0 = kvb >> p.log2P;
  const int npages = min(((kve - 1) >> p.log2P) + 1 - page0, kMaxItemPages);
  bool bad_page = false;
  for (int i = tid; i < npages; i += NW * 64) {
    int pg = p.kv_indices[pb + page0 + i];
    if ((unsigned)pg >= (unsigned)p.num_pages) {
      bad_page = true;  // reads the pool's first page instead
      pg = 0;
    }
    s_pages[i] = pg;
  }
  if (tid == 0) s_redo = 0;

  // this lane's query row and its causal limit; the wave's smallest and
  // largest limit (rows past the tile's end load its first row, masked out)
  const int row = wave * 32 + r32;
  const bool row_ok = row < nrows;
  const int tau = row / G;
  const int gam = row - tau * G;
  const int lim = row_ok ? lim0 + (p.causal ? tau : 0) : -1;
  const int w_lo = lim0 + (p.causal ? (wave * 32) / G : 0);
  const int w_hi = wave * 32 >= nrows ? -1
                   : lim0 + (p.causal ? min(wave * 32 + 31, nrows - 1) / G : 0);
  bf16x8 qf[KC];
  {
    const bf16* qrow = p.q + (row_ok ? ((size_t)(qs + tau) * p.Hq + h * G + gam) * D
                                     : ((size_t)qs * p.Hq + h * G) * D);
#pragma unroll
    for (int c = 0; c < KC; ++c) qf[c] = load_bf16x8(qrow + 16 * c + 8 * g);
  }
  // Q has landed before the first copy is issued (the compiler does not see
  // the copies: its own wait for Q would drain them)
#pragma unroll
  for (int c = 0; c < KC; ++c) asm volatile("" ::"v"(__builtin_bit_cast(u32x4, qf[c])));
  __syncthreads();  // page ids visible

  floatx16 oacc[DT];
  float m_run = kMaskVal, l_run = 0.f;

  // LDS read offsets (bytes inside a K or V tile).  K fragment c of half s:
  // token 32 s + r32, logical chunk 2 c + g (the swizzle repeats every 16
  // rows).  V^T fragment (dt, m, hh): lane i of a 16-lane group addresses
  // token 16 m + 8 hh + 4 g + i / 4, columns 32 dt + 16 dh + 4 (i % 4) .. + 3,
  // and receives column i of the group's 16 for tokens j = 0..3.  (The other
  // fragments' offsets differ by an XOR of bits the swizzles leave alone.)
  const int koff = 2 * (r32 * D + ((g ^ swz_k<D>(r32)) * 8));  // fragment c: koff ^ 32 c
  int voff[2];  // fragment (dt, hh): voff[hh] ^ 64 dt; the swizzle repeats every 8 rows
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    const int i = lane & 15, dh = (lane >> 4) & 1;
    const int t = 8 * hh + 4 * g + (i >> 2);
    const int c = 16 * dh + 4 * (i & 3);
    voff[hh] = 2 * (t * D + (((c >> 3) ^ swz_vt<D>(t)) << 3) + (c & 7));
  }

  const int n_it = (kve - kvb + kStep - 1) / kStep;
  const int last_tok = kve - 1;
  // ---- filling a slot, bf16 pool: row block i of this wave holds token rows
  //      (wave + NW i) TPI .. + TPI of a step, for K and for V; lane: row
  //      lane / CPR, physical chunk lane % CPR ----
  const size_t tok_bytes = (size_t)p.Hkv * D * 2;
  const char* kbase = reinterpret_cast<const char*>(p.kc + (size_t)h * D);
  const char* vbase = reinterpret_cast<const char*>(p.vc + (size_t)h * D);
  const uint32_t ring_lds = lds_addr(&ring[0][0][0]);
  int d_t[NR];
  uint32_t d_k[NR], d_v[NR], d_lds[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int t0 = (wave + NW * i) * TPI;
    const int t = t0 + lane / CPR;
    const int pc = lane % CPR;
    d_t[i] = t;
    d_k[i] = (pc ^ swz_k<D>(t)) * 16;
    d_v[i] = (pc ^ swz_vt<D>(t)) * 16;
    d_lds[i] = t0 * D * 2;
  }
  // tokens past the item's end repeat its last one (masked out)
  auto issue = [&](int it, int slot) {
    const uint32_t sb = ring_lds + (uint32_t)slot * (2 * TILE * 2);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int tok = min(kvb + it * kStep + d_t[i], last_tok);
      const int page = s_pages[min((tok >> p.log2P) - page0, kMaxItemPages - 1)];
      const size_t off = ((size_t)(uint32_t)page * P + (tok & (P - 1))) * tok_bytes;
      dma16(sb + d_lds[i], kbase + off + d_k[i]);
      dma16(sb + 2 * TILE + d_lds[i], vbase + off + d_v[i]);
    }
  };
  // ---- 8-bit pool: run i of this thread is codes 16 c .. + 15 of token row t ----
  constexpr int NC = KV8 ? D / 16 / NW : 1;
  u32x4 k8[NC], v8[NC];
  uint32_t ke[NC], ve[NC];
  auto fetch = [&](int it) {  // a step's codes and scales into registers
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int id = tid + i * NW * 64;
      const int tok = min(kvb + it * kStep + id / (D / 16), last_tok);
      const size_t page = (uint32_t)s_pages[min((tok >> p.log2P) - page0, kMaxItemPages - 1)];
      const int at = tok & (P - 1);
      const size_t off = ((page * P + at) * p.Hkv + h) * D + (id % (D / 16)) * 16;
      const uint8_t* sc = p.kv_scale + ((page * p.Hkv + h) * 2 << p.log2P) + at;
      k8[i] = *reinterpret_cast<const u32x4*>(p.kc8 + off);
      v8[i] = *reinterpret_cast<const u32x4*>(p.vc8 + off);
      ke[i] = sc[0];
      ve[i] = sc[P];
    }
  };
  auto commit = [&](int slot) {  // ... and from there, as bf16, into a ring slot
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int id = tid + i * NW * 64;
      const int t = id / (D / 16), c = 2 * (id % (D / 16));
      // A V row that is NaN is kept out of the tile, where a masked row's
      // probability of zero would meet it; its K row's NaN scores stand in
      const bool nan = ve[i] == kE8M0NaN;
      const float ks = e8m0_scale(nan ? kE8M0NaN : ke[i]), vs = nan ? 1.f : e8m0_scale(ve[i]);
      const u32x4 kw = k8[i], vw = nan ? u32x4{0, 0, 0, 0} : v8[i];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const fp8_u32x2 ka = from_fp8x4(kw[2 * x], ks), kb = from_fp8x4(kw[2 * x + 1], ks);
        const fp8_u32x2 va = from_fp8x4(vw[2 * x], vs), vb = from_fp8x4(vw[2 * x + 1], vs);
        *reinterpret_cast<u32x4*>(&ring[slot][0][t * D + ((c + x) ^ swz_k<D>(t)) * 8]) =
            u32x4{ka[0], ka[1], kb[0], kb[1]};
        *reinterpret_cast<u32x4*>(&ring[slot][1][t * D + ((c + x) ^ swz_vt<D>(t)) * 8]) =
            u32x4{va[0], va[1], vb[0], vb[1]};
      }
    }
  };

  floatx16 sacc[2];  // S^T of the current step
  u32x4 pf[4];       // P^T of it in bf16: one B operand per 16 tokens
  auto qk = [&](int slot) {
    const char* Kt = reinterpret_cast<const char*>(&ring[slot][0][0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 16; ++i) sacc[s][i] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bf16x8 kf = *reinterpret_cast<const bf16x8*>(Kt + 32 * s * D * 2 + (koff ^ (32 * c)));
        sacc[s] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[c], sacc[s], 0, 0, 0);
      }
    feed<2 * KC, 1, 4>();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto mask = [&](int t0) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = t0 + 32 * s + 8 * (i >> 2) + 4 * g + (i & 3);
        if (j > lim || j >= kve) sacc[s][i] = kMaskVal;
      }
  };
  auto row_max = [&]() {  // of the step's scores, as an exponent base
    float mx = kMaskVal;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sacc[s][i]);
    mx = max_xor32(mx);
    return mx == kMaskVal ? kMaskVal : mx * p.scale_log2;
  };
  auto full = [&](int t0) { return t0 + kStep - 1 <= w_lo && t0 + kStep <= kve; };
  auto probs = [&](auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    float ps = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float pv[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(sacc[s][i], p.scale_log2, -m_run));
        pv[i] = MASKED && sacc[s][i] == kMaskVal ? 0.f : e;
        ps += pv[i];
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
        pf[2 * s + m] = u32x4{cvt_pk_bf16(pv[8 * m], pv[8 * m + 1]),
                              cvt_pk_bf16(pv[8 * m + 2], pv[8 * m + 3]),
                              cvt_pk_bf16(pv[8 * m + 4], pv[8 * m + 5]),
                              cvt_pk_bf16(pv[8 * m + 6], pv[8 * m + 7])};
    }
    l_run += ps;
  };
  int first = kvb;  // the step that sets the base (none in the second pass)
  auto softmax = [&](int t0) {
    const bool whole = full(t0);
    if (!whole) mask(t0);
    if (t0 == first) m_run = row_max();
    if (whole)
      probs(std::false_type{});
    else
      probs(std::true_type{});
  };
  auto pv_mul = [&](int slot) {  // O^T += V^T P^T
    const char* Vt = reinterpret_cast<const char*>(&ring[slot][1][0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) v4i16*)(Vt + 16 * m * D * 2 + (voff[0] ^ (64 * dt))));
        const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) v4i16*)(Vt + 16 * m * D * 2 + (voff[1] ^ (64 * dt))));
        const v8i16 w = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        oacc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, pf[m]), oacc[dt], 0, 0, 0);
      }
    }
    feed<4 * DT, 2, 4>();
    __builtin_amdgcn_sched_barrier(0);
  };
  // A workgroup-wide phase boundary: every LDS access of this wave has
  // completed, nothing moves across.
  auto phase = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  };

  for (;;) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;
    l_run = 0.f;
    if constexpr (PP) {
      // Two wave groups half a step apart: a SIMD holds one wave of each, and
      // while one runs its matrix phase (O += P V of step i - 1, S = K Q of
      // step i) the other runs its softmax phase, so the matrix cores and the
      // vector ALU work side by side.  Phase n of the workgroup: group 0 is in
      // the matrix phase of step n / 2 (n even) or the softmax of n / 2 (odd),
      // group 1 one phase behind.  Slot i % 4 is read in phases 2 i .. 2 i + 3
      // (K by both groups, then V), so from phase 2 i + 4 on it takes step
      // i + 4; a step's copies go out three phases ahead or more (8-bit pool:
      // its conversion is done there, one phase boundary before its first
      // reader, and its successor's loads go out).
      const int grp = wave >> 2;
      if constexpr (KV8) {
        fetch(0);
        commit(0);
        if (1 < n_it) {
          fetch(1);
          commit(1);
        }
        if (2 < n_it) fetch(2);
      } else {
        issue(0, 0);
        if (1 < n_it) issue(1, 1);
        wait_steps<NI, 1>(min(n_it - 1, 1));
      }
      phase();  // phase 0 begins: step 0 in LDS
      if (grp == 1) {
        if constexpr (KV8) {
          if (2 < n_it) commit(2);
          if (3 < n_it) fetch(3);
        } else {
          if (2 < n_it) issue(2, 2);
          wait_steps<NI, 1>(min(max(n_it - 2, 0), 1));  // step 1 (if any) landed
        }
        phase();
      }
      bool had = false;  // the previous step's P is pending
      for (int it = 0; it < n_it; ++it) {
        const int t0 = kvb + it * kStep;
        const bool vis = t0 <= w_hi;  // something visible to this wave's rows
        if (had) pv_mul((it - 1) & 3);
        if (vis) qk(it & 3);
        had = vis;
        if constexpr (!KV8) {
          if (grp == 1) wait_steps<NI, 1>(min(max(n_it - 2 - it, 0), 1));
        }
        phase();
        const int nx = it + 2 + grp;
        if constexpr (KV8) {
          if (nx < n_it) commit(nx & 3);
          __builtin_amdgcn_sched_barrier(0);
          if (nx + 1 < n_it) fetch(nx + 1);
          __builtin_amdgcn_sched_barrier(0);
        } else {
          if (nx < n_it) issue(nx, nx & 3);
        }
        if (vis) softmax(t0);
        if constexpr (!KV8) {
          if (grp == 0) wait_steps<NI, 1>(min(max(n_it - 2 - it, 0), 1));
        }
        phase();
      }
      if (had) pv_mul((n_it - 1) & 3);
      if (grp == 0) phase();  // group 1's last softmax phase
    } else if constexpr (KV8) {
      fetch(0);
      commit(0);
      if (1 < n_it) fetch(1);
      for (int it = 0; it < n_it; ++it) {
        phase();  // step `it` in LDS for every wave, the other slot free
        if (it + 1 < n_it) commit((it + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
        if (it + 2 < n_it) fetch(it + 2);
        __builtin_amdgcn_sched_barrier(0);
        const int t0 = kvb + it * kStep;
        if (t0 > w_hi) continue;  // nothing visible to this wave's rows
        qk(it & 1);
        softmax(t0);
        pv_mul(it & 1);
      }
    } else {
#pragma unroll
      for (int it = 0; it < NBUF - 1; ++it)
        if (it < n_it) issue(it, it);
      int slot = 0;
      for (int it = 0; it < n_it; ++it) {
        // step `it` landed for this wave (the later issued steps stay in
        // flight), and for every wave; slot (it - 1) is free
        wait_steps<NI, NBUF - 2>(min(n_it - 1 - it, NBUF - 2));
        phase();
        const int cur = slot;
        if (it + NBUF - 1 < n_it) issue(it + NBUF - 1, slot == 0 ? NBUF - 1 : slot - 1);
        slot = slot + 1 == NBUF ? 0 : slot + 1;
        const int t0 = kvb + it * kStep;
        if (t0 > w_hi) continue;
        qk(cur);
        softmax(t0);
        pv_mul(cur);
      }
    }
    if (first < 0) break;
    // did a row pass 2^60, or overflow?  (as integers: NaN counts too)
    uint32_t top = __float_as_uint(l_run) >= 0x5d800000u ? 0x7f800000u : 0u;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(oacc[dt][i]) & 0x7fffffffu);
    if (row_ok && top >= 0x7f800000u) s_redo = 1;
    phase();
    if (!__builtin_amdgcn_readfirstlane(s_redo)) break;
    // a pass over K for the rows' maxima (no pipelining), then all once more
    first = -1;
    m_run = kMaskVal;
    for (int it = 0; it < n_it; ++it) {
      if constexpr (KV8) {
        fetch(it);
        commit(0);
      } else {
        issue(it, 0);
        wait_steps<NI, 0>(0);
      }
      phase();
      qk(0);
      const int t0 = kvb + it * kStep;
      if (!full(t0)) mask(t0);
      m_run = fmaxf(m_run, row_max());
      phase();
    }
  }

  if (bad_page) atomicOr(p.flags, 1);
  const float l = sum_xor32(l_run);
  if (!row_ok) return;
  if constexpr (PART) {
    float* prow = p.partials + (((size_t)wi * p.Hkv + h) * (32 * NW) + row) * (D + 4);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const floatx16 o = oacc[dt];
        *reinterpret_cast<floatx4*>(prow + 32 * dt + 8 * a + 4 * g) =
            floatx4{o[4 * a], o[4 * a + 1], o[4 * a + 2], o[4 * a + 3]};
      }
    if (g == 0) {
      prow[D] = m_run;
      prow[D + 1] = l;
    }
  } else {
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // l NaN stays NaN
    bf16* orow = p.out + ((size_t)(qs + tau) * p.Hq + h * G + gam) * D + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const floatx16 o = oacc[dt];
        *reinterpret_cast<u32x2*>(orow + 32 * dt + 8 * a) =
            u32x2{cvt_pk_bf16(o[4 * a] * inv, o[4 * a + 1] * inv),
                  cvt_pk_bf16(o[4 * a + 2] * inv, o[4 * a + 3] * inv)};
      }
  }
}

template <bool KV8, bool PART>
int32_t launch_tiles(int head_dim, int waves, int num_work, const AttnParams& prm,
                     hipStream_t stream) {
  const dim3 grid(prm.Hkv, num_work), block(waves * 64);
  if (head_dim == 64 && waves == 4)
    hipLaunchKernelGGL((attn_tile_kernel<64, 4, KV8, PART>), grid, block, 0, stream, prm);
  else if (head_dim == 128 && waves == 4)
    hipLaunchKernelGGL((attn_tile_kernel<128, 4, KV8, PART>), grid, block, 0, stream, prm);
  else if (head_dim == 128 && waves == 8)
    hipLaunchKernelGGL((attn_tile_kernel<128, 8, KV8, PART>), grid, block, 0, stream, prm);
  else {
    set_error("attention tiles: head_dim %d, %d waves", head_dim, waves);
    return NSG_ERR_ARG;
  }
  return launch_status("attn_tile_kernel");
}

}  // namespace
}  // namespace nsg
