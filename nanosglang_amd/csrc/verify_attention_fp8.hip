// Verify attention over the 8-bit KV pool (format: fp8_kv.hpp): the same plans,
// masks, partials and merge as verify_attention.hip, K and V read as e4m3 codes
// with one power-of-two scale per token and KV head.
//
//   s[r, j] = sm_scale * q_r . (2^(ek_j - 127) kcode_j),   j <= causal limit of r
//   o_r     = sum_j p[r, j] 2^(ev_j - 127) vcode_j / sum_j p[r, j]
//
// Reference semantics: nano_sglang/model/causal_lm.py:359-471 on the pool's
// values.  A long context is bound by the K / V stream, which is half of the
// bf16 pool's, a decode step's by memory round trips.  Codes are exact in bf16,
// so both products run on bf16 MFMA with Q unrounded; K's scale rides in the
// conversion (a lane's K fragment is one token), V's multiplies the
// probabilities (a lane's V fragment is one column of eight tokens).
//
// Per workgroup RT * KS waves: KS groups take contiguous shares of the item's
// 64-token steps, wave w of a group rows [16 w, 16 w + 16).  Per step:
//   * K and V rows and the 128 scale bytes go straight to an LDS ring slot
//     (global_load_lds, 16 bytes a lane for codes, one byte widened to a dword
//     for scales);
//   * S^T = K Q^T on 16x16x32 MFMA (M = tokens, N = query rows).  The order of
//     the products' k index is free as long as K and Q share it: lane group g
//     takes columns D/4 g .. D/4 (g + 1), so a lane reads its K codes in whole
//     16-byte chunks;
//   * P^T in bf16 is the B operand of O^T += V^T P^T; ds_read_b64_tr_b8 gives
//     a lane the 8 tokens of its column.
// 64 tokens of 8-bit rows are the bytes of 32 bf16 ones: the same bytes in
// flight per ring slot, half the steps.
#include "attention.hpp"
#include "fp8_kv.hpp"

namespace nsg {
namespace {

constexpr int kTok = 64;          // KV tokens per step
constexpr int kListPages = 768;   // page ids staged in LDS; an item's later ones are read from memory
constexpr int kHeader = 256;      // workspace: flags word + padding
constexpr int ring_slots(int KS) { return KS == 1 ? 3 : 4; }
constexpr int groups_of(int D) { return D == 64 ? 4 : 2; }

typedef int i32x2 __attribute__((ext_vector_type(2)));

// LDS tile swizzles: 16-byte chunk c of token row t is stored at chunk c ^ f(t).
// K: 16 consecutive tokens' reads of one chunk fall on 16 different 16-byte
// bank groups; V: so do the 16 rows (4 a + b and 16 + 4 a + b, a < 2) that half
// a wave reads transposed.
template <int D>
__device__ __forceinline__ int swz8_k(int t) {
  return D == 64 ? (t >> 2) & 3 : (t >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int swz8_v(int t) {
  return D == 64 ? ((t >> 2) & 1) | ((t >> 3) & 2) : ((t >> 1) & 3) | ((t >> 2) & 4);
}

// LDS DMA in asm: the compiler's wait-count pass, which would wait for every
// copy in flight before each LDS read, does not see these; the ring's own
// waits order them.  Lane l lands at lds + 16 l (codes), lds + 4 l (a scale
// byte, zero-extended).  NT: no reuse expected.
// Source: a wave-uniform base plus 32 bits a lane, or a lane's own address.
template <bool NT>
__device__ __forceinline__ void dma_codes(uint32_t lds, uint64_t base, uint32_t off) {
  if constexpr (NT)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :
                 : "s"(lds), "v"(off), "s"(base)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(off), "s"(base)
                 : "memory", "m0");
}
__device__ __forceinline__ void dma_codes(uint32_t lds, const uint8_t* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(src)
               : "memory", "m0");
}
__device__ __forceinline__ void dma_scale(uint32_t lds, const uint8_t* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off"
               :
               : "s"(lds), "v"(src)
               : "memory", "m0");
}

template <int D, int RT, int KS>
__global__ __launch_bounds__(RT * KS * 64) void verify_attn_fp8_kernel(AttnParams p) {
  constexpr int KC = D / 32;            // k chunks of S^T = K Q^T
  constexpr int DT = D / 16;            // d tiles of O^T
  constexpr int CPR = D / 16;           // 16-byte chunks per token row
  constexpr int TPI = 64 / CPR;         // token rows per DMA instruction
  constexpr int NBLK = kTok / TPI;      // row blocks per step (K and V each)
  constexpr int NB = (NBLK + RT - 1) / RT;   // row blocks a wave copies
  constexpr int NS = RT == 1 ? 2 : 1;   // scale instructions a wave issues
  constexpr int NI = 2 * NB + NS;
  constexpr int TILE = kTok * D;        // bytes of a K (or V) tile
  constexpr int SLOT = 2 * TILE + 2 * kTok * 4;
  constexpr int NBUF = ring_slots(KS);
  constexpr int ROWS = RT * 16;
  constexpr int PSTRIDE = D + 4;        // partial row: O[D], m, l, 2 pad
  constexpr int NTHR = RT * KS * 64;
  static_assert((NBUF - 1) * NI <= 63, "vmcnt counts to 63");
  static_assert(KS * ROWS * PSTRIDE * 4 <= KS * NBUF * SLOT, "combine partials fit the rings");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[KS * NBUF * SLOT];
  __shared__ int s_pages[kListPages];

  int wi = blockIdx.y;
  int h = blockIdx.x;
  if constexpr (D == 64 && KS == 1) {
    // Two heads' rows of 64 bytes share a cache line: workgroups L and L + 8,
    // which the round-robin puts on one XCD, take the two heads of a pair, so
    // that a line comes to one L2 instead of two.  40 requests x 2 rows over
    // 1000 - 5000 tokens, 16 heads of 64: 97 us without, 76.5 with; 64 x 5 rows over
    // 1000 - 8192, 2 KV heads: 43 and 36.  Several KV groups, short contexts: 5.0 us
    // without, 5.2 with (one request of 350 tokens).  Blocks of 16, the last as
    // wide as it is.
    if ((p.Hkv & 1) == 0) {
      const uint32_t n = gridDim.x * gridDim.y, l = blockIdx.y * gridDim.x + blockIdx.x;
      const uint32_t b0 = l & ~15u, half = min(16u, n - b0) / 2, at = l - b0;
      const uint32_t odd = at >= half ? 1 : 0;
      const uint32_t pair = b0 / 2 + (odd ? at - half : at);
      const uint32_t pairs = gridDim.x / 2;  // of an item
      wi = (int)(pair / pairs);
      h = (int)(2 * (pair - (uint32_t)wi * pairs) + odd);
    }
  }
  const int* wk = p.work + (size_t)wi * NSG_ATTN_WORK_INTS;
  const int qs = wk[0], qn = wk[1], lim0 = wk[2], pb = wk[3], kvb = wk[4], kve = wk[5];
  const int nsplit = wk[6];
  if (qn == 0) return;  // padding item of a fixed-size work list
  const int P = 1 << p.log2P;
  const int G = p.G;
  const int nrows = qn * G;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wid / RT;
  const int wave = wid % RT;
  const int r16 = lane & 15;
  const int g4 = lane >> 4;

  // this group's share of the item's steps
  const int n_all = (kve - kvb + kTok - 1) / kTok;
  const int per = (n_all + KS - 1) / KS;
  const int n_it = max(0, min(per, n_all - grp * per));
  const int gkvb = kvb + grp * per * kTok;
  const int last_tok = kve - 1;

  // Page ids: a step takes one a lane (of token t0 + lane).  Those of the first
  // steps come straight from memory, beside Q; the item's list goes to LDS for
  // the later ones.
  const int page0 = kvb >> p.log2P;
  const int npages = kve > kvb ? (last_tok >> p.log2P) - page0 + 1 : 0;
  int vp[NBUF - 1];
#pragma unroll
  for (int it = 0; it < NBUF - 1; ++it)
    vp[it] = n_it ? p.kv_indices[pb + (min(gkvb + it * kTok + lane, last_tok) >> p.log2P)] : 0;
  int list_id = per > NBUF - 1 && tid < npages ? p.kv_indices[pb + page0 + tid] : 0;

  // this lane's query row and its causal limit (rows past the tile's end load
  // its first row, all their scores masked)
  const int row = wave * 16 + r16;
  const bool row_ok = row < nrows;
  const int tau = row / G;
  const int gam = row - tau * G;
  const int lim = row_ok ? lim0 + (p.causal ? tau : 0) : -1;
  bf16x8 qf[KC];
  {
    const bf16* qrow = p.q + (row_ok ? ((size_t)(qs + tau) * p.Hq + h * G + gam) * D
                                     : ((size_t)qs * p.Hq + h * G) * D);
#pragma unroll
    for (int c = 0; c < KC; ++c) qf[c] = load_bf16x8(qrow + (D / 4) * g4 + 8 * c);
  }
#pragma unroll
  for (int c = 0; c < KC; ++c) asm volatile("" ::"v"(__builtin_bit_cast(u32x4, qf[c])));

  floatx4 oacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) oacc[dt] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m_run = kMaskVal, l_run = 0.f;
  bool bad_page = false;

  const uint32_t ring0 = __builtin_amdgcn_readfirstlane(lds_addr(ring) + grp * (NBUF * SLOT));
  const uint8_t* gring = ring + grp * (NBUF * SLOT);
  const uint32_t tok_bytes = (uint32_t)(p.Hkv * D);
  const uint32_t page_bytes = tok_bytes << p.log2P;  // (below 2^31: checked at the entry point)
  const uint32_t scale_bytes = (uint32_t)(2 * p.Hkv) << p.log2P;
  // A lane's source offset inside a block of TPI token rows, for K and V
  // (block 0; the swizzles of block `blk` differ in one bit), and its scale's.
  const int tr = lane / CPR, pc = lane % CPR;
  const uint32_t row_off = (uint32_t)tr * tok_bytes;
  const uint32_t koff0 = row_off + (pc ^ swz8_k<D>(tr)) * 16;
  const uint32_t voff0 = row_off + (pc ^ swz8_v<D>(tr)) * 16;
  const uint8_t* sbase = p.kv_scale + ((size_t)(2 * h) << p.log2P);
  // This wave's copies of step `it` into slot `slot`, given its page ids.
  auto issue = [&](int it, int slot, int pg) {
    const int t0 = gkvb + it * kTok;
    const uint32_t sb = ring0 + (uint32_t)slot * SLOT;
    if ((unsigned)pg >= (unsigned)p.num_pages) {
      bad_page = true;  // reads the pool's first page instead
      pg = 0;
    }
    if (P >= TPI && t0 + kTok <= kve) {
      // a block's rows lie on one page: scalar addresses
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int blk = (wave + RT * i) % NBLK;  // (a padding copy repeats a real one)
        const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(pg, blk * TPI);
        const uint64_t off = (uint64_t)page * page_bytes +
                             (uint32_t)((t0 + blk * TPI) & (P - 1)) * tok_bytes + (uint32_t)(h * D);
        const uint32_t dst = sb + blk * (TPI * D);
        dma_codes<KS == 1>(dst, (uint64_t)p.kc8 + off, koff0 ^ ((swz8_k<D>(blk * TPI)) * 16));
        dma_codes<KS == 1>(dst + TILE, (uint64_t)p.vc8 + off, voff0 ^ ((swz8_v<D>(blk * TPI)) * 16));
      }
    } else {
      // small pages, or the item's last step, where tokens past the end
      // repeat the last one (masked out)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int blk = (wave + RT * i) % NBLK;
        const int t = blk * TPI + tr;
        const int tok = min(t0 + t, last_tok);
        const uint32_t page = (uint32_t)__shfl(pg, t);
        const size_t off = (size_t)page * page_bytes + (uint32_t)(tok & (P - 1)) * tok_bytes +
                           (uint32_t)(h * D);
        const uint32_t dst = sb + blk * (TPI * D);
        dma_codes(dst, p.kc8 + off + (pc ^ swz8_k<D>(t)) * 16);
        dma_codes(dst + TILE, p.vc8 + off + (pc ^ swz8_v<D>(t)) * 16);
      }
    }
    const int tok = min(t0 + lane, last_tok);
    const uint8_t* so = sbase + (size_t)(uint32_t)pg * scale_bytes + (tok & (P - 1));
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int which = RT == 1 ? i : wave & 1;
      dma_scale(sb + 2 * TILE + which * (kTok * 4), so + ((size_t)which << p.log2P));
    }
  };

  // LDS read offsets: K codes of sub-tile s are rows 16 s + r16; V^T fragment
  // (m, dt): rows 32 m + vt, 16-byte chunk dt
  int koff[KC / 2];
#pragma unroll
  for (int c = 0; c < KC / 2; ++c)
    koff[c] = r16 * D + (((KC / 2) * g4 + c) ^ swz8_k<D>(r16)) * 16;
  const int vj = r16 >> 1;
  const int vt = 4 * g4 + (vj & 3) + 16 * (vj >> 2);
  const int voff = vt * D + 8 * (r16 & 1);
  const int vswz = swz8_v<D>(vt);

  // (all ids have landed before any copy is issued: the compiler's wait for
  // one of them would otherwise drain the copies)
#pragma unroll
  for (int it = 0; it < NBUF - 1; ++it) asm volatile("" ::"v"(vp[it]));
  asm volatile("" : "+v"(list_id));
#pragma unroll
  for (int it = 0; it < NBUF - 1; ++it)
    if (it < n_it) issue(it, it, vp[it]);
  // the page list, where there are later steps (the same for every wave)
  const bool long_list = npages > kListPages;
  if (per > NBUF - 1) {
    if (tid < kListPages) s_pages[tid] = list_id;
    for (int i = tid + NTHR; i < min(npages, kListPages); i += NTHR)
      s_pages[i] = p.kv_indices[pb + page0 + i];
    __syncthreads();
  }
  auto step_pages = [&](int it) {
    const int i = (min(gkvb + it * kTok + lane, last_tok) >> p.log2P) - page0;
    int pg = s_pages[min(i, kListPages - 1)];
    // (kept apart from the load below: one load from either address would be a
    // flat load, whose wait drains the ring)
    asm volatile("" : "+v"(pg));
    if (long_list && i >= kListPages) pg = p.kv_indices[pb + page0 + i];
    return pg;
  };

  const int n_loop = RT == 1 ? n_it : per;  // groups of several waves keep their barriers matched
  int slot = 0;
  for (int it = 0; it < n_loop; ++it) {
    const bool real = RT == 1 || it < n_it;
    // step `it` landed; the later ones issued so far stay in flight
    if (real) wait_steps<NI, NBUF - 2>(min(n_it - 1 - it, NBUF - 2));
    // every LDS read of this wave has returned: the slot of step it - 1 is free
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (RT > 1) {
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    if (it + NBUF - 1 < n_it)
      issue(it + NBUF - 1, slot == 0 ? NBUF - 1 : slot - 1, step_pages(it + NBUF - 1));
    const uint8_t* Kt = gring + slot * SLOT;
    slot = slot + 1 == NBUF ? 0 : slot + 1;
    if (!real || wave * 16 >= nrows) continue;  // (no row of this wave: it only copies)
    const uint8_t* Vt = Kt + TILE;
    const uint32_t* sk = reinterpret_cast<const uint32_t*>(Kt + 2 * TILE);
    const uint32_t* sv = sk + kTok;
    const int t0 = gkvb + it * kTok;

    // ---- S^T: lane holds tokens 16 s + 4 g4 + i of query row r16 ----
    floatx4 sacc[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const float ks = e8m0_scale(sk[16 * s + r16]);
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC / 2; ++c) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(Kt + 16 * s * D + koff[c]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const fp8_u32x2 a = from_fp8x4(w[2 * x], ks), b = from_fp8x4(w[2 * x + 1], ks);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]}), qf[2 * c + x], acc, 0, 0,
              0);
        }
      }
      sacc[s] = acc;
    }

    // ---- online softmax (base 2, lazy rescaling) ----
    u32x4 pf[2];
    auto softmax = [&](auto masked) {
      constexpr bool MASKED = decltype(masked)::value;
      float mx = kMaskVal;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (MASKED) {
            const int j = t0 + 16 * s + 4 * g4 + i;
            if (j > lim || j >= kve) sacc[s][i] = kMaskVal;
          }
          mx = fmaxf(mx, sacc[s][i]);
        }
      mx = max_xor16_32(mx);
      mx = (MASKED && mx == kMaskVal) ? kMaskVal : mx * p.scale_log2;
      const bool grow = mx > m_run + kLazyRescale;
      if (__builtin_amdgcn_ballot_w64(grow)) {
        const float mnew = grow ? mx : m_run;
        const float alpha = __builtin_amdgcn_exp2f(m_run - mnew);
        m_run = mnew;
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
      }
      float ps = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const u32x4 e = *reinterpret_cast<const u32x4*>(sv + 16 * s + 4 * g4);
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = __builtin_amdgcn_exp2f(fmaf(sacc[s][i], p.scale_log2, -m_run));
          const bool out = MASKED && sacc[s][i] == kMaskVal;
          ps += out ? 0.f : x;
          w[i] = out ? 0.f : x * e8m0_scale(e[i]);
        }
        pf[s >> 1][2 * (s & 1)] = cvt_pk_bf16(w[0], w[1]);
        pf[s >> 1][2 * (s & 1) + 1] = cvt_pk_bf16(w[2], w[3]);
      }
      l_run += ps;
    };
    if (t0 + kTok - 1 <= lim0 && t0 + kTok <= kve)
      softmax(std::false_type{});  // every row of the tile sees every token
    else
      softmax(std::true_type{});

    // ---- O^T += V^T P^T; element e of lane group g4 is token 32 m + 4 g4 + e
    //      (e < 4) or 32 m + 16 + 4 g4 + e - 4 ----
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(Vt + 32 * m * D + voff + ((dt ^ vswz) << 4)));
        const fp8_u32x2 a = from_fp8x4((uint32_t)w[0], 1.f), b = from_fp8x4((uint32_t)w[1], 1.f);
        oacc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]}),
            __builtin_bit_cast(bf16x8, pf[m]), oacc[dt], 0, 0, 0);
      }
  }

  if (bad_page) atomicOr(p.flags, 1);
  const float l = sum_xor16_32(l_run);
  float* prow = p.partials + ((size_t)wi * p.Hkv + h) * ROWS * PSTRIDE + (size_t)row * PSTRIDE;
  bf16* orow = p.out + ((size_t)(qs + tau) * p.Hq + h * G + gam) * D + 4 * g4;
  if constexpr (KS == 1) {
    if (!row_ok) return;
    if (nsplit == 1) {
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // l NaN stays NaN
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const floatx4 o = oacc[dt];
        *reinterpret_cast<u32x2*>(orow + dt * 16) =
            u32x2{cvt_pk_bf16(o[0] * inv, o[1] * inv), cvt_pk_bf16(o[2] * inv, o[3] * inv)};
      }
    } else {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<floatx4*>(prow + dt * 16 + 4 * g4) = oacc[dt];
      if (g4 == 0) {
        prow[D] = m_run;
        prow[D + 1] = l;
      }
    }
  } else {
    // ---- the KV groups meet in LDS: every group writes its partial rows,
    //      group g finishes d tiles g, g + KS, ... ----
    constexpr int OWN = DT / KS;
    static_assert(DT % KS == 0, "d tiles split evenly over the KV groups");
    __syncthreads();  // the rings are idle
    float* sc = reinterpret_cast<float*>(ring);
    {
      float* mine = sc + ((size_t)grp * ROWS + row) * PSTRIDE;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<floatx4*>(mine + dt * 16 + 4 * g4) = oacc[dt];
      *reinterpret_cast<floatx2*>(mine + D) = floatx2{m_run, l};
    }
    __syncthreads();
    float mg[KS], lg[KS], M = kMaskVal;
#pragma unroll
    for (int g = 0; g < KS; ++g) {
      const floatx2 ml = *reinterpret_cast<const floatx2*>(sc + ((size_t)g * ROWS + row) * PSTRIDE + D);
      mg[g] = ml[0];
      lg[g] = ml[1];
      M = fmaxf(M, ml[0]);
    }
    float lsum = 0.f;
    floatx4 acc[OWN];
#pragma unroll
    for (int j = 0; j < OWN; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < KS; ++g) {
      const float w = __builtin_amdgcn_exp2f(mg[g] - M);
      lsum += w * lg[g];
      const float* o = sc + ((size_t)g * ROWS + row) * PSTRIDE + 4 * g4;
#pragma unroll
      for (int j = 0; j < OWN; ++j)
        acc[j] += w * *reinterpret_cast<const floatx4*>(o + (grp + KS * j) * 16);
    }
    if (!row_ok) return;
    if (nsplit == 1) {
      const float inv = lsum > 0.f ? 1.f / lsum : (lsum == 0.f ? 0.f : lsum);
#pragma unroll
      for (int j = 0; j < OWN; ++j) {
        const floatx4 o = acc[j];
        *reinterpret_cast<u32x2*>(orow + (grp + KS * j) * 16) =
            u32x2{cvt_pk_bf16(o[0] * inv, o[1] * inv), cvt_pk_bf16(o[2] * inv, o[3] * inv)};
      }
    } else {
#pragma unroll
      for (int j = 0; j < OWN; ++j)
        *reinterpret_cast<floatx4*>(prow + (grp + KS * j) * 16 + 4 * g4) = acc[j];
      if (g4 == 0 && grp == 0) {
        prow[D] = M;
        prow[D + 1] = lsum;
      }
    }
  }
}

template <int D, int RT>
int32_t launch_rt(const nsg_attn_plan_t* plan, const AttnParams& prm, hipStream_t stream) {
  const dim3 grid(plan->num_kv_heads, plan->num_work);
  constexpr int KSX = groups_of(D);
  if (plan->kv_groups == KSX)
    hipLaunchKernelGGL((verify_attn_fp8_kernel<D, RT, KSX>), grid, dim3(RT * KSX * 64), 0, stream,
                       prm);
  else if (plan->kv_groups == 1)
    hipLaunchKernelGGL((verify_attn_fp8_kernel<D, RT, 1>), grid, dim3(RT * 64), 0, stream, prm);
  else {
    set_error("kv_groups %d not supported for head_dim %d", plan->kv_groups, D);
    return NSG_ERR_ARG;
  }
  return launch_status("verify_attn_fp8_kernel");
}

template <int D>
int32_t launch_d(const nsg_attn_plan_t* plan, const AttnParams& prm, hipStream_t stream) {
  switch (plan->row_tiles) {
    case 1: return launch_rt<D, 1>(plan, prm, stream);
    case 2: return launch_rt<D, 2>(plan, prm, stream);
    case 3: return launch_rt<D, 3>(plan, prm, stream);
    case 4: return launch_rt<D, 4>(plan, prm, stream);
    default: set_error("row_tiles %d out of range", plan->row_tiles); return NSG_ERR_ARG;
  }
}

}  // namespace

int32_t launch_verify_attn_fp8(const nsg_attn_plan_t* plan, const AttnParams& prm,
                               hipStream_t stream) {
  return plan->head_dim == 64 ? launch_d<64>(plan, prm, stream) : launch_d<128>(plan, prm, stream);
}

}  // namespace nsg

using namespace nsg;

extern "C" int32_t nsg_attn_run_fp8(const nsg_attn_plan_t* plan, const int32_t* work_d,
                                    const void* q, const void* k_cache, const void* v_cache,
                                    const void* kv_scale, void* out, const int32_t* kv_indices,
                                    int32_t page_size, int32_t num_pages, float sm_scale,
                                    int32_t causal, void* workspace, int64_t workspace_bytes,
                                    nsg_stream_t stream) {
  NSG_CHECK_ARG(plan != nullptr, "null plan");
  if (plan->num_work == 0) {
    clear_error();
    return NSG_OK;
  }
  NSG_CHECK_ARG(work_d && q && k_cache && v_cache && kv_scale && out && kv_indices && workspace,
                "null pointer argument");
  NSG_CHECK_ARG(page_size > 0 && (page_size & (page_size - 1)) == 0,
                "page_size %d must be a power of two", page_size);
  NSG_CHECK_ARG(num_pages > 0, "num_pages %d", num_pages);
  NSG_CHECK_ARG(sm_scale > 0.f, "sm_scale %g must be positive", (double)sm_scale);
  NSG_CHECK_ARG((int64_t)page_size * plan->num_kv_heads * plan->head_dim < 1ll << 31,
                "a page of %d tokens is too large", page_size);
  NSG_CHECK_ARG(((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)q | (uintptr_t)out) % 16 == 0,
                "q, out and the caches must be 16-byte aligned");
  if (plan->head_dim != 64 && plan->head_dim != 128) {
    set_error("head_dim %d not supported", plan->head_dim);
    return NSG_ERR_UNSUPPORTED;
  }
  if (workspace_bytes < plan->workspace_bytes) {
    set_error("workspace has %lld bytes, plan needs %lld", (long long)workspace_bytes,
              (long long)plan->workspace_bytes);
    return NSG_ERR_WORKSPACE;
  }
  AttnParams prm{};
  prm.q = static_cast<const bf16*>(q);
  prm.kc8 = static_cast<const uint8_t*>(k_cache);
  prm.vc8 = static_cast<const uint8_t*>(v_cache);
  prm.kv_scale = static_cast<const uint8_t*>(kv_scale);
  prm.out = static_cast<bf16*>(out);
  prm.kv_indices = kv_indices;
  prm.work = work_d;
  prm.num_work = plan->num_work;
  prm.Hq = plan->num_qo_heads;
  prm.Hkv = plan->num_kv_heads;
  prm.G = plan->num_qo_heads / plan->num_kv_heads;
  prm.log2P = __builtin_ctz((unsigned)page_size);
  prm.num_pages = num_pages;
  prm.causal = causal ? 1 : 0;
  prm.scale_log2 = sm_scale * 1.4426950408889634f;
  char* ws = static_cast<char*>(workspace);
  prm.flags = reinterpret_cast<int*>(ws);
  prm.partials = reinterpret_cast<float*>(ws + kHeader);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (plan->row_tiles == 8 || plan->row_tiles == 16) {
    NSG_CHECK_ARG(plan->max_splits == 1 && plan->num_merge == 0,
                  "prefill tiles are never split: plan has %d KV splits, %d merge items",
                  plan->max_splits, plan->num_merge);
    return launch_prefill_attn_fp8(plan->head_dim, plan->row_tiles / 2, plan->num_work, prm, s);
  }
  if (int32_t rc = launch_verify_attn_fp8(plan, prm, s)) return rc;
  if (plan->num_merge == 0) return NSG_OK;
  return launch_attn_merge(plan, prm, work_d + (size_t)plan->num_work * NSG_ATTN_WORK_INTS, s);
}
