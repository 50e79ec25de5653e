// Attention for a batch whose requests share the first part of their context:
// groups of consecutive requests, each with one prefix on shared pages, then
// every request's own tokens on its own pages.
//
//   o_r = sum over prefix and own tokens of softmax(sm_scale q_r . k) v,
//
// the prefix visible to every row of its group, the own part under the
// bottom-right causal rule (nano_sglang/model/causal_lm.py:359-471 over the
// concatenated context; the shared pages are what RadixCache.match_prefix,
// nano_sglang/engine/radix_cache.py:68, hands to several requests).
//
// The prefix is attended to once per group: its query tiles run over the
// group's packed query tokens as if they were one request, so K and V of the
// prefix are read once per tile of up to 256 rows instead of once per request,
// and a decode step's few rows per request fill MFMA tiles together.  The own
// parts and the prefix tiles leave partial rows (O, m, l; the kernels of
// verify_attention.hip, verify_attention_fp8.hip and prefill_tiles.hpp, over
// shares of the KV range), in one launch where groups have few rows, else in
// two; the merge below joins a row's partials of both.
#include <algorithm>
#include <vector>

#include "attention.hpp"

namespace nsg {
namespace {

constexpr int64_t kHeader = 256;   // workspace: flags word + padding
constexpr int kThreads = 256;
constexpr int kBatch = 8;          // partial rows whose loads a merge thread has in flight
constexpr int kAll = 0x3fffffff;   // causal limit of prefix tiles: everything is visible
constexpr int kStep = 64;          // shares of a prefix are whole steps of this many tokens

struct MergeParams {
  const int* merge;
  const float* own;      // partial rows of the own parts, own_rows per item and KV head
  const float* prefix;   // ... of the prefix tiles
  bf16* out;
  int own_rows, prefix_rows, prefix_tokens;  // rows per item; query tokens per prefix tile
  int Hq, Hkv, G;
};

// Merge item: [first query token, query tokens, first own item, own splits,
// the group's first prefix item, its shares, its first query token, its prefix
// tiles]; a tile's shares are that many items apart.  A piece
// is 8 columns of a row; its partials are folded in batches of kBatch, whose
// loads are in flight together, by one lane, or (LANES = 4, few pieces: memory
// round trips count) every fourth by each of the lanes l, l + 16, l + 32, l + 48 of
// a wave, which then meet: 32 decode rows of 32 heads of 128 with 16 / 64 partials
// 5.3 / 14 -> 4.3 / 10 us, but 576 rows with 8 partials 11.8 -> 24.
template <int D, int LANES>
__global__ __launch_bounds__(kThreads) void prefix_merge_kernel(MergeParams p) {
  constexpr int PSTRIDE = D + 4;
  constexpr int CH = D / 8;
  const int* mw = p.merge + (size_t)blockIdx.x * NSG_ATTN_WORK_INTS;
  const int qs = mw[0], qn = mw[1], wi0 = mw[2], ns = mw[3], pw0 = mw[4], pns = mw[5];
  const int lane = threadIdx.x & 63;
  const int sub = LANES == 4 ? lane >> 4 : 0;
  const int item = LANES == 4 ? ((int)blockIdx.z * (kThreads / 64) + (int)(threadIdx.x >> 6)) * 16 +
                                    (lane & 15)
                              : (int)blockIdx.z * kThreads + (int)threadIdx.x;
  if (item >= qn * p.G * CH) return;  // whole pieces; a padding item has no query tokens
  const int h = blockIdx.y;
  const int row = item / CH;
  const int c0 = (item - row * CH) * 8;
  const int tau = row / p.G;
  const int gam = row - tau * p.G;
  const int at = qs + tau - mw[6];  // the token's place in its group
  const int tile = at / p.prefix_tokens;
  const int prow = (at - tile * p.prefix_tokens) * p.G + gam;
  const float* own = p.own + (((size_t)wi0 * p.Hkv + h) * p.own_rows + row) * PSTRIDE;
  const size_t own_step = (size_t)p.Hkv * p.own_rows * PSTRIDE;
  const float* pre =
      p.prefix + (((size_t)(pw0 + tile) * p.Hkv + h) * p.prefix_rows + prow) * PSTRIDE;
  const size_t pre_step = (size_t)mw[7] * p.Hkv * p.prefix_rows * PSTRIDE;
  float M = kMaskVal, lsum = 0.f;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int n = ns + pns;
  for (int s0 = sub; s0 < n; s0 += LANES * kBatch) {
    floatx4 ml[kBatch], a[kBatch], b[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {  // past the last: re-reads it
      const int s = min(s0 + LANES * j, n - 1);
      const float* r = s < ns ? own + s * own_step : pre + (s - ns) * pre_step;
      ml[j] = *reinterpret_cast<const floatx4*>(r + D);
      a[j] = *reinterpret_cast<const floatx4*>(r + c0);
      b[j] = *reinterpret_cast<const floatx4*>(r + c0 + 4);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (s0 + LANES * j >= n) break;
      const float Mn = fmaxf(M, ml[j][0]);
      const float sc = __builtin_amdgcn_exp2f(M - Mn);
      const float wt = __builtin_amdgcn_exp2f(ml[j][0] - Mn);
      lsum = lsum * sc + wt * ml[j][1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = o[i] * sc + wt * a[j][i];
        o[4 + i] = o[4 + i] * sc + wt * b[j][i];
      }
      M = Mn;
    }
  }
  if constexpr (LANES == 4) {
    const float sc = __builtin_amdgcn_exp2f(M - max_xor16_32(M));
    lsum = sum_xor16_32(lsum * sc);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = sum_xor16_32(o[i] * sc);
    if (sub) return;
  }
  const float inv = lsum > 0.f ? 1.f / lsum : (lsum == 0.f ? 0.f : lsum);
  bf16* orow = p.out + ((size_t)(qs + tau) * p.Hq + h * p.G + gam) * D + c0;
  *reinterpret_cast<u32x4*>(orow) =
      u32x4{cvt_pk_bf16(o[0] * inv, o[1] * inv), cvt_pk_bf16(o[2] * inv, o[3] * inv),
            cvt_pk_bf16(o[4] * inv, o[5] * inv), cvt_pk_bf16(o[6] * inv, o[7] * inv)};
}

// Rows of a prefix tile for groups of at most `rows` rows: the verify kernel's
// 16-row tiles up to 64, the prefill kernel's 128 or (head dim 128) 256 beyond.
int prefix_rows(int64_t rows, int head_dim) {
  if (rows <= 64) return (int)std::max<int64_t>(16, (rows + 15) / 16 * 16);
  return rows <= 128 || head_dim == 64 ? 128 : 256;
}

// Estimated times (us).  A kernel: a workgroup's start and 64-token step.  From 66
// runs of prefixes of 2048 - 16384 tokens at 1 - 64 steps per item; within 10 % where
// the steps count.  (128 rows, 32 / 8 heads of 128, 4096 tokens: 32 / 16 / 8 / 4 items
// a head 14.2 / 15.5 / 18.6 / 27.0; 2304 rows, 8192 tokens: 18 / 27 / 36 / 54 / 72 items
// 133 / 100 / 140 / 109 / 127, 36 being just over a round of workgroups.)
struct TileFit {
  double start, step;
};
TileFit tile_fit(int rows, int head_dim) {
  if (rows <= 64) return head_dim == 64 ? TileFit{4.0, 0.37} : TileFit{5.0, 0.85};
  if (head_dim == 64) return {5.5, 0.95};
  return rows == 128 ? TileFit{8.0, 1.35} : TileFit{6.0, 2.25};
}
// The partial rows of a prefix written and read again, and the merge's round trips.
double partials_us(int64_t wgs, int rows, int head_dim, int shares) {
  return 2.0 * wgs * rows * (head_dim + 4) * 4 / 5.0e6 + 0.12 * shares;
}
// One launch of items of at most `longest` steps, `steps` over all workgroups, where a
// CU's workgroups take turns: a start per round, and the steps over the CUs with
// a third of the longest item left over at the end (in whole items where all
// are alike).
double launch_us(const TileFit& f, int64_t wgs, double steps, int64_t longest, bool alike,
                 int num_cus) {
  const int64_t rounds = (wgs + num_cus - 1) / num_cus;
  return alike ? f.start + f.step * longest * rounds
               : f.start * rounds +
                     f.step * std::max((double)longest, steps / num_cus + 0.3 * longest);
}
constexpr double kLaunchGap = 1.5;
// One launch of tiles of up to 64 rows with one KV group, several workgroups to a
// CU: the longest item's steps, or the CU's share of all steps (of the prefix, which
// comes from L2, and of own parts) and a third of the longest item's.
double shared_us(int head_dim, double steps, double own_steps, int64_t longest, int num_cus) {
  const bool d64 = head_dim == 64;
  const double item = (d64 ? 1.27 : 1.84) * longest;
  const double all = d64 ? 0.8 * steps + 0.6 * own_steps : steps + 1.2 * own_steps;
  return (d64 ? 6.0 : 11.0) + std::max(item, all / num_cus + 0.35 * item);
}
// The own parts' launch, with one KV group.
double own_us(int head_dim, double own_steps, int64_t longest, int num_cus) {
  const double step = head_dim == 64 ? 0.8 : 1.2, all = head_dim == 64 ? 0.8 : 1.6;
  return 4.0 + std::max(step * longest, all * own_steps / num_cus);
}
constexpr int kFixedJointRows = 512;  // fixed plans: one launch up to so many rows

struct Sizes {
  bool fixed;
  int max_batch, max_q_len, max_kv_len, max_work, max_prefix_work, max_merge;
};

int32_t plan_impl(const int32_t* qo, const int32_t* groups, int32_t num_groups,
                  const int32_t* pkv, const int32_t* plast, const int32_t* kvp,
                  const int32_t* last, int32_t batch, int32_t Hq, int32_t Hkv, int32_t head_dim,
                  int32_t page_size, int32_t causal, int32_t num_cus, const Sizes& sz,
                  int32_t* work_h, int32_t work_capacity, nsg_prefix_attn_plan_t* plan) {
  NSG_CHECK_ARG(plan && qo && groups && pkv && plast && kvp && last, "null argument");
  NSG_CHECK_ARG(batch >= 0 && num_groups >= 0, "batch %d, %d groups", batch, num_groups);
  NSG_CHECK_ARG(groups[0] == 0 && groups[num_groups] == batch,
                "group_indptr must run from 0 to the batch (%d), has %d .. %d", batch, groups[0],
                groups[num_groups]);
  NSG_CHECK_ARG(pkv[0] == 0, "prefix_kv_indptr must start at 0");
  if (num_cus <= 0) num_cus = 256;
  NSG_CHECK_ARG(Hkv > 0 && Hq > 0 && Hq % Hkv == 0,
                "num_qo_heads %d must be a positive multiple of num_kv_heads %d", Hq, Hkv);
  const int G = Hq / Hkv;
  NSG_CHECK_ARG(page_size > 0, "page_size %d must be a power of two", page_size);
  int64_t most = 0;  // rows of the largest group
  for (int g = 0; g < num_groups; ++g) {
    NSG_CHECK_ARG(groups[g] <= groups[g + 1] && groups[g + 1] <= batch,
                  "group %d: decreasing group_indptr", g);
    const int np = pkv[g + 1] - pkv[g];
    NSG_CHECK_ARG(np >= 0, "group %d: decreasing prefix_kv_indptr", g);
    NSG_CHECK_ARG(np == 0 || (plast[g] >= 1 && plast[g] <= page_size),
                  "group %d: prefix last_page_len %d outside [1, %d]", g, plast[g], page_size);
    NSG_CHECK_ARG(np <= kAll / page_size, "group %d: prefix of %d pages", g, np);
    most = std::max<int64_t>(most, (int64_t)(qo[groups[g + 1]] - qo[groups[g]]) * G);
  }
  if (sz.fixed) most = (int64_t)sz.max_batch * sz.max_q_len * G;
  // ---- the own parts: an attention plan whose items all leave partials.  The
  //      merge is there anyway, so several KV groups per workgroup (a whole CU
  //      per tile of 16 rows) only for up to two rounds of tiles (64 decode
  //      rows of 32 / 8 heads of 128 behind 300 / 4000 tokens 29 / 41 -> 21 / 32 us;
  //      four rounds, 320 rows behind 4000: 61 -> 83) ----
  int64_t tiles16 = 0;
  const int t16 = std::max(1, 16 / G);
  if (sz.fixed)
    tiles16 = (int64_t)sz.max_batch * ((sz.max_q_len + t16 - 1) / t16);
  else
    for (int b = 0; b < batch; ++b) tiles16 += (qo[b + 1] - qo[b] + t16 - 1) / t16;
  const int regime = tiles16 * Hkv <= 2 * num_cus ? 1 : 0;
  std::vector<int32_t> own(1024 * NSG_ATTN_WORK_INTS);
  nsg_attn_plan_t op{};
  for (;;) {
    const int32_t cap = (int32_t)(own.size() / NSG_ATTN_WORK_INTS);
    const int32_t rc = plan_attn(qo, kvp, last, batch, Hq, Hkv, head_dim, page_size, causal,
                                 num_cus, own.data(), cap, sz.fixed ? sz.max_work : -1,
                                 sz.max_merge, sz.max_q_len, sz.max_kv_len, regime, &op);
    if (rc == NSG_OK) break;
    // (a fixed list that is too small stays so whatever the buffer)
    const bool grow = rc == NSG_ERR_WORKSPACE &&
                      (sz.fixed ? cap < sz.max_work + sz.max_merge : cap < (1 << 22));
    if (!grow) return rc;
    own.resize(own.size() * 4);
  }
  // ---- the prefix tiles: steps per item, of the shares that the longest
  //      prefix can be cut into those with the least estimated time; in a launch of
  //      their own, or (tiles of at most 64 rows, each of which reads the prefix)
  //      in one with the own parts, of whichever the estimate is lowest: workgroups
  //      of several KV groups, one to a CU, where few tiles leave time on the table
  //      (32 decode rows of 32 / 8 heads of 128 behind 4001 tokens: apart 33 us
  //      without the merge, joint 24), or of one KV group, several to a CU (128
  //      decode rows behind 1000: apart 40.6 us, joint 27; behind 12000 67 and 87.
  //      576 batches of 2 - 320 rows a request group behind 300 - 12000: 1.05 times
  //      as fast in the mean as with several KV groups only, 0.85 - 1.8). ----
  auto prefix_len = [&](int g) {
    const int np = pkv[g + 1] - pkv[g];
    return np ? (np - 1) * page_size + plast[g] : 0;
  };
  auto steps_of = [&](int g) { return (int64_t)(prefix_len(g) + kStep - 1) / kStep; };
  auto tiles_of = [&](int g, int T) { return (qo[groups[g + 1]] - qo[groups[g]] + T - 1) / T; };
  int64_t longest = 0;
  for (int g = 0; g < num_groups; ++g)
    if (tiles_of(g, 1)) longest = std::max(longest, steps_of(g));
  // an item's page ids must fit the kernels' list
  const int64_t by_pages =
      std::max<int64_t>(1, (int64_t)(kMaxItemPages - 2) * page_size / kStep);
  const int64_t fewest = std::max<int64_t>(1, (longest + by_pages - 1) / by_pages);
  int64_t own_steps = 0, own_items = 0, own_longest = 0;
  for (int i = 0; i < op.num_work; ++i) {
    const int32_t* w = own.data() + (size_t)i * NSG_ATTN_WORK_INTS;
    const int64_t n = (w[5] - w[4] + kStep - 1) / kStep;
    own_steps += n;
    own_items += w[1] > 0;
    own_longest = std::max(own_longest, n);
  }
  // Shares of `chunk` steps; with `rest`, the last one of that many instead.
  struct Choice {
    double us = -1;
    int64_t chunk = 1, rest = 0;
  };
  enum How { Apart, Joint, Shared };  // a launch of its own; with the own parts: in KV groups, in one
  auto choose = [&](int rows, How how) {
    Choice best;
    const TileFit fit = tile_fit(rows, head_dim);
    const int T = std::max(1, rows / G), real_rows = (int)std::min<int64_t>(rows, most);
    for (int64_t n = fewest; n <= std::max(fewest, std::min<int64_t>(longest, 64)); ++n) {
      const int64_t c = std::max<int64_t>(1, (longest + n - 1) / n);
      int64_t items = 0, steps = 0;
      for (int g = 0; g < num_groups; ++g) {
        items += tiles_of(g, T) * ((steps_of(g) + c - 1) / c);
        steps += tiles_of(g, T) * steps_of(g);
      }
      if (sz.fixed && items > sz.max_prefix_work && best.us >= 0) break;
      const double us =
          partials_us(items * Hkv, real_rows, head_dim, (int)n) +
          (how == Shared ? shared_us(head_dim, (double)steps * Hkv, (double)own_steps * Hkv,
                                     std::max(c, own_longest), num_cus)
           : how == Joint
               ? launch_us(fit, (items + own_items) * Hkv, (double)(steps + own_steps) * Hkv,
                           std::max(c, own_longest), false, num_cus)
               : launch_us(fit, items * Hkv, (double)steps * Hkv, c, num_groups == 1, num_cus));
      if (best.us < 0 || us < best.us) best = {us, c, 0};
    }
    // One group's tiles of a whole CU each, n shares of which leave an eighth of
    // the CUs or more without any: those take a last, short share of every tile, r
    // one after the other in the time of one long one (2304 rows behind 8192
    // tokens, 8-bit pool, 9 x 8 tiles: 108 -> 99 us and a merge of 11.4 for 10.2;
    // 45 other batches 1 - 1.19 times as fast, 1.06 in the mean; 660 rows behind
    // 7700, where a sixteenth is idle, 56 -> 62).
    const int64_t tiles = num_groups == 1 ? tiles_of(0, T) * Hkv : 0, n = tiles ? num_cus / tiles : 0;
    if (how == Apart && !sz.fixed && rows == 256 && n >= fewest && (num_cus - n * tiles) * 8 >= num_cus) {
      const int64_t r = (tiles + num_cus - n * tiles - 1) / (num_cus - n * tiles);
      const double again = (r - 1) * fit.start / fit.step;  // steps' worth of their starts
      const int64_t b = (int64_t)((longest - n * again) / (n * r + 1));
      const int64_t c = (longest - b + n - 1) / n;
      const double us = partials_us(tiles * (n + 1), real_rows, head_dim, (int)n + 1) + fit.start +
                        fit.step * std::max((double)c, r * b + again);
      if (b >= 1 && us < best.us) best = {us, c, b};
    }
    return best;
  };
  int rows = prefix_rows(most, head_dim);
  Choice choice = choose(rows, Apart);
  const int joint_rows =
      std::max(op.row_tiles * 16, prefix_rows(std::min<int64_t>(most, 64), head_dim));
  const Choice groups_joint = op.kv_groups > 1 ? choose(joint_rows, Joint) : Choice{};
  const Choice shared = choose(joint_rows, Shared);
  bool one_launch, share_cus;
  if (sz.fixed) {  // (a fixed plan's shape must not depend on the lengths of one step)
    one_launch = most <= kFixedJointRows;
    share_cus = op.kv_groups == 1 || tiles16 * Hkv > num_cus;
  } else {
    const double apart =
        choice.us + kLaunchGap +
        (op.kv_groups > 1 ? launch_us(tile_fit(16, head_dim), own_items * Hkv,
                                      (double)own_steps * Hkv, own_longest, false, num_cus)
                          : own_us(head_dim, (double)own_steps * Hkv, own_longest, num_cus));
    // (workgroups of 16 waves, four KV groups of head dim 64, run late by as much)
    share_cus = op.kv_groups == 1 ||
                shared.us < groups_joint.us * (head_dim == 64 ? 1.15 : 1.0);
    // (below 16 tokens a page both launches would be of the one-group kernel)
    one_launch = longest > 0 && ((rows <= 64 && page_size < 16) ||
                                 (share_cus ? shared.us : groups_joint.us) < apart);
  }
  if (one_launch) {
    rows = joint_rows;
    choice = share_cus ? shared : groups_joint;
    if (share_cus) op.kv_groups = 1;
  }
  const int T = std::max(1, rows / G);
  const int own_rows = one_launch ? rows : op.row_tiles * 16;
  std::vector<int32_t> pre;
  std::vector<int> first(num_groups), splits(num_groups);
  for (int g = 0; g < num_groups; ++g) {
    const int len = prefix_len(g), tiles = tiles_of(g, T), q0 = qo[groups[g]], q1 = qo[groups[g + 1]];
    const int64_t steps = steps_of(g), even = steps - choice.rest;
    const int n = (int)((even + choice.chunk - 1) / choice.chunk), ns = n + (choice.rest > 0);
    first[g] = (int)(pre.size() / NSG_ATTN_WORK_INTS);
    splits[g] = ns;
    for (int s = 0; s < ns; ++s)  // (the short shares last)
      for (int t = 0; t < tiles; ++t) {
        const int b = (int)(s < n ? even * s / n : even) * kStep;
        const int e = (int)(s < n ? even * (s + 1) / n : steps) * kStep;
        pre.insert(pre.end(), {q0 + t * T, std::min(T, q1 - q0 - t * T), kAll, pkv[g], b,
                               std::min(len, e), 2, 0});
      }
  }
  const int n_pre = (int)(pre.size() / NSG_ATTN_WORK_INTS);
  if (sz.fixed && n_pre > sz.max_prefix_work) {
    set_error("plan needs %d prefix items, the fixed list holds %d", n_pre, sz.max_prefix_work);
    return NSG_ERR_WORKSPACE;
  }
  // ---- merge items: one per query tile of the own parts, whose splits are
  //      consecutive items ----
  const int pre_slots = sz.fixed ? sz.max_prefix_work : n_pre;
  const int own0 = one_launch ? pre_slots : 0;  // first own item among the partials
  std::vector<int32_t> merge;
  int g = 0;
  for (int i = 0; i < op.num_work;) {
    int32_t* w = own.data() + (size_t)i * NSG_ATTN_WORK_INTS;
    if (w[1] == 0) break;  // padding
    const int ns = std::max(1, w[6]);
    for (int s = 0; s < ns; ++s) {
      w[(size_t)s * NSG_ATTN_WORK_INTS + 3] += pkv[num_groups];  // after the prefixes' page ids
      w[(size_t)s * NSG_ATTN_WORK_INTS + 6] = std::max(2, ns);
    }
    // (tiles need not come in the requests' order)
    g = (int)(std::upper_bound(groups, groups + num_groups + 1, 0,
                               [&](int, int32_t b) { return qo[b] > w[0]; }) -
              groups) - 1;
    merge.insert(merge.end(), {w[0], w[1], i + own0, ns, first[g], splits[g], qo[groups[g]],
                             tiles_of(g, T)});
    i += ns;
  }
  const int n_merge = (int)(merge.size() / NSG_ATTN_WORK_INTS);
  plan->own = op;
  plan->num_prefix_work = pre_slots;
  plan->num_merge = sz.fixed ? sz.max_merge : n_merge;
  plan->prefix_rows = rows;
  plan->prefix_tile_tokens = T;
  const int64_t q_rows = sz.fixed ? (int64_t)sz.max_batch * sz.max_q_len : qo[batch];
  plan->merge_lanes = q_rows * Hq * (head_dim / 8) <= 65536 ? 4 : 1;
  plan->prefix_kv_groups = rows <= 64 && page_size >= 16 ? (head_dim == 64 ? 4 : 2) : 1;
  plan->one_launch = one_launch;
  plan->own_rows = own_rows;
  const int64_t row_bytes = (int64_t)Hkv * (head_dim + 4) * 4;
  const int64_t own_bytes = (int64_t)op.num_work * own_rows * row_bytes;
  const int64_t pre_bytes = (int64_t)pre_slots * rows * row_bytes;
  // (one launch: the prefix items come first, in the list and among the partials)
  plan->prefix_partials = kHeader + (one_launch ? 0 : own_bytes);
  plan->workspace_bytes = kHeader + own_bytes + pre_bytes;
  const int64_t items = (int64_t)op.num_work + plan->num_prefix_work + plan->num_merge;
  if (sz.fixed && n_merge > sz.max_merge) {
    set_error("plan needs %d merge items, the fixed list holds %d", n_merge, sz.max_merge);
    return NSG_ERR_WORKSPACE;
  }
  if (!work_h || items > work_capacity) {
    set_error("work list needs %lld items, buffer holds %d", (long long)items, work_capacity);
    return NSG_ERR_WORKSPACE;
  }
  auto put = [&](const std::vector<int32_t>& from, int n, int slots) {
    std::copy(from.begin(), from.begin() + (size_t)n * NSG_ATTN_WORK_INTS, work_h);
    std::fill(work_h + (size_t)n * NSG_ATTN_WORK_INTS, work_h + (size_t)slots * NSG_ATTN_WORK_INTS,
              0);
    work_h += (size_t)slots * NSG_ATTN_WORK_INTS;
  };
  if (one_launch) put(pre, n_pre, pre_slots);
  put(own, op.num_work, op.num_work);
  if (!one_launch) put(pre, n_pre, pre_slots);
  put(merge, n_merge, plan->num_merge);
  clear_error();
  return NSG_OK;
}

}  // namespace
}  // namespace nsg

using namespace nsg;

extern "C" int32_t nsg_prefix_attn_plan(
    const int32_t* qo_indptr_h, const int32_t* group_indptr_h, int32_t num_groups,
    const int32_t* prefix_kv_indptr_h, const int32_t* prefix_kv_last_page_len_h,
    const int32_t* kv_indptr_h, const int32_t* kv_last_page_len_h, int32_t batch,
    int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
    int32_t causal, int32_t num_cus, int32_t* work_h, int32_t work_capacity,
    nsg_prefix_attn_plan_t* plan) {
  return guarded([&] {
    return plan_impl(qo_indptr_h, group_indptr_h, num_groups, prefix_kv_indptr_h,
                     prefix_kv_last_page_len_h, kv_indptr_h, kv_last_page_len_h, batch,
                     num_qo_heads, num_kv_heads, head_dim, page_size, causal, num_cus, Sizes{},
                     work_h, work_capacity, plan);
  });
}

extern "C" int32_t nsg_prefix_attn_fixed_capacity(int32_t batch, int32_t max_q_len,
                                                  int32_t max_groups, int32_t num_qo_heads,
                                                  int32_t num_kv_heads, int32_t head_dim,
                                                  int32_t num_cus, int32_t max_kv_len,
                                                  int32_t max_prefix_pages, int32_t page_size,
                                                  int32_t* max_work, int32_t* max_prefix_work,
                                                  int32_t* max_merge) {
  NSG_CHECK_ARG(max_work && max_prefix_work && max_merge, "null argument");
  NSG_CHECK_ARG(max_groups >= 1 && max_prefix_pages >= 0 && page_size >= 1,
                "max_groups %d, max_prefix_pages %d, page_size %d", max_groups, max_prefix_pages,
                page_size);
  NSG_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim %d (64 or 128)", head_dim);
  if (int32_t rc = nsg_attn_fixed_capacity(batch, max_q_len, num_qo_heads, num_kv_heads, num_cus,
                                           max_kv_len, max_work, max_merge))
    return rc;
  if (num_cus <= 0) num_cus = 256;
  const int G = num_qo_heads / num_kv_heads;
  const int64_t rows_all = (int64_t)batch * max_q_len * G;
  // (the lowest tiles such a plan takes)
  const int rows = prefix_rows(rows_all <= kFixedJointRows ? std::min<int64_t>(rows_all, 64)
                                                           : rows_all, head_dim);
  const int T = std::max(1, rows / G);
  // tiles: one more per group for its last, partly filled one; shares: the
  // target, one more per tile for rounding, or what an item's page list forces
  const int64_t tiles = ((int64_t)batch * max_q_len + T - 1) / T + max_groups;
  const int64_t steps = ((int64_t)max_prefix_pages * page_size + kStep - 1) / kStep;
  const int64_t by_pages =
      std::max<int64_t>(1, (int64_t)(kMaxItemPages - 2) * page_size / kStep);
  const int64_t forced = tiles * ((steps + by_pages - 1) / by_pages);
  const int64_t n = std::max<int64_t>(forced, 2 * num_cus / num_kv_heads + tiles);
  NSG_CHECK_ARG(n <= 1 << 24, "too many prefix items (%lld)", (long long)n);
  *max_prefix_work = (int32_t)n;
  *max_merge = *max_work;  // every query tile of the own parts meets its prefix
  clear_error();
  return NSG_OK;
}

extern "C" int32_t nsg_prefix_attn_plan_fixed(
    const int32_t* qo_indptr_h, const int32_t* group_indptr_h, int32_t num_groups,
    const int32_t* prefix_kv_indptr_h, const int32_t* prefix_kv_last_page_len_h,
    const int32_t* kv_indptr_h, const int32_t* kv_last_page_len_h, int32_t batch,
    int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
    int32_t causal, int32_t num_cus, int32_t max_batch, int32_t max_q_len, int32_t max_kv_len,
    int32_t max_work, int32_t max_prefix_work, int32_t max_merge, int32_t* work_h,
    int32_t work_capacity, nsg_prefix_attn_plan_t* plan) {
  NSG_CHECK_ARG(max_prefix_work >= 0, "max_prefix_work %d", max_prefix_work);
  NSG_CHECK_ARG(batch <= max_batch, "batch %d exceeds the fixed plan's %d", batch, max_batch);
  NSG_CHECK_ARG(max_q_len >= 1 && max_work >= 1 && max_merge >= 1,
                "max_q_len %d, max_work %d, max_merge %d", max_q_len, max_work, max_merge);
  NSG_CHECK_ARG(page_size > 0 && max_kv_len <= (kMaxItemPages - 2) * (int64_t)page_size,
                "max_kv_len %d exceeds one work item's page list (%lld tokens)", max_kv_len,
                (kMaxItemPages - 2) * (long long)page_size);
  return guarded([&] {
    return plan_impl(qo_indptr_h, group_indptr_h, num_groups, prefix_kv_indptr_h,
                     prefix_kv_last_page_len_h, kv_indptr_h, kv_last_page_len_h, batch,
                     num_qo_heads, num_kv_heads, head_dim, page_size, causal, num_cus,
                     Sizes{true, max_batch, max_q_len, max_kv_len, max_work, max_prefix_work, max_merge},
                     work_h, work_capacity, plan);
  });
}

extern "C" int32_t nsg_prefix_attn_run(const nsg_prefix_attn_plan_t* plan, const int32_t* work_d,
                                       const void* q, const void* k_cache, const void* v_cache,
                                       const void* kv_scale, void* out,
                                       const int32_t* kv_indices, int32_t page_size,
                                       int32_t num_pages, float sm_scale, int32_t causal,
                                       void* workspace, int64_t workspace_bytes,
                                       nsg_stream_t stream) {
  NSG_CHECK_ARG(plan != nullptr, "null plan");
  if (plan->own.num_work == 0) {
    clear_error();
    return NSG_OK;
  }
  NSG_CHECK_ARG(work_d && q && k_cache && v_cache && out && kv_indices && workspace,
                "null pointer argument");
  NSG_CHECK_ARG(page_size > 0 && (page_size & (page_size - 1)) == 0,
                "page_size %d must be a power of two", page_size);
  NSG_CHECK_ARG(num_pages > 0, "num_pages %d", num_pages);
  NSG_CHECK_ARG(sm_scale > 0.f, "sm_scale %g must be positive", (double)sm_scale);
  NSG_CHECK_ARG(((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)q | (uintptr_t)out) % 16 == 0,
                "q, out and the caches must be 16-byte aligned");
  const nsg_attn_plan_t& own = plan->own;
  NSG_CHECK_ARG((int64_t)page_size * own.num_kv_heads * own.head_dim < 1ll << 31,
                "a page of %d tokens is too large", page_size);
  if (own.head_dim != 64 && own.head_dim != 128) {
    set_error("head_dim %d not supported", own.head_dim);
    return NSG_ERR_UNSUPPORTED;
  }
  NSG_CHECK_ARG((own.kv_groups == 1 && plan->prefix_kv_groups == 1) || page_size >= 16,
                "page_size %d: the plan's %d KV groups need pages of 16+ tokens (plan and run "
                "with the same page size)", page_size, std::max(own.kv_groups,
                                                               plan->prefix_kv_groups));
  if (workspace_bytes < plan->workspace_bytes) {
    set_error("workspace has %lld bytes, plan needs %lld", (long long)workspace_bytes,
              (long long)plan->workspace_bytes);
    return NSG_ERR_WORKSPACE;
  }
  const bool fp8 = kv_scale != nullptr;
  char* ws = static_cast<char*>(workspace);
  AttnParams prm{};
  prm.q = static_cast<const bf16*>(q);
  prm.kc = static_cast<const bf16*>(k_cache);
  prm.vc = static_cast<const bf16*>(v_cache);
  prm.kc8 = static_cast<const uint8_t*>(k_cache);
  prm.vc8 = static_cast<const uint8_t*>(v_cache);
  prm.kv_scale = static_cast<const uint8_t*>(kv_scale);
  prm.out = static_cast<bf16*>(out);
  prm.Hq = own.num_qo_heads;
  prm.Hkv = own.num_kv_heads;
  prm.G = own.num_qo_heads / own.num_kv_heads;
  prm.log2P = __builtin_ctz((unsigned)page_size);
  prm.num_pages = num_pages;
  prm.causal = causal ? 1 : 0;
  prm.scale_log2 = sm_scale * 1.4426950408889634f;
  prm.flags = reinterpret_cast<int*>(ws);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](const nsg_attn_plan_t& pl) {
    if (pl.row_tiles >= 8)
      return fp8 ? launch_tiles_part_fp8(pl.head_dim, pl.row_tiles / 2, pl.num_work, prm, s)
                 : launch_tiles_part(pl.head_dim, pl.row_tiles / 2, pl.num_work, prm, s);
    return (fp8 ? launch_verify_attn_fp8 : launch_verify_attn)(&pl, prm, s);
  };
  prm.work = work_d;
  prm.kv_indices = kv_indices;
  prm.partials = reinterpret_cast<float*>(ws + kHeader);
  nsg_attn_plan_t pl = own;
  pl.num_work = own.num_work + (plan->one_launch ? plan->num_prefix_work : 0);
  pl.row_tiles = plan->own_rows / 16;
  prm.num_work = pl.num_work;
  if (int32_t rc = launch(pl)) return rc;
  if (!plan->one_launch && plan->num_prefix_work > 0) {
    prm.work = work_d + (size_t)own.num_work * NSG_ATTN_WORK_INTS;
    prm.partials = reinterpret_cast<float*>(ws + plan->prefix_partials);
    pl.num_work = prm.num_work = plan->num_prefix_work;
    pl.row_tiles = plan->prefix_rows / 16;
    pl.kv_groups = plan->prefix_kv_groups;
    if (int32_t rc = launch(pl)) return rc;
  }
  MergeParams m{};
  m.merge = work_d + (size_t)(own.num_work + plan->num_prefix_work) * NSG_ATTN_WORK_INTS;
  m.own = reinterpret_cast<const float*>(ws + kHeader);
  m.prefix = reinterpret_cast<const float*>(ws + plan->prefix_partials);
  m.out = prm.out;
  m.own_rows = plan->own_rows;
  m.prefix_rows = plan->prefix_rows;
  m.prefix_tokens = plan->prefix_tile_tokens;
  m.Hq = prm.Hq;
  m.Hkv = prm.Hkv;
  m.G = prm.G;
  const int pieces = kThreads / plan->merge_lanes;  // a workgroup's
  const unsigned slices =
      (unsigned)((own.q_tile_tokens * prm.G * (own.head_dim / 8) + pieces - 1) / pieces);
  const dim3 grid(plan->num_merge, prm.Hkv, slices);
  const dim3 block(kThreads);
  const bool four = plan->merge_lanes == 4;
  if (own.head_dim == 64 && four)
    hipLaunchKernelGGL((prefix_merge_kernel<64, 4>), grid, block, 0, s, m);
  else if (own.head_dim == 64)
    hipLaunchKernelGGL((prefix_merge_kernel<64, 1>), grid, block, 0, s, m);
  else if (four)
    hipLaunchKernelGGL((prefix_merge_kernel<128, 4>), grid, block, 0, s, m);
  else
    hipLaunchKernelGGL((prefix_merge_kernel<128, 1>), grid, block, 0, s, m);
  return launch_status("prefix_merge_kernel");
}
