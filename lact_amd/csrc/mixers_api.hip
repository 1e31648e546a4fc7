// Host side of the token mixers of liblact_hip.so (masked_attention.h, attention_step.h, linear_attention.h): checks the arguments and
// enqueues the kernels on the caller's stream.  No allocation, no synchronisation.
#include "../../include/lact_hip.h"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "host_common.h"
#include "attention_step.h"
#include "linear_attention.h"

using namespace lact;

namespace {

constexpr int COMPUTE_UNITS = 256;
constexpr long long MAX_GRID = (1LL << 31) - 1;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int check_type(int act) { return act == LACT_BF16 || act == LACT_F32 ? 0 : fail("act_dtype must be LACT_BF16 or LACT_F32"); }

// [B, L, heads, D] with heads contiguous inside a token
int check_rows(const void* ptr, int ld, long long bs, int width, int act, const char* what) {
  const int al = act == LACT_BF16 ? 8 : 4;
  if (!ptr) return fail(std::string("null pointer: ") + what);
  if (ld % al || bs % al || ld < width || bs < 0 || !aligned16(ptr)) return fail(std::string(what) + ": rows must be 16-byte aligned and hold all heads");
  if (ld > (1 << 23)) return fail(std::string(what) + ": row stride too large");
  return 0;
}

// ---- attention ----------------------------------------------------------------------------------
int check_attention(const lact_attention_desc_t* d) {
  if (!d) return fail("null descriptor");
  if (check_type(d->act_dtype)) return -1;
  if (d->B <= 0 || d->L <= 0 || d->H <= 0 || d->HK <= 0 || d->window <= 0) return fail("masked attention: B, L, H, HK and window must be positive");
  if (d->D != 64 && d->D != 128) return fail("masked attention: head size must be 64 or 128");
  if (d->H % d->HK) return fail("masked attention: the number of key heads must divide that of query heads");
  if (d->L > (1 << 24) || (long long)d->B * d->H > (1 << 20) || (long long)d->B * d->H * ceil_div(d->L, 128) > MAX_GRID || d->B > 65535)
    return fail("masked attention: sequence or batch too large");
  if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return fail("masked attention: the scale must be positive");
  if (!(d->score_cap >= 0.f) || !std::isfinite(d->score_cap)) return fail("masked attention: the score cap must be positive, or 0 for none");
  if (d->n_documents < 0 || d->n_documents > (1 << 24)) return fail("masked attention: bad number of documents");
  if (!d->n_documents && (d->documents || d->prefixes)) return fail("masked attention: documents or prefixes without their number");
  return 0;
}

template <typename T>
int attention_params(const lact_attention_desc_t* d, const void* q, const void* k, const void* v, void* ranges, MaskedAttnParams<T>* p) {
  memset(p, 0, sizeof(*p));
  if (check_rows(q, d->q_ld, d->q_bs, d->H * d->D, d->act_dtype, "q") || check_rows(k, d->k_ld, d->k_bs, d->HK * d->D, d->act_dtype, "k") ||
      check_rows(v, d->v_ld, d->v_bs, d->HK * d->D, d->act_dtype, "v"))
    return -1;
  if (d->n_documents && !ranges) return fail("null pointer: ranges");
  p->B = d->B; p->L = d->L; p->H = d->H; p->HK = d->HK; p->group = d->H / d->HK;
  p->window = std::min(d->window, d->L);
  p->q = static_cast<const T*>(q); p->k = static_cast<const T*>(k); p->v = static_cast<const T*>(v);
  p->ldq = d->q_ld; p->ldk = d->k_ld; p->ldv = d->v_ld;
  p->bsq = d->q_bs; p->bsk = d->k_bs; p->bsv = d->v_bs;
  if (d->n_documents) {
    p->rows = static_cast<const int2*>(ranges);
    p->cols = p->rows + (size_t)d->B * d->L;
  }
  p->slopes = d->slopes; p->scale = d->scale; p->cap = d->score_cap;
  p->by_kv = make_udiv(d->B * d->HK);
  return 0;
}

// Splits of the queries that a block of keys walks, where the blocks of 128 keys of all heads are fewer than the compute units: two blocks to a unit,
// four tiles of 64 queries at least to a block (in fp32, whose tiles take some eight times as long, one: 300 tokens, 48 / 19 us and 4 for the sums).
int key_splits(const lact_attention_desc_t* d) {
  const long long blocks = (long long)ceil_div(d->L, 128) * d->B * d->HK;
  if (blocks >= COMPUTE_UNITS) return 1;
  const long long tiles = (long long)ceil_div(std::min(d->L, std::min(d->window, d->L) + 127), 64) * (d->H / d->HK);
  return (int)std::max<long long>(1, std::min<long long>({2 * COMPUTE_UNITS / blocks, tiles / (d->act_dtype == LACT_BF16 ? 4 : 1), 16}));
}
size_t attention_workspace(const lact_attention_desc_t* d) {
  const int n = key_splits(d);
  return n > 1 ? (size_t)2 * n * d->B * d->L * d->HK * d->D * sizeof(float) : 0;
}

// Whether two waves share 32 queries, each with half of the keys of every tile, in blocks of 64 queries: where those of 128 leave places of the compute units
// (two blocks to a unit) empty, so that a block's walk is what the time is.  Blocks of 128 / 64 queries, forward and backward, us: 1 x 4096 tokens, 12 heads of
// 128 (384 blocks of 128) 108 + 324 / 95 + 282; 300 tokens in fp32 (12) 36 + 97 / 20 + 75; but 15 heads and a window of 512 (480) 48 + 151 / 57 + 160.
bool half_rows(long long blocks) { return blocks <= COMPUTE_UNITS * 3 / 2; }

// WHICH: 0 forward, 1 dq, 2 dk and dv (in `splits`)
template <int WHICH, typename T, int D, int BENT, int HALVES>
void launch_attention(int splits, const MaskedAttnParams<T>& p, dim3 grid, hipStream_t s) {
  const dim3 block(64 * MASK_WAVES * (WHICH == 2 ? HALVES : 1));
  constexpr int SM = mask_lds_bytes<T, D>(WHICH == 2, MASK_WAVES / (WHICH == 2 ? 1 : HALVES), HALVES);
  const double w = p.window, f = 2.0 * ((double)p.L * w - w * (w - 1) / 2) * D * p.B * p.H;      // without documents
  if constexpr (WHICH == 0) {
    LACT_BIG_LDS((k_masked_attn_fwd<T, D, BENT, HALVES>), SM);
    LACT_LAUNCH_SMEM("k_masked_attn_fwd", "masked_attn", 2 * f, (k_masked_attn_fwd<T, D, BENT, HALVES>), grid, block, SM, s, p);
  } else if constexpr (WHICH == 1) {
    LACT_BIG_LDS((k_masked_attn_dq<T, D, BENT, HALVES>), SM);
    LACT_LAUNCH_SMEM("k_masked_attn_dq", "masked_attn_bwd", 3 * f, (k_masked_attn_dq<T, D, BENT, HALVES>), grid, block, SM, s, p);
  } else {
    LACT_BIG_LDS((k_masked_attn_dkv<T, D, BENT>), SM);
    LACT_LAUNCH_SMEM("k_masked_attn_dkv", "masked_attn_bwd", 4 * f, (k_masked_attn_dkv<T, D, BENT>), grid, block, SM, s, p);
    if (splits > 1) {
      const long long n = (long long)p.B * p.L * p.HK * D;
      LACT_LAUNCH("k_attn_sum", "masked_attn_bwd", 0.0, (k_attn_sum<T>), dim3((unsigned)((n / 4 + 255) / 256), 2), dim3(256), s, n, splits, p.part, p.dk, p.dv);
    }
  }
}
template <int WHICH, typename T, int D, int BENT>
void launch_attention(int splits, MaskedAttnParams<T> p, hipStream_t s) {
  const int heads = p.B * (WHICH == 2 ? p.HK * splits : p.H);
  p.splits = splits;
  p.by_heads = make_udiv(heads);
  const dim3 grid(ceil_div(p.L, 32 * MASK_WAVES) * heads);
  if constexpr (WHICH == 2) launch_attention<WHICH, T, D, BENT, mask_halves<T, D, BENT>()>(splits, p, grid, s);
  else if (half_rows(grid.x)) launch_attention<WHICH, T, D, BENT, 2>(splits, p, dim3(ceil_div(p.L, 16 * MASK_WAVES) * heads), s);
  else launch_attention<WHICH, T, D, BENT, 1>(splits, p, grid, s);
}
template <int WHICH, typename T, int D>
void launch_attention(int splits, const MaskedAttnParams<T>& p, hipStream_t s) {
  if (!(p.cap > 0.f || p.slopes)) return launch_attention<WHICH, T, D, SCORES_PLAIN>(splits, p, s);
  if constexpr (sizeof(T) == 2)
    if (p.cap > CAP_QUICK) return launch_attention<WHICH, T, D, SCORES_FAR_CAP>(splits, p, s);
  launch_attention<WHICH, T, D, SCORES_BENT>(splits, p, s);
}
template <int WHICH, typename T>
void launch_attention(int splits, int D, const MaskedAttnParams<T>& p, hipStream_t s) {
  if (D == 128) launch_attention<WHICH, T, 128>(splits, p, s);
  else launch_attention<WHICH, T, 64>(splits, p, s);
}

template <typename T>
int attention_forward(const lact_attention_desc_t* d, const void* q, const void* k, const void* v, void* out, float* lse, void* ranges, hipStream_t s) {
  MaskedAttnParams<T> p;
  if (d->n_documents > 1 && !d->documents) return fail("null pointer: documents");
  if (attention_params(d, q, k, v, ranges, &p) || check_ptrs({out, lse}, "masked attention outputs")) return -1;
  p.out = static_cast<T*>(out); p.lse = lse;
  if (d->n_documents)
    LACT_LAUNCH("k_attn_ranges", "masked_attn", 0.0, k_attn_ranges, dim3(ceil_div(d->L, 256), d->B), dim3(256), s, d->L, d->n_documents, p.window, d->documents,
                d->prefixes, const_cast<int2*>(p.rows), const_cast<int2*>(p.cols));
  launch_attention<0>(1, d->D, p, s);
  LACT_CHECK_LAUNCH();
  return 0;
}
template <typename T>
int attention_backward(const lact_attention_desc_t* d, const void* q, const void* k, const void* v, const void* out, const float* lse, const void* ranges,
                       const void* dout, float* delta, void* dq, void* dk, void* dv, void* workspace, hipStream_t s) {
  MaskedAttnParams<T> p;
  if (attention_workspace(d) && !workspace) return fail("null pointer: masked attention workspace");
  if (attention_params(d, q, k, v, const_cast<void*>(ranges), &p) || check_rows(dout, d->do_ld, d->do_bs, d->H * d->D, d->act_dtype, "dout") ||
      check_ptrs({out, lse, delta, dq, dk, dv}, "masked attention backward tensors"))
    return -1;
  p.o = static_cast<const T*>(out); p.lse = const_cast<float*>(lse); p.delta = delta;
  p.dout = static_cast<const T*>(dout); p.lddo = d->do_ld; p.bsdo = d->do_bs;
  p.dq = static_cast<T*>(dq); p.dk = static_cast<T*>(dk); p.dv = static_cast<T*>(dv); p.part = static_cast<float*>(workspace);
  launch_attention<1>(1, d->D, p, s);
  launch_attention<2>(key_splits(d), d->D, p, s);
  LACT_CHECK_LAUNCH();
  return 0;
}

// ---- one token of it ----------------------------------------------------------------------------
int check_step(const lact_attention_step_desc_t* d) {
  if (!d) return fail("null descriptor");
  if (check_type(d->act_dtype)) return -1;
  if (d->B <= 0 || d->N <= 0 || d->H <= 0 || d->HK <= 0 || d->window <= 0) return fail("attention step: B, N, H, HK and window must be positive");
  if (d->D != 64 && d->D != 128) return fail("attention step: head size must be 64 or 128");
  if (d->H % d->HK) return fail("attention step: the number of key heads must divide that of query heads");
  if ((long long)d->B * d->H > (1 << 20) || d->N > (1 << 24)) return fail("attention step: cache or batch too large");
  if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return fail("attention step: the scale must be positive");
  if (!(d->score_cap >= 0.f) || !std::isfinite(d->score_cap)) return fail("attention step: the score cap must be positive, or 0 for none");
  const int al = d->act_dtype == LACT_BF16 ? 8 : 4;
  if (d->q_bs % al || d->k_ld % al || d->k_bs % al || d->k_hs % al || d->v_ld % al || d->v_bs % al || d->v_hs % al)
    return fail("attention step: rows must be 16-byte aligned");
  if (d->k_ld < 0 || d->v_ld < 0 || d->k_bs < 0 || d->v_bs < 0 || d->k_hs < 0 || d->v_hs < 0 || d->q_bs < 0 || d->k_ld > (1 << 23) || d->v_ld > (1 << 23))
    return fail("attention step: strides must be positive, those between tokens at most 2^23");
  return 0;
}
template <typename T, int D>
int step_blocks(const lact_attention_step_desc_t* d) {
  const long long tiles = ceil_div(d->H / d->HK, 32), steps = ceil_div(std::min(d->N, d->window), AttnStepShape<T, D>::KEYS);
  return (int)std::min<long long>(COMPUTE_UNITS, d->B * d->HK * tiles * steps);
}
template <typename T, int D>
size_t step_workspace(const lact_attention_step_desc_t* d) {
  return (size_t)2 * step_blocks<T, D>(d) * std::min(d->H / d->HK, 32) * (D + 2) * sizeof(float);
}
template <typename T, int D>
int step_run(const lact_attention_step_desc_t* d, const void* q, const void* k, const void* v, const int32_t* lengths, void* out, void* workspace, hipStream_t s) {
  AttnStepParams<T> p;
  memset(&p, 0, sizeof(p));
  p.B = d->B; p.N = d->N; p.H = d->H; p.HK = d->HK; p.group = d->H / d->HK; p.tiles = ceil_div(p.group, 32);
  p.window = std::min(d->window, d->N);
  p.blocks = step_blocks<T, D>(d);
  p.q = static_cast<const T*>(q); p.bsq = d->q_bs;
  p.k = static_cast<const T*>(k); p.ldk = d->k_ld; p.bsk = d->k_bs; p.hsk = d->k_hs;
  p.v = static_cast<const T*>(v); p.ldv = d->v_ld; p.bsv = d->v_bs; p.hsv = d->v_hs;
  p.lengths = lengths; p.slopes = d->slopes; p.scale = d->scale; p.cap = d->score_cap;
  p.out = static_cast<T*>(out); p.part = static_cast<float*>(workspace);
  auto launch = [&](auto kind) {
    constexpr int SM = AttnStepShape<T, D>::LDS, BENT = decltype(kind)::value;
    LACT_BIG_LDS((k_attn_step<T, D, BENT>), SM);
    LACT_LAUNCH_SMEM("k_attn_step", "attn_step", 0.0, (k_attn_step<T, D, BENT>), dim3(p.blocks), dim3(64 * AttnStepShape<T, D>::NW), SM, s, p);
  };
  if (sizeof(T) == 2 && p.cap > CAP_QUICK) launch(std::integral_constant<int, sizeof(T) == 2 ? SCORES_FAR_CAP : SCORES_BENT>());
  else launch(std::integral_constant<int, SCORES_BENT>());
  LACT_LAUNCH("k_attn_step_join", "attn_step", 0.0, (k_attn_step_join<T, D>), dim3(p.B * p.H), dim3(512), s, p);
  LACT_CHECK_LAUNCH();
  return 0;
}

// ---- linear attention ---------------------------------------------------------------------------
int check_linear(const lact_linear_desc_t* d) {
  if (!d) return fail("null descriptor");
  if (check_type(d->act_dtype)) return -1;
  if (d->b <= 0 || d->l <= 0 || d->h <= 0) return fail("linear attention: b, l and h must be positive");
  if ((d->dk != 64 && d->dk != 128) || (d->dv != 64 && d->dv != 128)) return fail("linear attention: key and value sizes must be 64 or 128");
  if ((long long)d->b * d->h > (1 << 20) || d->l > (1 << 30)) return fail("linear attention: sequence or batch too large");
  if (!std::isfinite(d->scale)) return fail("linear attention: the scale must be finite");
  return 0;
}

struct LinCut {
  int segments, chunks;      // chunks of a segment
  int stretches() const { return ceil_div(chunks, LIN_STRETCH); }
};
// One block walks a segment of a head; enough segments that the walks of all heads give every compute unit two blocks.  Sequences of a few chunks
// are walked as a whole: two launches less.
LinCut lin_cut(const lact_linear_desc_t* d) {
  const int chunks = ceil_div(d->l, LIN_CHUNK), heads = d->b * d->h;
  if (chunks <= (d->act_dtype == LACT_BF16 ? 4 : 2)) return LinCut{1, chunks};      // (fp32 products take some seven times as long)
  const int want = std::max(1, std::min(chunks, 2 * COMPUTE_UNITS / heads)), per = ceil_div(chunks, want);
  return LinCut{ceil_div(chunks, per), per};
}
struct LinBuffers {
  size_t weights, states, sums, end;     // of `states`: what tokens weigh, where segments start, sums of their decays
  size_t ends, rsums, up, down, part, between, dbetween, scratch;
};
LinBuffers lin_buffers(const lact_linear_desc_t* d) {
  const LinCut cut = lin_cut(d);
  const size_t heads = (size_t)d->b * d->h, elems = (size_t)d->dk * d->dv, tokens = (size_t)d->l * heads;
  auto round = [](size_t n) { return (n + 255) & ~size_t(255); };
  LinBuffers o;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t a = at; at += round(n); return a; };
  const size_t several = cut.segments > 1;
  o.weights = take(heads * ceil_div(d->l, LIN_CHUNK) * LIN_CHUNK * sizeof(float4));
  o.states = take(several * cut.segments * heads * elems * 4);
  o.sums = take(several * cut.segments * heads * 4);
  o.end = at;
  at = 0;
  o.ends = take(several * cut.segments * heads * elems * 4);
  o.rsums = take(several * cut.segments * heads * 4);
  o.up = take(tokens * 8);
  o.down = take(tokens * 4);
  o.part = take(d->decay_per_token ? 0 : cut.segments * cut.stretches() * heads * 8);
  const size_t between = (size_t)cut.segments * (cut.stretches() - 1) * heads * elems * 4;
  o.between = take(between);
  o.dbetween = take(between);
  o.scratch = at;
  return o;
}

template <typename T>
LinParams<T> lin_params(const lact_linear_desc_t* d, const char* states) {
  LinParams<T> p;
  memset(&p, 0, sizeof(p));
  const LinCut cut = lin_cut(d);
  p.B = d->b; p.L = d->l; p.H = d->h; p.segments = cut.segments; p.seg_chunks = cut.chunks; p.stretches = cut.stretches();
  p.weights = reinterpret_cast<const float*>(states + lin_buffers(d).weights);
  p.by_heads = make_udiv(d->h);
  return p;
}

template <typename T, int DX, int DZ, bool REV>
void lin_segments(const LinParams<T>& p, const float* initial, float* states, float* sums, hipStream_t s) {
  constexpr int SM = 2 * (MaskTile<T, DX>::BYTES + MaskTile<T, DZ>::BYTES + 1024);
  LACT_BIG_LDS((k_lin_segments<T, DX, DZ, REV>), SM);
  const int heads = p.B * p.H;
  LACT_LAUNCH_SMEM("k_lin_segments", "linear_attn", 2.0 * heads * p.L * DX * DZ, (k_lin_segments<T, DX, DZ, REV>), dim3((p.segments - 1) * heads), dim3(256), SM, s, p,
                   states, sums);
  LACT_LAUNCH("k_lin_scan", "linear_attn", 0.0, k_lin_scan, dim3((unsigned)(((long long)heads * DX * DZ / 4 + 255) / 256)), dim3(256), s, p.segments, (long long)heads,
              DX * DZ, (int)REV, initial, sums, states);
}

template <typename T, int DK, int DV>
int lin_forward(const lact_linear_desc_t* d, const void* q, const void* k, const void* v, const float* g, const float* state, void* out, float* last, char* states,
                hipStream_t s) {
  const LinBuffers buf = lin_buffers(d);
  LinParams<T> p = lin_params<T>(d, states);
  p.x = {static_cast<const T*>(q), d->q_ld, d->q_bs};
  p.y = {static_cast<const T*>(k), d->k_ld, d->k_bs};
  p.z = {static_cast<const T*>(v), d->v_ld, d->v_bs};
  p.pair_scale = p.state_scale = d->scale; p.source_scale = 1.f;
  p.out = static_cast<T*>(out); p.last = last;
  const int heads = d->b * d->h;
  LACT_LAUNCH("k_lin_weights", "linear_attn", 0.0, k_lin_weights, dim3((unsigned)(((long long)heads * ceil_div(d->l, LIN_CHUNK) + 3) / 4)), dim3(256), s, d->b, d->l, d->h,
              (LinDecay{g, d->decay_per_token}), const_cast<float*>(p.weights));
  if (p.segments > 1) {
    float* at = reinterpret_cast<float*>(states + buf.states);
    lin_segments<T, DK, DV, false>(p, state, at, reinterpret_cast<float*>(states + buf.sums), s);
    p.states = at;
  } else {
    p.state0 = state;
  }
  constexpr int SM = LinShape<T, DK, DV, false>::LDS;
  LACT_BIG_LDS((k_lin_forward<T, DK, DV>), SM);
  LACT_LAUNCH_SMEM("k_lin_forward", "linear_attn", 4.0 * heads * p.L * DK * DV, (k_lin_forward<T, DK, DV>), dim3(p.segments * heads), dim3(256), SM, s, p);
  LACT_CHECK_LAUNCH();
  return 0;
}

template <typename T, int DK, int DV, bool GATE>
void lin_gradients(const LinBackward<T>& p, hipStream_t s) {
  constexpr int SM = std::max({LinShape<T, DV, DK, GATE>::LDS, LinShape<T, DK, DV, GATE>::LDS, LinShape<T, DV, DK, false>::LDS});
  LACT_BIG_LDS((k_lin_backward<T, DK, DV, GATE>), SM);
  LACT_LAUNCH_SMEM("k_lin_backward", "linear_attn_bwd", 12.0 * p.dq.B * p.dq.H * p.dq.L * DK * DV, (k_lin_backward<T, DK, DV, GATE>), dim3(ceil_div(p.items, 8) * 24),
                   dim3(256), SM, s, p);
}

template <typename T, int DK, int DV>
int lin_backward(const lact_linear_desc_t* d, const void* q, const void* k, const void* v, const float* g, const float* state, const float* last, const char* states,
                 const void* dout, const float* dlast, void* dq, void* dk, void* dv, float* dg, float* dstate, char* scratch, hipStream_t s) {
  const LinBuffers buf = lin_buffers(d);
  const LinRows<T> rq{static_cast<const T*>(q), d->q_ld, d->q_bs}, rk{static_cast<const T*>(k), d->k_ld, d->k_bs}, rv{static_cast<const T*>(v), d->v_ld, d->v_bs},
      ro{static_cast<const T*>(dout), d->do_ld, d->do_bs};
  const LinParams<T> base = lin_params<T>(d, states);
  float* up = reinterpret_cast<float*>(scratch + buf.up);
  float* down = reinterpret_cast<float*>(scratch + buf.down);
  float* ends = reinterpret_cast<float*>(scratch + buf.ends);
  const float* starts = reinterpret_cast<const float*>(states + buf.states);
  const bool several = base.segments > 1;
  const int heads = d->b * d->h;
  LinBackward<T> all{base, base, base, base.segments * heads};
  LinParams<T>& a = all.dq;      // forwards with dout, v, k and the transposed state
  a.x = ro; a.y = rv; a.z = rk; a.w = rq;
  a.pair_scale = a.state_scale = d->scale; a.source_scale = 1.f;
  a.out = static_cast<T*>(dq); a.transposed = 1; a.dots = up;
  if (several) a.states = starts;
  else a.state0 = state;
  LinParams<T>& r = all.dv;      // backwards in time
  r.x = rk; r.y = rq; r.z = ro; r.w = rv;
  r.pair_scale = d->scale; r.state_scale = 1.f; r.source_scale = d->scale;
  if (several) {
    lin_segments<T, DK, DV, true>(r, dlast, ends, reinterpret_cast<float*>(scratch + buf.rsums), s);
    r.states = ends;
  } else {
    r.state0 = dlast;
  }
  all.dk = r;
  r.out = static_cast<T*>(dv); r.last = dstate; r.dots = down;
  LinParams<T>& c = all.dk;
  c.x = rv; c.y = ro; c.z = rq;
  c.out = static_cast<T*>(dk); c.transposed = 1;
  float *between = reinterpret_cast<float*>(scratch + buf.between), *dbetween = reinterpret_cast<float*>(scratch + buf.dbetween);
  if (base.stretches > 1) {
    a.between = between;
    r.between = dbetween;
  }
  if (dg) lin_gradients<T, DK, DV, true>(all, s);
  else lin_gradients<T, DK, DV, false>(all, s);
  if (dg) {
    double* part = reinterpret_cast<double*>(scratch + buf.part);
    LACT_LAUNCH("k_lin_decay_grad", "linear_attn_bwd", 0.0, k_lin_decay_grad, dim3(base.segments * base.stretches * heads), dim3(256), s, d->b, d->l, d->h, base.segments,
                base.seg_chunks, base.stretches, DK * DV, base.weights, up, down, starts, ends, last, dlast, between, dbetween, (LinDecay{g, d->decay_per_token}),
                state == nullptr, dg, part);
    if (!d->decay_per_token)
      LACT_LAUNCH("k_lin_decay_sum", "linear_attn_bwd", 0.0, k_lin_decay_sum, dim3(d->h), dim3(64), s, base.segments * base.stretches * d->b, d->h, part, dg);
  }
  LACT_CHECK_LAUNCH();
  return 0;
}

// f(T(), key size, value size as integral constants) for the descriptor's
template <typename F>
int by_sizes(int act, int dk, int dv, F f) {
  using C64 = std::integral_constant<int, 64>;
  using C128 = std::integral_constant<int, 128>;
  auto values = [&](auto t, auto k) { return dv == 64 ? f(t, k, C64()) : f(t, k, C128()); };
  auto keys = [&](auto t) { return dk == 64 ? values(t, C64()) : values(t, C128()); };
  return act == LACT_BF16 ? keys(uint16_t()) : keys(float());
}
int check_linear_rows(const lact_linear_desc_t* d, const void* q, const void* k, const void* v) {
  return check_rows(q, d->q_ld, d->q_bs, d->h * d->dk, d->act_dtype, "q") || check_rows(k, d->k_ld, d->k_bs, d->h * d->dk, d->act_dtype, "k") ||
         check_rows(v, d->v_ld, d->v_bs, d->h * d->dv, d->act_dtype, "v");
}
int check_states(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (!aligned16(p)) return fail("linear attention: states must be 16-byte aligned");
  return 0;
}

}  // namespace

extern "C" {

size_t lact_attention_ranges_bytes(const lact_attention_desc_t* d) {
  return d && d->n_documents > 0 && d->B > 0 && d->L > 0 ? (size_t)d->B * d->L * 2 * sizeof(int2) : 0;
}

size_t lact_masked_attention_workspace_bytes(const lact_attention_desc_t* d) { return check_attention(d) ? 0 : attention_workspace(d); }

int lact_masked_attention_forward(const lact_attention_desc_t* d, const void* q, const void* k, const void* v, void* out, float* lse, void* ranges, void* stream) {
  if (check_attention(d)) return -1;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return d->act_dtype == LACT_BF16 ? attention_forward<uint16_t>(d, q, k, v, out, lse, ranges, s) : attention_forward<float>(d, q, k, v, out, lse, ranges, s);
}

int lact_masked_attention_backward(const lact_attention_desc_t* d, const void* q, const void* k, const void* v, const void* out, const float* lse, const void* ranges,
                                   const void* dout, float* delta, void* dq, void* dk, void* dv, void* workspace, void* stream) {
  if (check_attention(d)) return -1;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return d->act_dtype == LACT_BF16 ? attention_backward<uint16_t>(d, q, k, v, out, lse, ranges, dout, delta, dq, dk, dv, workspace, s)
                                   : attention_backward<float>(d, q, k, v, out, lse, ranges, dout, delta, dq, dk, dv, workspace, s);
}

size_t lact_attention_step_workspace_bytes(const lact_attention_step_desc_t* d) {
  if (check_step(d)) return 0;
  if (d->act_dtype == LACT_BF16) return d->D == 128 ? step_workspace<uint16_t, 128>(d) : step_workspace<uint16_t, 64>(d);
  return d->D == 128 ? step_workspace<float, 128>(d) : step_workspace<float, 64>(d);
}

int lact_attention_step(const lact_attention_step_desc_t* d, const void* q, const void* k, const void* v, const int32_t* lengths, void* out, void* workspace,
                        void* stream) {
  if (check_step(d) || check_ptrs({q, k, v, lengths, out, workspace}, "attention step tensors")) return -1;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return fail("attention step: rows must be 16-byte aligned");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (d->act_dtype == LACT_BF16)
    return d->D == 128 ? step_run<uint16_t, 128>(d, q, k, v, lengths, out, workspace, s) : step_run<uint16_t, 64>(d, q, k, v, lengths, out, workspace, s);
  return d->D == 128 ? step_run<float, 128>(d, q, k, v, lengths, out, workspace, s) : step_run<float, 64>(d, q, k, v, lengths, out, workspace, s);
}

int lact_linear_attention_sizes(const lact_linear_desc_t* d, size_t* states_bytes, size_t* scratch_bytes) {
  if (check_linear(d)) return -1;
  const LinBuffers buf = lin_buffers(d);
  if (states_bytes) *states_bytes = buf.end;
  if (scratch_bytes) *scratch_bytes = buf.scratch;
  return 0;
}

int lact_linear_attention_forward(const lact_linear_desc_t* d, const void* q, const void* k, const void* v, const float* g, const float* state, void* out, float* last,
                                  void* states, void* stream) {
  if (check_linear(d) || check_linear_rows(d, q, k, v) || check_ptrs({g, out}, "linear attention tensors") || check_states({state, last, states})) return -1;
  if (!states) return fail("null pointer: linear attention states");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return by_sizes(d->act_dtype, d->dk, d->dv, [&](auto t, auto dk, auto dv) {
    return lin_forward<decltype(t), decltype(dk)::value, decltype(dv)::value>(d, q, k, v, g, state, out, last, static_cast<char*>(states), s);
  });
}

int lact_linear_attention_backward(const lact_linear_desc_t* d, const void* q, const void* k, const void* v, const float* g, const float* state, const float* last,
                                   const void* states, const void* dout, const float* dlast, void* dq, void* dk_, void* dv_, float* dg, float* dstate, void* scratch,
                                   void* stream) {
  if (check_linear(d) || check_linear_rows(d, q, k, v) || check_rows(dout, d->do_ld, d->do_bs, d->h * d->dv, d->act_dtype, "dout") ||
      check_ptrs({g, dq, dk_, dv_, scratch}, "linear attention backward tensors") || check_states({state, last, states, dlast, dstate, scratch}))
    return -1;
  if (!states) return fail("null pointer: linear attention states");
  if (dg && dlast && !last) return fail("null pointer: the last state, for the gradient of the decays");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return by_sizes(d->act_dtype, d->dk, d->dv, [&](auto t, auto dk, auto dv) {
    return lin_backward<decltype(t), decltype(dk)::value, decltype(dv)::value>(d, q, k, v, g, state, last, static_cast<const char*>(states), dout, dlast, dq, dk_, dv_, dg,
                                                                               dstate, static_cast<char*>(scratch), s);
  });
}

int lact_linear_attention_step(int32_t act_dtype, int32_t b, int32_t h, int32_t dk, int32_t dv, int32_t decay_per_token, float scale, const void* q, int64_t q_bs,
                               const void* k, int64_t k_bs, const void* v, int64_t v_bs, const float* g, const float* state, float* state_out, void* out,
                               void* stream) {
  if (check_type(act_dtype)) return -1;
  if (b <= 0 || h <= 0 || (long long)b * h > (1 << 20)) return fail("linear attention step: b and h must be positive, with at most 2^20 states");
  if ((dk != 64 && dk != 128) || (dv != 64 && dv != 128)) return fail("linear attention step: key and value sizes must be 64 or 128");
  if (!std::isfinite(scale)) return fail("linear attention step: the scale must be finite");
  if (check_ptrs({q, k, v, g, state, state_out, out}, "linear attention step tensors") || check_states({state, state_out})) return -1;
  const int al = act_dtype == LACT_BF16 ? 8 : 4;
  if (v_bs % al || v_bs < 0 || q_bs < 0 || k_bs < 0 || !aligned16(v)) return fail("linear attention step: rows of v must be 16-byte aligned");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto run = [&](auto t) {
    using T = decltype(t);
    LinStepParams<T> p;
    memset(&p, 0, sizeof(p));
    p.H = h; p.DK = dk; p.DV = dv; p.per_token = decay_per_token != 0;
    p.q = static_cast<const T*>(q); p.k = static_cast<const T*>(k); p.v = static_cast<const T*>(v);
    p.bsq = q_bs; p.bsk = k_bs; p.bsv = v_bs;
    p.g = g; p.state = state; p.state_out = state_out; p.scale = scale; p.out = static_cast<T*>(out);
    LACT_LAUNCH("k_lin_step", "linear_attn_step", 0.0, (k_lin_step<T>), dim3(b * h * (dv / 32)), dim3(256), s, p);
  };
  if (act_dtype == LACT_BF16) run(uint16_t());
  else run(float());
  LACT_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
