// Host side of the paged cache and of rotary positions (paged_cache.h, paged_attention.h, rotary.h): checks the arguments and enqueues the kernels on the caller's
// stream.  No allocation, no synchronisation.
#include "../../include/lact_hip.h"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "host_common.h"
#include "paged_attention.h"
#include "rotary.h"

using namespace lact;

namespace {

constexpr int COMPUTE_UNITS = 256;
constexpr long long MAX_ROWS = (1LL << 31) - 1;
constexpr long long MAX_BLOCKS = (1LL << 24) - 1;      // of 256 threads: a launch counts its threads in 32 bits

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int check_type(int act) { return act == LACT_BF16 || act == LACT_F32 ? 0 : fail("act_dtype must be LACT_BF16 or LACT_F32"); }

int check_cache(const lact_paged_cache_t* c, int act, const int32_t* table) {
  if (!c) return fail("null descriptor");
  if (check_type(act)) return -1;
  if (c->dtype != LACT_E4M3 && c->dtype != act) return fail("paged cache: pages must be of act_dtype or LACT_E4M3");
  if (c->pages <= 0 || c->page_size <= 0 || c->HK <= 0 || c->width <= 0) return fail("paged cache: pages, page_size, HK and width must be positive");
  if (c->D != 64 && c->D != 128) return fail("paged cache: head size must be 64 or 128");
  if (c->page_size % 16) return fail("paged cache: the page size must be a multiple of 16");
  if ((long long)c->width * c->page_size > (1 << 24) || (long long)c->HK * c->page_size > (1 << 24)) return fail("paged cache: too many places in a sequence, or rows in a page");
  const long long al = c->dtype == LACT_E4M3 ? 16 : c->dtype == LACT_BF16 ? 8 : 4, rows = (long long)c->HK * c->page_size;
  if (!c->k || !c->v || !table) return fail("null pointer: paged cache");
  if (c->k_page % al || c->v_page % al || !aligned16(c->k) || !aligned16(c->v)) return fail("paged cache: pages must be 16-byte aligned");
  if (c->k_page < rows * c->D || c->v_page < rows * c->D) return fail("paged cache: pages must not overlap");
  if (c->dtype == LACT_E4M3) {
    if (!c->k_exponents || !c->v_exponents) return fail("null pointer: paged cache exponents");
    if (c->ke_page % 16 || c->ve_page % 16 || !aligned16(c->k_exponents) || !aligned16(c->v_exponents)) return fail("paged cache: exponents must be 16-byte aligned");
    if (c->ke_page < rows || c->ve_page < rows) return fail("paged cache: pages of exponents must not overlap");
  }
  return 0;
}
Pages pages_of(const lact_paged_cache_t* c, const int32_t* table) {
  Pages p;
  memset(&p, 0, sizeof(p));
  p.pages = c->pages; p.size = c->page_size; p.wide = c->width; p.HK = c->HK;
  p.by_size = make_udiv(c->page_size);
  p.table = table;
  p.k_page = c->k_page; p.v_page = c->v_page; p.ks_page = c->ke_page; p.vs_page = c->ve_page;
  p.k = c->k; p.v = c->v; p.ks = c->k_exponents; p.vs = c->v_exponents;
  return p;
}

// Memory that is written, or that is read meanwhile: `n` pieces of `len` bytes, `stride` apart.
struct Pieces {
  uintptr_t at;
  long long n, stride, len;
  uintptr_t end() const { return at + (n - 1) * stride + len; }
};
bool disjoint(const Pieces& a, const Pieces& b) {
  if (a.end() <= b.at || b.end() <= a.at) return true;
  if (a.n > 1 && b.n > 1 && a.stride != b.stride) return false;      // (nobody's layout)
  // one between two of the other's, or parts of the same page, however many pages apart they begin: how far behind one of a's the next one of b's begins
  const long long stride = a.n > 1 ? a.stride : b.stride;
  if (stride <= 0) return false;      // (single ones, which share memory)
  long long d = (long long)(b.at - a.at) % stride;      // (signed: either may begin first)
  if (d < 0) d += stride;
  return d >= a.len && stride - d >= b.len;
}
// What a write goes to, nothing of which may lie in another part of it or in what is read.
int check_apart(const lact_paged_cache_t* c, std::initializer_list<Pieces> read) {
  const long long rows = (long long)c->HK * c->page_size, size = c->dtype == LACT_E4M3 ? 1 : c->dtype == LACT_BF16 ? 2 : 4;
  auto pages = [&](const void* p, long long stride, long long len) { return Pieces{reinterpret_cast<uintptr_t>(p), c->pages, stride, len}; };
  const Pieces to[4] = {pages(c->k, c->k_page * size, rows * c->D * size), pages(c->v, c->v_page * size, rows * c->D * size), pages(c->k_exponents, c->ke_page, rows),
                        pages(c->v_exponents, c->ve_page, rows)};
  const int n = c->dtype == LACT_E4M3 ? 4 : 2;
  for (int i = 0; i < n; ++i)
    for (int j = 0; j < i; ++j)
      if (!disjoint(to[i], to[j])) return fail("paged cache write: keys, values and exponents must not overlap");
  for (int i = 0; i < n; ++i)
    for (const Pieces& r : read)
      if (r.at && !disjoint(to[i], r)) return fail("paged cache write: what is read must not lie in the cache");
  return 0;
}

// f(type of the tokens, type of the pages, head size)
template <typename F>
int by_types(int act, int held, int D, F f) {
  auto with = [&](auto t, auto c) { return D == 128 ? f(t, c, std::integral_constant<int, 128>()) : f(t, c, std::integral_constant<int, 64>()); };
  if (act == LACT_BF16) return held == LACT_E4M3 ? with(uint16_t(), uint8_t()) : with(uint16_t(), uint16_t());
  return held == LACT_E4M3 ? with(float(), uint8_t()) : with(float(), float());
}

int check_tokens(const lact_paged_cache_t* c, int B, int L) {
  if (B <= 0 || L <= 0) return fail("paged cache: B and L must be positive");
  // (tiles of at least 8 tokens, and one more at each end)
  if ((long long)B * (L / 8 + 2) > MAX_BLOCKS || c->HK > 65535) return fail("paged cache: too many tokens or heads in one call");
  return 0;
}
template <typename T, int D>
dim3 cache_grid(const lact_paged_cache_t* c, int B, int L, const int32_t* starts, bool along, CacheRows* r) {
  using A = CacheTile<T, D>;
  const int tiles = along ? ceil_div(A::tiles(L), A::TURNS) : A::tiles(L), groups = ceil_div(c->HK, along ? A::ACROSS : A::HEADS);
  *r = CacheRows{B, L, c->HK, make_udiv(tiles), make_udiv(groups), starts};
  return dim3(B * tiles, 2 * groups);
}

// ---- one token's attention --------------------------------------------------------------------------
int check_step(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d, const int32_t* table) {
  if (!d) return fail("null descriptor");
  if (check_cache(c, d->act_dtype, table)) return -1;
  if (d->B <= 0 || d->H <= 0 || d->window <= 0) return fail("paged attention step: B, H and window must be positive");
  if (d->H % c->HK) return fail("paged attention step: the number of key heads must divide that of query heads");
  if ((long long)d->B * d->H > (1 << 20)) return fail("paged attention step: batch too large");
  if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return fail("paged attention step: the scale must be positive");
  if (!(d->score_cap >= 0.f) || !std::isfinite(d->score_cap)) return fail("paged attention step: the score cap must be positive, or 0 for none");
  if (d->q_bs < 0 || d->q_bs % (d->act_dtype == LACT_BF16 ? 8 : 4)) return fail("paged attention step: queries must be 16-byte aligned");
  return 0;
}
int places(const lact_paged_cache_t* c) { return c->width * c->page_size; }
// (a window that begins inside a piece of 16 reaches up to 15 places further back)
template <typename A>
int most_steps(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d) {
  return ceil_div(std::min(places(c), std::min(d->window, places(c)) + 15), A::KEYS);
}
int step_columns(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d) { return d->H / c->HK <= 16 ? 16 : 32; }
int step_items(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d) { return d->B * c->HK * ceil_div(d->H / c->HK, step_columns(c, d)); }
template <typename A>
bool step_whole(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d) { return most_steps<A>(c, d) <= A::WHOLE; }
template <typename A>
int step_blocks(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d) {
  const int items = step_items(c, d);
  return step_whole<A>(c, d) ? items : (int)std::min<long long>(A::BLOCKS * COMPUTE_UNITS, (long long)items * most_steps<A>(c, d));
}
template <typename A, int D>
size_t step_workspace(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d) {
  return step_whole<A>(c, d) ? 0 : (size_t)2 * step_blocks<A>(c, d) * std::min(d->H / c->HK, 32) * (D + 2) * sizeof(float);
}
template <typename T, typename C, int D>
int step_run(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d, const void* q, const int32_t* table, const int32_t* lengths, void* out, void* workspace,
             hipStream_t s) {
  using A = PagedShape<T, C, D>;
  PagedStepParams<T> p;
  memset(&p, 0, sizeof(p));
  p.kv = pages_of(c, table);
  p.B = d->B; p.N = places(c); p.H = d->H; p.HK = c->HK; p.group = d->H / c->HK;
  p.columns = step_columns(c, d); p.tiles = ceil_div(p.group, p.columns);
  p.window = std::min(d->window, p.N);
  p.whole = step_whole<A>(c, d);
  p.blocks = step_blocks<A>(c, d);
  p.q = static_cast<const T*>(q); p.bsq = d->q_bs;
  p.lengths = lengths; p.slopes = d->slopes; p.scale = d->scale; p.cap = d->score_cap;
  p.out = static_cast<T*>(out); p.part = static_cast<float*>(workspace);
  if (!p.whole && !workspace) return fail("null pointer: paged attention step workspace");
  auto launch_for = [&](auto kind, auto tiles) {
    constexpr int BENT = decltype(kind)::value, QT = decltype(tiles)::value;
    LACT_BIG_LDS((k_paged_step<T, C, D, QT, BENT>), A::LDS);
    LACT_LAUNCH_SMEM("k_paged_step", "paged_step", 0.0, (k_paged_step<T, C, D, QT, BENT>), dim3(p.blocks), dim3(64 * A::NW), A::LDS, s, p);
  };
  auto launch = [&](auto kind) { p.columns == 16 ? launch_for(kind, std::integral_constant<int, 1>()) : launch_for(kind, std::integral_constant<int, 2>()); };
  constexpr int FAR = sizeof(T) == 2 ? SCORES_FAR_CAP : SCORES_BENT;
  if (!(p.cap > 0.f || p.slopes)) launch(std::integral_constant<int, SCORES_PLAIN>());
  else if (p.cap > CAP_QUICK) launch(std::integral_constant<int, FAR>());
  else launch(std::integral_constant<int, SCORES_BENT>());
  const int items = step_items(c, d);
  if (!p.whole && p.blocks > 1) {
    const dim3 grid(p.blocks - 1, std::min(p.group, 32));
    // (threads by the parts that an item has, as k_paged_join says.  All 512: 32 sequences of up to 8192, 8 heads of 128, e4m3 65 us for 61; all 128: one of 131072 104 for 102)
    if (p.blocks > 8 * items) LACT_LAUNCH("k_paged_join", "paged_step", 0.0, (k_paged_join<T, D, A::KEYS, 512>), grid, dim3(512), s, p);
    else LACT_LAUNCH("k_paged_join", "paged_step", 0.0, (k_paged_join<T, D, A::KEYS, 128>), grid, dim3(128), s, p);
  }
  LACT_CHECK_LAUNCH();
  return 0;
}

// ---- rotary positions -------------------------------------------------------------------------------
int check_rotary(const lact_rotary_desc_t* d) {
  if (!d) return fail("null descriptor");
  if (check_type(d->act_dtype)) return -1;
  if (d->B <= 0 || d->L <= 0 || d->H <= 0 || d->HK < 0) return fail("rotary: B, L and H must be positive");
  if (d->D <= 0 || d->D % 2 || d->D > 2 * ROTARY_PAIRS) return fail("rotary: head size must be even and at most 256");
  if (d->pairs <= 0 || 2 * d->pairs > d->D) return fail("rotary: pairs must be positive and fit the head");
  if (d->n_axes <= 0 || d->n_axes > 256) return fail("rotary: 1 to 256 axes");
  if ((long long)d->B * d->L > MAX_ROWS || (long long)d->H + d->HK > 65535) return fail("rotary: too many tokens or heads");
  if (d->position_type < 0 || d->position_type > 2) return fail("rotary: positions must be int32, int64 or fp32");
  if (!d->frequencies || !d->axis_of_pair) return fail("null pointer: rotary tables");
  for (int i = 0; i < d->pairs; ++i)
    if (d->axis_of_pair[i] < 0 || d->axis_of_pair[i] >= d->n_axes || !std::isfinite(d->frequencies[i])) return fail("rotary: axes of pairs or frequencies out of range");
  return 0;
}
template <typename T, int V, bool SIDE>
int launch_rotary(RotaryParams p, hipStream_t s) {
  p.units = SIDE ? p.D / V : p.pairs / V + (p.D - 2 * p.pairs) / V;
  p.by_units = make_udiv(p.units);
  const int heads = p.op[0].heads + p.op[1].heads;
  // heads side by side, each of which forms the angles: with few heads fewer, so that angles are formed for six at least (rotary.h)
  p.across = std::min(std::max(1, std::min(4, heads / 6)), 256 / p.units);
  p.by_across = make_udiv(p.across);
  p.tokens = 256 / p.units / p.across;
  const long long blocks = ((long long)p.B * p.L + p.tokens - 1) / p.tokens;
  if (blocks > MAX_BLOCKS) return fail("rotary: too many tokens or heads");
  // as many heads to a block, for which it forms a token's angles once, as leave eight blocks to a compute unit
  p.per = (int)std::max<long long>(p.across, std::min<long long>(heads, blocks * heads / (8 * COMPUTE_UNITS)));
  LACT_LAUNCH("k_rotary", "rotary", 0.0, (k_rotary<T, V, SIDE>), dim3((unsigned)blocks, ceil_div(heads, p.per)), dim3(256), s, p);
  LACT_CHECK_LAUNCH();
  return 0;
}
template <typename T>
int launch_rotary(const RotaryParams& p, bool side, hipStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  bool wide = p.D % E == 0 && (side || p.pairs % E == 0);
  for (const auto& o : p.op) wide = wide && (!o.heads || (aligned16(o.x) && aligned16(o.y) && o.bs % E == 0 && o.ls % E == 0 && o.hs % E == 0));
  if (side) return wide ? launch_rotary<T, E, true>(p, s) : launch_rotary<T, 2, true>(p, s);
  return wide ? launch_rotary<T, E, false>(p, s) : launch_rotary<T, 1, false>(p, s);
}

}  // namespace

extern "C" {

int lact_paged_cache_write(const lact_paged_cache_t* c, int32_t act_dtype, int32_t B, int32_t L, const void* k, int64_t k_ld, int64_t k_bs, const void* v, int64_t v_ld,
                           int64_t v_bs, const int32_t* table, const int32_t* starts, const int32_t* counts, void* stream) {
  if (check_cache(c, act_dtype, table) || check_tokens(c, B, L) || check_ptrs({k, v}, "paged cache write tensors")) return -1;
  const int al = act_dtype == LACT_BF16 ? 8 : 4;
  if (k_ld % al || k_bs % al || v_ld % al || v_bs % al || !aligned16(k) || !aligned16(v) || k_ld < 0 || k_bs < 0 || v_ld < 0 || v_bs < 0)
    return fail("paged cache write: rows must be 16-byte aligned");
  const long long size = act_dtype == LACT_BF16 ? 2 : 4, row = (long long)c->HK * c->D;
  auto whole = [](const void* p, long long bytes) { return Pieces{reinterpret_cast<uintptr_t>(p), 1, 0, bytes}; };
  if (check_apart(c, {whole(k, ((B - 1) * k_bs + (L - 1) * k_ld + row) * size), whole(v, ((B - 1) * v_bs + (L - 1) * v_ld + row) * size),
                      whole(table, (long long)B * c->width * 4), whole(starts, B * 4LL), whole(counts, B * 4LL)}))
    return -1;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return by_types(act_dtype, c->dtype, c->D, [&](auto t, auto h, auto d) {
    using T = decltype(t);
    using C = decltype(h);
    constexpr int D = decltype(d)::value;
    CacheWriteParams<T> p;
    memset(&p, 0, sizeof(p));
    p.to = pages_of(c, table);
    const bool along = CacheTile<T, D>::along(c->HK, L);
    const dim3 grid = cache_grid<T, D>(c, B, L, starts, along, &p.rows);
    p.k = static_cast<const T*>(k); p.v = static_cast<const T*>(v);
    p.ldk = k_ld; p.bsk = k_bs; p.ldv = v_ld; p.bsv = v_bs;
    p.counts = counts;
    if (along) LACT_LAUNCH("k_cache_write", "paged_cache", 0.0, (k_cache_write<T, C, D, true>), grid, dim3(256), s, p);
    else LACT_LAUNCH("k_cache_write", "paged_cache", 0.0, (k_cache_write<T, C, D, false>), grid, dim3(256), s, p);
    LACT_CHECK_LAUNCH();
    return 0;
  });
}

int lact_paged_cache_read(const lact_paged_cache_t* c, int32_t act_dtype, int32_t B, int32_t L, const int32_t* table, const int32_t* starts, const int32_t* lengths,
                          void* k, void* v, void* stream) {
  if (check_cache(c, act_dtype, table) || check_tokens(c, B, L) || check_ptrs({k, v, lengths}, "paged cache read tensors")) return -1;
  if (!aligned16(k) || !aligned16(v)) return fail("paged cache read: rows must be 16-byte aligned");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return by_types(act_dtype, c->dtype, c->D, [&](auto t, auto h, auto d) {
    using T = decltype(t);
    using C = decltype(h);
    constexpr int D = decltype(d)::value;
    CacheReadParams<T> p;
    memset(&p, 0, sizeof(p));
    p.from = pages_of(c, table);
    const bool along = CacheTile<T, D>::along(c->HK, L);
    const dim3 grid = cache_grid<T, D>(c, B, L, starts, along, &p.rows);
    p.k = static_cast<T*>(k); p.v = static_cast<T*>(v);
    p.lengths = lengths;
    if (along) LACT_LAUNCH("k_cache_read", "paged_cache", 0.0, (k_cache_read<T, C, D, true>), grid, dim3(256), s, p);
    else LACT_LAUNCH("k_cache_read", "paged_cache", 0.0, (k_cache_read<T, C, D, false>), grid, dim3(256), s, p);
    LACT_CHECK_LAUNCH();
    return 0;
  });
}

int lact_paged_attention_step_workspace_bytes(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d, const int32_t* table, size_t* bytes) {
  if (check_step(c, d, table) || check_ptrs({bytes}, "paged attention step workspace bytes")) return -1;
  return by_types(d->act_dtype, c->dtype, c->D, [&](auto t, auto h, auto e) {
    constexpr int D = decltype(e)::value;
    *bytes = step_workspace<PagedShape<decltype(t), decltype(h), D>, D>(c, d);
    return 0;
  });
}

int lact_paged_attention_step(const lact_paged_cache_t* c, const lact_paged_step_desc_t* d, const void* q, const int32_t* table, const int32_t* lengths, void* out,
                              void* workspace, void* stream) {
  if (check_step(c, d, table) || check_ptrs({q, lengths, out}, "paged attention step tensors")) return -1;
  if (!aligned16(q)) return fail("paged attention step: queries must be 16-byte aligned");
  return by_types(d->act_dtype, c->dtype, c->D, [&](auto t, auto h, auto e) {
    return step_run<decltype(t), decltype(h), decltype(e)::value>(c, d, q, table, lengths, out, workspace, reinterpret_cast<hipStream_t>(stream));
  });
}

int lact_axial_rotary(const lact_rotary_desc_t* d, const void* q, const void* k, const void* positions, void* q_out, void* k_out, void* stream) {
  if (check_rotary(d) || check_ptrs({q, positions, q_out}, "rotary tensors") || (d->HK && check_ptrs({k, k_out}, "rotary tensors"))) return -1;
  RotaryParams p;
  memset(&p, 0, sizeof(p));
  p.op[0] = RotaryOperand{q, q_out, d->q_bs, d->q_ls, d->q_hs, d->H};
  p.op[1] = RotaryOperand{k, k_out, d->k_bs, d->k_ls, d->k_hs, d->HK};
  p.B = d->B; p.L = d->L; p.D = d->D; p.pairs = d->pairs;
  p.by_l = make_udiv(d->L);
  p.positions = positions; p.position_type = d->position_type; p.pos_bs = d->p_bs; p.pos_ls = d->p_ls;
  p.sign = d->inverse ? -1.f : 1.f;
  for (int i = 0; i < d->pairs; ++i) {
    p.frequency[i] = d->frequencies[i] * 0.63661977236758134308;      // 2 / pi: quarter turns
    p.axis[i] = (uint8_t)d->axis_of_pair[i];
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return d->act_dtype == LACT_BF16 ? launch_rotary<uint16_t>(p, d->interleaved, s) : launch_rotary<float>(p, d->interleaved, s);
}

}  // extern "C"
