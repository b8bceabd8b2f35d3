// C ABI of the paged cache (declared in include/pe_paged.h): argument checks, host-side sizing and the
// launches. Nothing here reads device memory, synchronises or allocates device memory.
#include "../../include/pe_paged.h"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>
#include <new>

#include "pe_paged_attn.h"
#include "pe_paged_rope.h"

namespace {

constexpr int64_t kCUs = 256;                      // compute units of an MI355X
constexpr int64_t kMaxGroups = 0xffffffff / 256;   // workgroups of 256 along a grid's axis: their threads count in 32 bits
constexpr int32_t kMaxKeys = PE_PAGED_MAX_KEYS;  // key positions and what is added to them stay in 32 bits

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool row_stride(int64_t s) { return s >= 0 && (s & 7) == 0; }
int launched() { return hipGetLastError() == hipSuccess ? PE_ATTN_OK : PE_ATTN_ELAUNCH; }

// Multiplier and shift of n / d for 0 <= n < 2^31, d >= 2: with 2^(L-1) < d <= 2^L, mul = ceil(2^(31+L) / d)
// is below 2^32 and exceeds 2^(31+L) / d by less than one, so the product's error stays below 2^31 / 2^(31+L)
// <= 1 / d and never reaches the next multiple.
void divider(uint32_t d, uint32_t *mul, uint32_t *shift) {
    uint32_t l = 1;
    while ((1ull << l) < d) ++l;
    *mul = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
    *shift = l - 1;
}

int check_pages(int32_t n_pages, int32_t page_size, int32_t max_pages, int64_t table_stride) {
    if (n_pages < 0 || max_pages < 0 || table_stride < 0 || page_size < PE_PAGED_PAGE_MULTIPLE) return PE_ATTN_EINVAL;
    if (page_size % PE_PAGED_PAGE_MULTIPLE) return PE_ATTN_EUNSUPPORTED;
    return PE_ATTN_OK;
}

// ----------------------------------------------------------------------------- attention

int check_paged(const pe_paged_args *a, bool need_pointers) {
    if (!a || a->struct_size != sizeof(pe_paged_args)) return PE_ATTN_EINVAL;
    if (a->dtype != PE_ATTN_DTYPE_BF16) return PE_ATTN_EUNSUPPORTED;
    if (a->n_seq < 0 || a->total_tokens < 0 || a->max_seqlen < 0 || a->max_seqlen_k < 0) return PE_ATTN_EINVAL;
    if (a->n_heads_q < 1 || a->n_heads_kv < 1 || a->n_heads_q % a->n_heads_kv) return PE_ATTN_EINVAL;
    if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return PE_ATTN_EUNSUPPORTED;
    if (!(a->softmax_scale > 0.0f) || a->softmax_scale > 3e38f) return PE_ATTN_EINVAL;
    if (a->window_left < -1 || a->window_right < -1) return PE_ATTN_EINVAL;
    if (a->causal != 0 && a->causal != 1) return PE_ATTN_EINVAL;
    if (const int status = check_pages(a->n_pages, a->page_size, a->max_pages, a->table_stride)) return status;
    // 32-bit positions and rows; one dimension of the grid holds tiles x kv heads, another query heads.
    if (a->max_seqlen_k > kMaxKeys || a->window_left > kMaxKeys || a->window_right > kMaxKeys ||
        (int64_t)a->max_seqlen * (a->n_heads_q / a->n_heads_kv) > kMaxKeys || a->n_heads_q > 65535)
        return PE_ATTN_EUNSUPPORTED;
    if (!need_pointers || a->n_seq == 0 || a->total_tokens == 0) return PE_ATTN_OK;
    if (!a->q || !a->o || !a->cu_seqlens || !a->seqlens_k) return PE_ATTN_EINVAL;
    if ((a->n_pages > 0 && (!a->k_pages || !a->v_pages)) || (a->max_pages > 0 && !a->page_table)) return PE_ATTN_EINVAL;
    const void *ptrs[4] = {a->q, a->k_pages, a->v_pages, a->o};
    for (const void *p : ptrs)
        if (!aligned16(p)) return PE_ATTN_EINVAL;
    const int64_t strides[10] = {a->q_stride_token, a->q_stride_head, a->k_stride_page,  a->k_stride_token, a->k_stride_head,
                                 a->v_stride_page,  a->v_stride_token, a->v_stride_head, a->o_stride_token, a->o_stride_head};
    for (int64_t s : strides)
        if (!row_stride(s)) return PE_ATTN_EINVAL;
    if (a->k_stride_token < a->head_dim || a->v_stride_token < a->head_dim) return PE_ATTN_EINVAL;
    if (a->total_tokens > 1 && a->o_stride_token < a->head_dim) return PE_ATTN_EINVAL;
    // A page's rows and a tile's output rows are addressed by 32-bit offsets.
    const int64_t limit = (int64_t)1 << 31;
    const int64_t page_span = a->k_stride_token > a->v_stride_token ? a->k_stride_token : a->v_stride_token;
    if (page_span >= limit / 2 / a->page_size) return PE_ATTN_EUNSUPPORTED;
    const int64_t head_span = a->n_heads_q > 1 ? (a->n_heads_q - 1) * (a->o_stride_head < limit ? a->o_stride_head : limit) : 0;
    const int64_t tile_tokens = (pe::kTileRows - 1) / (a->n_heads_q / a->n_heads_kv) + 1;  // from its first token to its last
    if (a->o_stride_token >= limit || head_span >= limit ||
        (tile_tokens * a->o_stride_token + head_span + a->head_dim) * 2 >= limit)
        return PE_ATTN_EUNSUPPORTED;
    return PE_ATTN_OK;
}

// The new tokens of a sequence that the call serves, at most.
int64_t longest_of(const pe_paged_args *a) { return a->max_seqlen < a->total_tokens ? a->max_seqlen : a->total_tokens; }

// How a call runs: paged_row_kernel for sequences of at most `few` rows (times the heads of a kv head) when
// row_blocks > 0, paged_tile_kernel for the others when tiles > 0.
struct PagedShape {
    int32_t few;
    int row_blocks;   // of 16 rows
    bool group;       // paged_group_kernel: a workgroup per sequence and kv head
    int32_t workers;  // waves per kv head
    int64_t tiles;    // items per kv head, at most
    int32_t goal;     // whole chunks its keys are split into, 0: not split
    int32_t chunk, least_chunk;  // steps of a chunk, 0: from goal, and then the least
    int64_t run_slots, tile_slots;  // rows of parts, at most
};

// Waves that run at once on a CU: as many as divide among its SIMDs and have their stages in its 160 KB of LDS
// (head_dim 64: 16 KB each, 128: 48 KB, 256: 64 KB). At head_dim 128, 64 decoding users of U{512..8192} keys, 32:8
// heads: three waves of three stages 213 us, four of two 213 us (of five rows each 255 and 278 us), five of two
// 258 us (a fifth wave per CU waits for a second round), two of four 220 us; 64 users of 12 heads of 64: eight of
// two stages 161 us, six of three 169 us, ten of two 182 us.
int row_waves(int head_dim) { return head_dim == 64 ? 8 : head_dim == 128 ? 3 : 2; }

// Keys that `tokens` neighbouring ones of a sequence reach, at most (from a multiple of 64 on).
int64_t reach_of(const pe_paged_args *a, int64_t tokens) {
    const int wr = a->causal ? 0 : a->window_right;
    const int64_t band = a->window_left >= 0 && wr >= 0 ? (int64_t)a->window_left + wr + tokens + 63 : a->max_seqlen_k;
    return band < a->max_seqlen_k ? band : a->max_seqlen_k;
}
int64_t tile_reach(const pe_paged_args *a) { return reach_of(a, (pe::kTileRows - 1) / (a->n_heads_q / a->n_heads_kv) + 3); }

// The least steps of 64 keys of a chunk: 4, or 8 where several sequences share the chip below head_dim 256
// (eight chunks of U{20..200} rows on U{200..2000} keys at 32:8 heads of 128 47 against 40 us; 300 rows of 8:2 of
// 256 on 900 keys 31 against 48).
constexpr int64_t kChunkSteps = 4;

// Steps of a chunk for a call of one sequence, 0: not split. Its tiles, cut into c chunks each, run in rounds of
// `at_once` workgroups (`most` items altogether), each as long as a chunk and what a workgroup costs beside
// (item, in steps of 64 keys); then the parts are added (four steps' time and six per round). 512 new rows
// on 16,384 keys at 32:8 heads of 128, by rounds: 1 154 us, 1.5 157, 2 163, 3 178; 700 rows 265, 208, 231, 222;
// 300 rows on 300 keys whole 11 us, with a second launch 16.
int32_t chunk_of(const pe_paged_args *a, int64_t tiles, int64_t at_once, int64_t most) {
    const int64_t item = a->head_dim == 64 ? 6 : a->head_dim == 128 ? 3 : 2;
    const int64_t steps = (tile_reach(a) + 63) / 64;
    int64_t best = 0, least = (tiles + at_once - 1) / at_once * (steps + item);
    for (int64_t c = 2; c * tiles <= most && c * kChunkSteps <= steps; ++c) {
        const int64_t chunk = (steps + c - 1) / c, items = c * tiles;
        const int64_t cost = (items + at_once - 1) / at_once * (chunk + item) + 6 * items / at_once + 4;
        if (cost < least) {
            least = cost;
            best = chunk;
        }
    }
    return (int32_t)best;
}

// Whether paged_group_kernel, a workgroup per sequence and kv head, ends sooner than waves with equal runs and a
// second launch, by an estimate in microseconds for sequences of up to max_seqlen_k keys in reach, half of that
// on average. A group's waves take their share of the keys step by step (1 us each at head_dim 128, of four
// waves, 0.7 at 64, 1.5 at 256, of two) after 5 us, in rounds of the workgroups that fit the chip, or at HBM's
// rate; the runs take 11 us more than HBM does. Measured, runs against groups, n sequences of k keys each, 32:8
// heads of 128: 1 x 64 5.9 / 5.2 us, 4 x 256 10.3 / 6.5, 1 x 1,024 10.5 / 12.2, 4 x 2,048 16 / 21, 32 x 256 18 /
// 10, 64 x 512 37 / 31, 64 x 1,536 84 / 76, 256 x 64 27 / 38; 8:2 of 256: 4 x 256 11.2 / 10.2, 32 x 768 19 / 23,
// 128 x 512 34 / 28; 12 of 64: 4 x 1,024 10.1 / 9.3, 128 x 512 51 / 41, 256 x 64 22 / 25. Past 2,048 keys the
// longest sequence decides, and the runs are the even ones. Under a window its reach counts (86 on 2,500 keys, one
// token: 11.3 / 7.3, 8:2 of 256 12.6 / 10.5, 12 of 64 9.8 / 5.7).
bool pays_group(const pe_paged_args *a) {
    const double keys = (double)reach_of(a, longest_of(a)), units = (double)a->n_seq * a->n_heads_kv;
    if (keys > 2048) return false;
    const int d = a->head_dim;
    const double step = d == 64 ? 0.7 : d == 128 ? 1.0 : 1.5, waves = d == 256 ? 2 : 4, at_once = (d == 64 ? 2 : 1) * kCUs;
    const double rounds = (double)(int64_t)((units + at_once - 1) / at_once), steps = (double)(int64_t)((keys + 32 * waves - 1) / (32 * waves));
    const double megabytes = 0.55 * units * keys * d * 4e-6;
    const double by_steps = rounds * (5 + steps * step), by_bytes = 4.5 + megabytes / 5.7;
    return (by_steps > by_bytes ? by_steps : by_bytes) < 11 + megabytes / 5.2;
}

// Whether the tiles of several sequences, `tiles` of the `at_once` that the chip holds, stay whole though
// there are fewer: those of few steps (of 64 keys, for the longest that may come), the fewer the emptier the chip.
// Measured at 32:8 heads of 128, split against whole, n chunks of r rows on k keys: 2 x 64 on 600 23 / 18 us, on
// 1,000 24 / 24, on 2,000 26 / 42; 8 x 64 on 1,000 30 / 26, on 2,000 41 / 44; 8 x 200 on 1,000 67 / 38, on 4,000
// 155 / 124, on U{400..2000} 48 / 43; 2 x 400 on 2,000 61 / 45, on U{400..2000} 30 / 40. 8:2 of 256: 8 x 200 on
// 600 47 / 35, on 1,000 50 / 49, on 2,000 79 / 87; 2 x 64 on 600 25 / 31. 12 of 64: 8 x 200 on 1,000 27 / 21, on
// 2,000 35 / 33; 24 x 40 on U{400..2000} 25 / 36.
bool whole_tiles(const pe_paged_args *a, int64_t steps, int64_t tiles, int64_t at_once) {
    return steps <= (a->head_dim == 256 ? 2 : 10) + (a->head_dim == 64 ? 48 : 64) * tiles / at_once;
}

PagedShape paged_shape(const pe_paged_args *a) {
    PagedShape s;
    std::memset(&s, 0, sizeof(s));
    const int64_t group = a->n_heads_q / a->n_heads_kv, rows = longest_of(a) * group;
    const int64_t n = a->n_seq, hkv = a->n_heads_kv;
    // A sequence's steps of 32 keys (one at least), summed over the sequences in 32 bits.
    const int64_t steps = (a->max_seqlen_k > 32 ? ((int64_t)a->max_seqlen_k + 31) / 32 : 1) * n;
    const bool uneven = n > 1 && 2 * (int64_t)a->total_tokens < n * longest_of(a);  // some sequences are short
    if ((rows <= 32 || (uneven && group <= 16)) && steps < (int64_t)1 << 30) {
        s.few = rows > 16 && rows <= 32 ? 32 : 16;
        s.row_blocks = s.few / 16;
        s.group = rows <= 32 && n * hkv <= kMaxGroups && pays_group(a);
        if (s.group) return s;
        const int waves = rows <= 32 ? row_waves(a->head_dim) : a->head_dim == 64 ? 4 : a->head_dim == 128 ? 2 : 1;
        int64_t workers = waves * kCUs / hkv;
        const int64_t most = (steps + pe::kRunSteps - 1) / pe::kRunSteps;
        if (workers > most) workers = most;
        if (workers > pe::kMaxParts) workers = pe::kMaxParts;
        s.workers = (int32_t)(workers < 1 ? 1 : workers);
        if (s.workers > 1) s.run_slots = s.workers * hkv * 2 * s.few;
        if (rows <= 32) return s;
    }
    // Tiles: at least as many as the rows fill, at most one more for every sequence with any.
    const int64_t fill = (a->total_tokens * group + pe::kTileRows - 1) / pe::kTileRows;
    int64_t with = a->total_tokens * group / (s.few + 1);
    if (with > n) with = n;
    s.tiles = fill + with;
    // Two workgroups per CU run at once (head_dim 64: three). Calls of fewer tiles split their keys.
    const int64_t at_once = (a->head_dim == 64 ? 3 : 2) * kCUs;
    s.least_chunk = n > 1 && a->head_dim < 256 ? 8 : kChunkSteps;
    const int64_t reach_steps = (tile_reach(a) + 63) / 64;
    if (fill * hkv >= at_once || reach_steps <= s.least_chunk) return s;
    const int64_t likely = s.few ? fill : s.tiles, each = n * ((rows + pe::kTileRows - 1) / pe::kTileRows);
    if (n > 1 && whole_tiles(a, reach_steps, (likely < each ? likely : each) * hkv, at_once)) return s;
    s.goal = (int32_t)((a->head_dim == 256 ? 3 : 4) * kCUs);  // (head_dim 256 has the largest parts)
    // The even share makes at most goal whole chunks, and one that is not of every tile; parts are left by
    // tiles of two chunks and more, so by at most 2 * goal.
    int64_t items = s.tiles + (s.goal + hkv - 1) / hkv;
    int64_t longest = s.tiles * ((a->max_seqlen_k + 64 * s.least_chunk - 1) / (64 * s.least_chunk));
    if (n == 1) {
        const int64_t tiles = (rows + pe::kTileRows - 1) / pe::kTileRows;
        s.chunk = chunk_of(a, tiles * hkv, at_once, 2 * s.goal);
        if (s.chunk == 0) {
            s.goal = 0;
            return s;
        }
        items = longest = tiles * ((a->max_seqlen_k + 64 * s.chunk - 1) / (64 * (int64_t)s.chunk));
    }
    s.tiles = items < longest ? items : longest;
    s.tile_slots = (longest * hkv < 2 * s.goal ? longest * hkv : 2 * s.goal) * pe::kTileRows;
    return s;
}

size_t workspace_of(const pe_paged_args *a, const PagedShape &s) { return (size_t)(s.run_slots + s.tile_slots) * (a->head_dim + 2) * 4; }

pe::PagedParams paged_params(const pe_paged_args *a, const PagedShape &s, void *workspace) {
    pe::PagedParams p;
    std::memset(&p, 0, sizeof(p));
    p.q = static_cast<const __bf16 *>(a->q);
    p.k = static_cast<const __bf16 *>(a->k_pages);
    p.v = static_cast<const __bf16 *>(a->v_pages);
    p.o = static_cast<__bf16 *>(a->o);
    p.table = a->page_table;
    p.cu = a->cu_seqlens;
    p.lens = a->seqlens_k;
    p.q_st = a->q_stride_token;
    p.q_sh = a->q_stride_head;
    p.k_sp = a->k_stride_page;
    p.k_st = a->k_stride_token;
    p.k_sh = a->k_stride_head;
    p.v_sp = a->v_stride_page;
    p.v_st = a->v_stride_token;
    p.v_sh = a->v_stride_head;
    p.o_st = a->o_stride_token;
    p.o_sh = a->o_stride_head;
    p.table_st = a->table_stride;
    p.n_seq = a->n_seq;
    p.hq = a->n_heads_q;
    p.hkv = a->n_heads_kv;
    p.group = a->n_heads_q / a->n_heads_kv;
    p.n_pages = a->n_pages;
    p.page = a->page_size;
    p.max_pages = a->max_pages;
    divider((uint32_t)a->page_size, &p.page_mul, &p.page_shift);
    if (p.group > 1) divider((uint32_t)p.group, &p.group_mul, &p.group_shift);
    if (p.hkv > 1) divider((uint32_t)p.hkv, &p.hkv_mul, &p.hkv_shift);
    p.wl = a->window_left;
    p.wr = a->causal ? 0 : a->window_right;
    p.max_seqlen = a->max_seqlen;
    p.max_seqlen_k = a->max_seqlen_k;
    p.few = s.few;
    p.workers = s.workers;
    p.goal = s.goal;
    p.chunk = s.chunk;
    p.least_chunk = s.least_chunk;
    p.tile_slots = s.run_slots;
    p.total_q = a->total_tokens;
    p.c = a->softmax_scale * pe::kLog2e;
    p.part_o = static_cast<float *>(workspace);
    if (workspace) p.part_ml = p.part_o + (s.run_slots + s.tile_slots) * a->head_dim;
    return p;
}

template <int D, bool RUNS, bool TILES>
int launch_merge(const pe_paged_args *a, const pe::PagedParams &p, hipStream_t stream) {
    // A wave per row and some heads once the rows fill the chip, else a workgroup for 64 dims of each.
    const int64_t items = (int64_t)a->total_tokens * a->n_heads_q;
    constexpr int heads = 64 / (D / 4);
    const int64_t waves = (int64_t)a->total_tokens * ((a->n_heads_q + heads - 1) / heads);
    if (items >= 2 * kCUs)
        hipLaunchKernelGGL((pe::paged_merge_kernel<D, RUNS, TILES>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, stream,
                           p);
    else
        hipLaunchKernelGGL((pe::paged_merge_long_kernel<D, RUNS, TILES>),
                           dim3((unsigned)a->total_tokens, (unsigned)a->n_heads_q, D / 64), dim3(256), 0, stream, p);
    return launched();
}

template <int D>
int launch_paged(const pe_paged_args *a, const PagedShape &s, const pe::PagedParams &p, hipStream_t stream) {
    const int64_t blocks = s.tiles * a->n_heads_kv;
    // Every launch fits its grid: tiles and row waves in one, and the merge's waves, one per row and head at most.
    const bool parts = s.run_slots || s.tile_slots;
    if (blocks > kMaxGroups - 8 * kCUs || (parts && (int64_t)a->total_tokens * a->n_heads_q > 4 * kMaxGroups))
        return PE_ATTN_EUNSUPPORTED;
    if (s.row_blocks && s.tiles) {
        const int groups = (int)((s.workers * a->n_heads_kv + pe::kRowWaves<D> - 1) / pe::kRowWaves<D>);
        const dim3 grid((unsigned)(blocks + groups));
        if (s.goal)
            hipLaunchKernelGGL((pe::paged_both_kernel<D, true>), grid, dim3(256), 0, stream, p, groups);
        else
            hipLaunchKernelGGL((pe::paged_both_kernel<D, false>), grid, dim3(256), 0, stream, p, groups);
    } else if (s.group) {
        const dim3 grid((unsigned)(a->n_seq * a->n_heads_kv)), threads(64 * pe::kGroupWaves<D>);
        if (s.row_blocks == 1)
            hipLaunchKernelGGL((pe::paged_group_kernel<D, 1>), grid, threads, 0, stream, p);
        else
            hipLaunchKernelGGL((pe::paged_group_kernel<D, 2>), grid, threads, 0, stream, p);
    } else if (s.row_blocks) {
        constexpr int NS = D == 128 ? 3 : 2;
        const dim3 grid((unsigned)(s.workers * a->n_heads_kv));
        if (s.row_blocks == 1)
            hipLaunchKernelGGL((pe::paged_row_kernel<D, 1, NS>), grid, dim3(64), 0, stream, p);
        else
            hipLaunchKernelGGL((pe::paged_row_kernel<D, 2, NS>), grid, dim3(64), 0, stream, p);
    } else if (s.goal) {
        hipLaunchKernelGGL((pe::paged_tile_kernel<D, true>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    } else {
        hipLaunchKernelGGL((pe::paged_tile_kernel<D, false>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    }
    if (const int status = launched()) return status;
    if (s.run_slots && s.tile_slots) return launch_merge<D, true, true>(a, p, stream);
    if (s.run_slots) return launch_merge<D, true, false>(a, p, stream);
    if (s.tile_slots) return launch_merge<D, false, true>(a, p, stream);
    return PE_ATTN_OK;
}

// ----------------------------------------------------------------------------- rotary positions

// Tokens and heads of a workgroup. Four tokens share a pass over the frequencies from two workgroups per CU
// on (26,000 new tokens of 8:2 heads of 256 appended in 69 us, one by one in 89; rotary of 16,384 tokens of 8
// heads of 128 12.1 against 15.0 us, of 40 heads 61 against 58). A call of fewer takes them one by one, and
// below two workgroups per CU spreads their heads, four at least in each (64 tokens of 40 heads of 128 2.8 us,
// whole tokens 3.2).
void turn_shape(int64_t tokens, int heads, int *per, int *slice) {
    *per = tokens >= 4 * 2 * kCUs ? pe::kTurnTokens : 1;
    const int64_t groups = (tokens + *per - 1) / *per;
    int slices = 1;
    while (groups * slices < 2 * kCUs && 4 * slices < heads) slices *= 2;
    *slice = (heads + slices - 1) / slices;
}

template <typename T, int V>
int launch_rotary(const pe_rotary_args *a, pe::RotaryParams &p, hipStream_t stream) {
    const int64_t groups = (a->n_tokens + p.per - 1) / p.per;
    if (groups > 0x7fffffffLL) return PE_ATTN_EUNSUPPORTED;
    const int64_t heads = (a->n_heads + p.slice - 1) / p.slice;
    for (p.group0 = 0; p.group0 < groups; p.group0 += kMaxGroups) {
        const int64_t left = groups - p.group0;
        const dim3 grid((unsigned)(left < kMaxGroups ? left : kMaxGroups), (unsigned)heads);
        if (a->interleaved)
            hipLaunchKernelGGL((pe::rotary_kernel<T, V, true>), grid, dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL((pe::rotary_kernel<T, V, false>), grid, dim3(256), 0, stream, p);
        if (const int status = launched()) return status;
    }
    return PE_ATTN_OK;
}

// Whether rows split into units of v elements: whole pieces of the turned and of the copied part.
bool in_pieces(int v, int d, int half, bool interleaved) {
    return d % v == 0 && (interleaved ? 2 * half : half) % v == 0 && (d - 2 * half) % v == 0;
}

}  // namespace

extern "C" {

int pe_paged_workspace_size(const pe_paged_args *args, size_t *bytes) {
    if (!bytes) return PE_ATTN_EINVAL;
    if (const int status = check_paged(args, false)) return status;
    *bytes = args->n_seq && args->total_tokens ? workspace_of(args, paged_shape(args)) : 0;
    return PE_ATTN_OK;
}

int pe_paged_attn_fwd(const pe_paged_args *args, void *workspace, size_t workspace_bytes, hipStream_t stream) {
    if (const int status = check_paged(args, true)) return status;
    if (args->n_seq == 0 || args->total_tokens == 0 || args->max_seqlen == 0) return PE_ATTN_OK;
    const PagedShape s = paged_shape(args);
    const size_t need = workspace_of(args, s);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return PE_ATTN_EWORKSPACE;
    const pe::PagedParams p = paged_params(args, s, workspace);
    if (args->head_dim == 64) return launch_paged<64>(args, s, p, stream);
    if (args->head_dim == 128) return launch_paged<128>(args, s, p, stream);
    return launch_paged<256>(args, s, p, stream);
}

int pe_rotary_fwd(const pe_rotary_args *a, hipStream_t stream) {
    if (!a || a->struct_size != sizeof(pe_rotary_args)) return PE_ATTN_EINVAL;
    if (a->dtype < PE_ROTARY_BF16 || a->dtype > PE_ROTARY_FP32) return PE_ATTN_EUNSUPPORTED;
    if (a->n_tokens < 0 || a->n_heads < 0 || a->head_dim < 1 || a->half < 1 || 2 * (int64_t)a->half > a->head_dim)
        return PE_ATTN_EINVAL;
    if ((a->interleaved | a->inverse | a->positions_32) & ~1) return PE_ATTN_EINVAL;
    if (a->half > PE_ROTARY_MAX_PAIRS) return PE_ATTN_EUNSUPPORTED;
    if (a->n_tokens == 0 || a->n_heads == 0) return PE_ATTN_OK;
    if (!a->x || !a->out || !a->positions || !a->inv_freq || a->x_stride_token < 0 || a->x_stride_head < 0)
        return PE_ATTN_EINVAL;
    pe::RotaryParams p;
    std::memset(&p, 0, sizeof(p));
    p.x = a->x;
    p.out = a->out;
    p.positions = a->positions;
    p.inv_freq = a->inv_freq;
    p.x_st = a->x_stride_token;
    p.x_sh = a->x_stride_head;
    p.tokens = a->n_tokens;
    p.heads = a->n_heads;
    p.d = a->head_dim;
    p.half = a->half;
    p.wide = a->positions_32 ? 0 : 1;
    p.scale = a->scale;
    p.sign = a->inverse ? -1.0f : 1.0f;
    turn_shape(a->n_tokens, a->n_heads, &p.per, &p.slice);
    if ((int64_t)pe::kTurnTokens * p.slice * a->head_dim > 0x7fffffffLL || (a->n_heads + p.slice - 1) / p.slice > 65535)
        return PE_ATTN_EUNSUPPORTED;
    // 16-byte pieces where the rows allow them, else single elements.
    const int v = a->dtype == PE_ROTARY_FP32 ? 4 : 8;
    const bool pieces = in_pieces(v, a->head_dim, a->half, a->interleaved) && a->x_stride_token % v == 0 &&
                        a->x_stride_head % v == 0 && aligned16(a->x) && aligned16(a->out);
    if (a->dtype == PE_ROTARY_BF16)
        return pieces ? launch_rotary<__bf16, 8>(a, p, stream) : launch_rotary<__bf16, 1>(a, p, stream);
    if (a->dtype == PE_ROTARY_FP16)
        return pieces ? launch_rotary<_Float16, 8>(a, p, stream) : launch_rotary<_Float16, 1>(a, p, stream);
    return pieces ? launch_rotary<float, 4>(a, p, stream) : launch_rotary<float, 1>(a, p, stream);
}

int pe_paged_append_fwd(const pe_append_args *a, hipStream_t stream) {
    if (!a || a->struct_size != sizeof(pe_append_args)) return PE_ATTN_EINVAL;
    if (a->dtype != PE_ATTN_DTYPE_BF16) return PE_ATTN_EUNSUPPORTED;
    if (a->n_seq < 0 || a->total_tokens < 0 || a->n_heads_q < 0 || a->n_heads_kv < 1 || a->head_dim < 8 || a->half < 0 ||
        2 * (int64_t)a->half > a->head_dim || (a->interleaved & ~1) || (a->q != nullptr) != (a->n_heads_q > 0))
        return PE_ATTN_EINVAL;
    if (const int status = check_pages(a->n_pages, a->page_size, a->max_pages, a->table_stride)) return status;
    if (a->head_dim % 8 || a->half > PE_ROTARY_MAX_PAIRS) return PE_ATTN_EUNSUPPORTED;
    if (a->n_seq == 0 || a->total_tokens == 0) return PE_ATTN_OK;
    if (!a->k || !a->v || !a->cu_seqlens || !a->seqlens_k || (a->q && !a->q_out) || (a->half && !a->inv_freq))
        return PE_ATTN_EINVAL;
    if ((a->n_pages > 0 && (!a->k_pages || !a->v_pages)) || (a->max_pages > 0 && !a->page_table)) return PE_ATTN_EINVAL;
    const void *ptrs[6] = {a->q, a->q_out, a->k, a->v, a->k_pages, a->v_pages};
    for (const void *p : ptrs)
        if (!aligned16(p)) return PE_ATTN_EINVAL;
    const int64_t strides[12] = {a->q_stride_token, a->q_stride_head,   a->k_stride_token,  a->k_stride_head,
                                 a->v_stride_token, a->v_stride_head,   a->kp_stride_page,  a->kp_stride_token,
                                 a->kp_stride_head, a->vp_stride_page,  a->vp_stride_token, a->vp_stride_head};
    for (int64_t s : strides)
        if (!row_stride(s)) return PE_ATTN_EINVAL;
    pe::AppendParams p;
    std::memset(&p, 0, sizeof(p));
    p.q = static_cast<const __bf16 *>(a->q);
    p.k = static_cast<const __bf16 *>(a->k);
    p.v = static_cast<const __bf16 *>(a->v);
    p.q_out = static_cast<__bf16 *>(a->q_out);
    p.k_pages = static_cast<__bf16 *>(a->k_pages);
    p.v_pages = static_cast<__bf16 *>(a->v_pages);
    p.table = a->page_table;
    p.cu = a->cu_seqlens;
    p.lens = a->seqlens_k;
    p.inv_freq = a->inv_freq;
    p.q_st = a->q_stride_token;
    p.q_sh = a->q_stride_head;
    p.k_st = a->k_stride_token;
    p.k_sh = a->k_stride_head;
    p.v_st = a->v_stride_token;
    p.v_sh = a->v_stride_head;
    p.kp_sp = a->kp_stride_page;
    p.kp_st = a->kp_stride_token;
    p.kp_sh = a->kp_stride_head;
    p.vp_sp = a->vp_stride_page;
    p.vp_st = a->vp_stride_token;
    p.vp_sh = a->vp_stride_head;
    p.table_st = a->table_stride;
    p.tokens = a->total_tokens;
    p.n_seq = a->n_seq;
    p.hq = a->n_heads_q;
    p.hkv = a->n_heads_kv;
    p.d = a->head_dim;
    p.half = a->half;
    p.n_pages = a->n_pages;
    p.page = a->page_size;
    p.max_pages = a->max_pages;
    divider((uint32_t)a->page_size, &p.page_mul, &p.page_shift);
    p.scale = a->rope_scale;
    const int64_t heads = (int64_t)a->n_heads_q + 2 * (int64_t)a->n_heads_kv;
    if (heads > 65535 || pe::kTurnTokens * heads * a->head_dim > 0x7fffffffLL) return PE_ATTN_EUNSUPPORTED;
    turn_shape(a->total_tokens, (int)heads, &p.per, &p.slice);
    if ((a->total_tokens + (int64_t)p.per - 1) / p.per > kMaxGroups) return PE_ATTN_EUNSUPPORTED;
    const dim3 grid((unsigned)((a->total_tokens + p.per - 1) / p.per), (unsigned)((heads + p.slice - 1) / p.slice));
    const bool pieces = in_pieces(8, a->head_dim, a->half, a->interleaved);
    if (pieces && a->interleaved)
        hipLaunchKernelGGL((pe::paged_append_kernel<8, true>), grid, dim3(256), 0, stream, p);
    else if (pieces)
        hipLaunchKernelGGL((pe::paged_append_kernel<8, false>), grid, dim3(256), 0, stream, p);
    else if (a->interleaved)
        hipLaunchKernelGGL((pe::paged_append_kernel<1, true>), grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((pe::paged_append_kernel<1, false>), grid, dim3(256), 0, stream, p);
    return launched();
}

int pe_copy_pages(void *const *bases, int32_t n_bases, int64_t page_stride, int64_t page_bytes, int32_t n_pages,
                  const int32_t *src, const int32_t *dst, int32_t n_pairs, hipStream_t stream) {
    if (n_bases < 0 || n_pairs < 0 || n_pages < 0 || page_bytes < 0 || page_stride < 0) return PE_ATTN_EINVAL;
    if ((page_bytes & 15) || (page_stride & 15)) return PE_ATTN_EUNSUPPORTED;
    if (n_bases == 0 || n_pairs == 0 || page_bytes == 0) return PE_ATTN_OK;
    if (!bases || !src || !dst || (n_pages > 1 && page_stride < page_bytes)) return PE_ATTN_EINVAL;
    for (int32_t i = 0; i < n_bases; ++i)
        if (!bases[i] || !aligned16(bases[i])) return PE_ATTN_EINVAL;
    unsigned char *seen = new (std::nothrow) unsigned char[(size_t)n_pages + 1]();  // 1: a source, 2: a target
    if (!seen) return PE_ATTN_EINVAL;
    bool ok = true;
    for (int32_t i = 0; ok && i < n_pairs; ++i) {
        ok = src[i] >= 0 && src[i] < n_pages && dst[i] >= 0 && dst[i] < n_pages;
        if (ok) seen[src[i]] = 1;
    }
    for (int32_t i = 0; ok && i < n_pairs; ++i) {
        ok = seen[dst[i]] == 0;
        seen[dst[i]] = 2;
    }
    delete[] seen;
    if (!ok) return PE_ATTN_EINVAL;
    pe::CopyParams p;
    std::memset(&p, 0, sizeof(p));
    p.stride = page_stride;
    p.pieces = page_bytes / 16;
    const int64_t blocks = (p.pieces + 256 * pe::kCopyPieces - 1) / (256 * pe::kCopyPieces);
    if (blocks > kMaxGroups) return PE_ATTN_EUNSUPPORTED;
    for (int32_t b = 0; b < n_bases; b += pe::kCopyBases) {
        const int32_t nb = n_bases - b < pe::kCopyBases ? n_bases - b : pe::kCopyBases;
        for (int32_t i = 0; i < nb; ++i) p.base[i] = static_cast<char *>(bases[b + i]);
        for (int32_t c = 0; c < n_pairs; c += pe::kCopyPairs) {
            const int32_t nc = n_pairs - c < pe::kCopyPairs ? n_pairs - c : pe::kCopyPairs;
            std::memcpy(p.src, src + c, (size_t)nc * 4);
            std::memcpy(p.dst, dst + c, (size_t)nc * 4);
            hipLaunchKernelGGL(pe::copy_pages_kernel, dim3((unsigned)blocks, (unsigned)nc, (unsigned)nb), dim3(256), 0,
                               stream, p);
            if (const int status = launched()) return status;
        }
    }
    return PE_ATTN_OK;
}

}  // extern "C"
