// Attention of new tokens over a paged cache (gfx950 MFMA): the arithmetic and operand layouts of the
// packed kernels (pe_attn_device.h), with the key rows found through a page table.
//
// A sequence's query rows are taken with the query heads of one kv head as one axis (row = token *
// group + head), so every row of a tile shares its keys whatever the group is, and a tile of few
// tokens is still a full MFMA operand.
//
// Pages: page_size is a multiple of 16 and a wave stages 16 (head_dim 256: 8) consecutive keys per
// load step, so each step of a wave reads one page. Its id is a scalar load, made a step ahead, and
// the loads go through a buffer resource that starts at the step's first row and ends with the page's
// last row that belongs to the sequence: what lies past it, or in no page at all, reads as zero
// without a branch, and a page may lie anywhere in memory (no 32-bit offset spans two pages).
#pragma once

#include "pe_attn_stage.h"

namespace pe {

struct PagedParams {
    const __bf16 *q, *k, *v;
    __bf16 *o;
    const int32_t *table, *cu, *lens;
    int64_t q_st, q_sh, k_sp, k_st, k_sh, v_sp, v_st, v_sh, o_st, o_sh, table_st;
    int32_t n_seq, hq, hkv, group;
    int32_t n_pages, page, max_pages;
    // n / d = (n * mul >> 32) >> shift for 0 <= n < 2^31 (d > 1; group_mul 0: a group of one)
    uint32_t page_mul, page_shift, group_mul, group_shift, hkv_mul, hkv_shift;
    int32_t wl, wr;                 // window (-1: unbounded); causal folded into wr = 0
    int32_t max_seqlen, max_seqlen_k;
    int32_t few;                    // sequences of at most this many rows are paged_row_kernel's (0: none)
    int32_t workers;                // its waves per kv head
    int32_t goal;                   // whole chunks that paged_tile_kernel's keys should come to, over the kv heads
    int32_t chunk, least_chunk;     // steps of a chunk, 0: from goal, and then the least
    int32_t total_q;
    float c;                        // softmax_scale * log2(e)
    int64_t tile_slots;             // first slot of paged_tile_kernel's parts
    float *part_o, *part_ml;        // split rows' parts [slots][D] and their maxima and sums [slots][2], fp32
};

__device__ __forceinline__ int page_of(const PagedParams &p, int key) {
    return (int)(__umulhi((uint32_t)key, p.page_mul) >> p.page_shift);
}

// Token of a sequence's row (token * group + head of the kv head).
__device__ __forceinline__ int token_of(const PagedParams &p, int row) {
    return p.group_mul ? (int)(__umulhi((uint32_t)row, p.group_mul) >> p.group_shift) : row;
}

__device__ __forceinline__ int over_kv_heads(const PagedParams &p, int n) {
    return p.hkv_mul ? (int)(__umulhi((uint32_t)n, p.hkv_mul) >> p.hkv_shift) : n;
}

// The page table as constant memory: a wave's uniform entry is then a scalar load, which the waits for its
// vector loads do not see (as ordinary memory, which the direct-to-LDS loads might change for all the
// compiler knows, it is a vector load behind every load in flight).
typedef const __attribute__((address_space(4))) int32_t *PageIds;

__device__ __forceinline__ PageIds page_ids_of(const PagedParams &p, int seq) {
    return (PageIds)(uintptr_t)(p.table + (int64_t)seq * p.table_st);
}

// 64 sequences from `base` on, one per lane: the new rows (times the heads of a kv head) of those that the call
// serves, 0 for the others, and their bounds.
struct Lanes {
    int start, rows, lk;
};

// Whether the call serves a sequence: `rows` new tokens from packed row `start` on, lk keys.
__device__ __forceinline__ bool served(const PagedParams &p, int start, int rows, int lk) {
    return rows > 0 && rows <= p.max_seqlen && lk >= 0 && lk <= p.max_seqlen_k && lk <= (int64_t)p.max_pages * p.page &&
           start >= 0 && (int64_t)start + rows <= p.total_q;
}

__device__ __forceinline__ Lanes lanes_from(const PagedParams &p, int base) {
    Lanes q;
    q.start = q.rows = q.lk = 0;
    const int s = base + (int)(threadIdx.x & 63);
    if (s < p.n_seq) {
        q.start = p.cu[s];
        const int L = p.cu[s + 1] - q.start;
        q.lk = p.lens[s];
        if (served(p, q.start, L, q.lk)) q.rows = L * p.group;
    }
    return q;
}

// Keys [klo, khi) that some of the rows [row0, row1) of a sequence reach by position, klo on a multiple of 64.
// `off` is the key position of its first new token.
__device__ __forceinline__ void keys_of(const PagedParams &p, int off, int lk, int row0, int row1, int &klo, int &khi) {
    klo = p.wl >= 0 ? max(0, off + token_of(p, row0) - p.wl) & ~63 : 0;
    khi = lk;
    if (p.wr >= 0) khi = (int)max((int64_t)0, min((int64_t)lk, (int64_t)off + token_of(p, row1 - 1) + 1 + p.wr));
}

// The 16-byte units of a row by key, as swz, but for rows of 512 bytes what it is for 256: the 32x32 operands'
// transposing reads take 8 keys by 4 units, which key & 15 would lay on half of the banks (60 % of the
// LDS cycles at head_dim 256 were conflicts). It depends on the key's low four bits alone.
template <int CPR>
__device__ __forceinline__ int unit_swz(int key) {
    return swz<(CPR == 8 ? 8 : 16)>(key);
}

// A masked key may hold an infinity or NaN, whose product with a zero probability is NaN. In blocks that
// not every row reaches whole, the products therefore run on values cleaned of them (clean8, which tells
// whether there was one), and where one was found each row that reaches it takes it by itself: a
// positive weight leaves an infinity or NaN what it is.
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

__device__ __forceinline__ uint32_t clean8(bf16x8 &x) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 u = __builtin_bit_cast(u32x4, x);
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bad = nonfinite2(u[i]);  // bit 15 of each such half
        u[i] &= ~((bad << 1) - (bad >> 15));
        any |= bad;
    }
    x = __builtin_bit_cast(bf16x8, u);
    return any;
}

__device__ __forceinline__ float only_nonfinite(__bf16 x) {
    const uint32_t u = __builtin_bit_cast(unsigned short, x);
    return (u & 0x7f80u) == 0x7f80u ? (float)x : 0.0f;
}

// Whether a row at key position pos reaches the key (mapped or not).
__device__ __forceinline__ bool reaches(const PagedParams &p, int pos, int key, int khi) {
    return key < khi && (p.wl < 0 || pos - key <= p.wl) && (p.wr < 0 || key - pos <= p.wr);
}

// `rows` rows from a page's `slot` on, of one head: a resource that ends with the last of them (rows <= 0: empty).
// A page spans less than 2 GiB (the host checks), so that only its own place takes 64 bits.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rows(const char *head, int page, uint64_t page_bytes, int slot,
                                                            int row_bytes, int rows, int d) {
    const char *first = head + (uint64_t)(uint32_t)page * page_bytes + (uint32_t)(slot * row_bytes);
    return make_rsrc(first, rows > 0 ? (uint32_t)(rows - 1) * (uint32_t)row_bytes + 2 * d : 0u);
}

// The 16 keys from `key` on (a multiple of 16) lie in a mapped page.
__device__ __forceinline__ bool mapped16(const PagedParams &p, PageIds table, int key) {
    return (uint32_t)table[min(page_of(p, key), p.max_pages - 1)] < (uint32_t)p.n_pages;
}

// ----------------------------------------------------------------------------- many rows

// Items of paged_tile_kernel: a query tile of 128 rows over a chunk of its keys. Calls of few tiles split their
// keys until they fill the chip, many tiles stay whole; sequences of any lengths are cut alike.
constexpr int kTileRows = 128;

struct TileLanes {
    Lanes seq;
    int tiles, reach;  // query tiles, and the most steps of 64 keys that one reaches
};

__device__ __forceinline__ TileLanes tile_lanes(const PagedParams &p, int base) {
    TileLanes t;
    t.seq = lanes_from(p, base);
    t.tiles = t.seq.rows > p.few ? (t.seq.rows + kTileRows - 1) / kTileRows : 0;
    int64_t keys = t.seq.lk;
    if (p.wl >= 0 && p.wr >= 0) keys = min(keys, (int64_t)p.wl + p.wr + token_of(p, kTileRows - 1) + 2 + 64);
    t.reach = (int)((keys + 63) >> 6);
    return t;
}

// The chunks of a sequence's tiles, at most; and its items that leave parts, one for each chunk of a tile.
__device__ __forceinline__ int chunks_of(const TileLanes &t, int steps) { return max(1, (t.reach + steps - 1) / steps); }
__device__ __forceinline__ int split_items(const TileLanes &t, int steps) {
    const int n = chunks_of(t, steps);
    return n > 1 ? t.tiles * n : 0;
}

// Steps of a chunk (SPLIT calls): the host's choice for a call of one sequence, whose work it knows, else the
// even share of all the call's work. Every wave works it out alike, from the bounds alone.
__device__ __forceinline__ int chunk_steps(const PagedParams &p, const TileLanes &first) {
    if (p.chunk > 0) return p.chunk;
    // The lanes' products, below 2^47 each, summed in two parts of 32 bits.
    uint64_t sum = 0;
    for (int base = 0; base < p.n_seq; base += 64) {
        const TileLanes t = base ? tile_lanes(p, base) : first;
        const uint64_t work = (uint64_t)(uint32_t)t.tiles * (uint32_t)t.reach;
        const uint32_t low = __builtin_amdgcn_readlane(wave_scan((int)(work & 0xffffff)), 63);
        const uint32_t high = __builtin_amdgcn_readlane(wave_scan((int)(work >> 24)), 63);
        sum += ((uint64_t)high << 24) + low;
    }
    sum = sum * p.hkv + p.goal - 1;
    const uint64_t steps = sum >> 32 ? sum / p.goal : (uint64_t)((uint32_t)sum / (uint32_t)p.goal);
    return uniform(max(p.least_chunk, (int)min(steps, (uint64_t)1 << 23)));
}

struct TileItem {
    int seq, start, rows, lk, off, row0, chunk;
    int slot;   // the item's place among those that leave parts
    bool valid;
};

template <bool SPLIT>
__device__ __forceinline__ TileItem find_item(const PagedParams &p, int entry, int &steps) {
    TileItem it;
    it.valid = false;
    TileLanes t = tile_lanes(p, 0);
    if constexpr (SPLIT) steps = chunk_steps(p, t);
    for (int base = 0, slots = 0;;) {
        const int n = SPLIT ? t.tiles * chunks_of(t, steps) : t.tiles;
        const int upto = wave_scan(n), all = __builtin_amdgcn_readlane(upto, 63);
        int parts = 0;
        if constexpr (SPLIT) parts = wave_scan(split_items(t, steps));
        if (entry < all) {
            const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > entry));
            const int at = entry - __builtin_amdgcn_readlane(upto - n, who), tiles = __builtin_amdgcn_readlane(t.tiles, who);
            it.seq = base + who;
            it.start = __builtin_amdgcn_readlane(t.seq.start, who);
            it.rows = __builtin_amdgcn_readlane(t.seq.rows, who);
            it.lk = __builtin_amdgcn_readlane(t.seq.lk, who);
            it.off = it.lk - token_of(p, it.rows);
            it.chunk = SPLIT ? at / tiles : 0;  // a chunk's tiles side by side: they read the same keys
            it.row0 = (at - it.chunk * tiles) * kTileRows;
            if constexpr (SPLIT)
                it.slot = slots + __builtin_amdgcn_readlane(parts - split_items(t, steps), who) + at;
            it.valid = true;
            return it;
        }
        entry -= all;
        base += 64;
        if (base >= p.n_seq) return it;
        if constexpr (SPLIT) slots += __builtin_amdgcn_readlane(parts, 63);
        t = tile_lanes(p, base);
    }
}

// First slot of an item's rows, row r of the tile at slot + r.
__device__ __forceinline__ int64_t tile_slot(const PagedParams &p, int item, int kvh) {
    return p.tile_slots + ((int64_t)item * p.hkv + kvh) * kTileRows;
}

// Four waves of 32 rows over keys that all of them read from LDS: chunks of prompts, and any call. Two stages
// of 64 keys (32 at head_dim 256), filled by direct global-to-LDS loads of the next while the waves work on
// one: 64 KB, two workgroups per CU (head_dim 64: three stages in 48 KB, three per CU). A key is read from LDS
// once for 32 rows, its page looked up once for 16. Bound by the products and, at head_dim 64, the exponentials
// beside them: 2,048 new rows on 16,384 keys at 32:8 heads of 128, 515 GFLOP, 494 us, 84 % of a large matrix
// product's rate; at 8:2 of 256 290 us, 72 %, at 12 of 64 132 us, 59 %.
template <int D>
constexpr int kTileStages = D == 64 ? 3 : 2;
template <int D>
constexpr int kTileLds = kTileStages<D> * 2 * (D == 256 ? 32 : 64) * D;  // elements

template <int D, bool SPLIT>
__device__ __forceinline__ void tile_item(const PagedParams &p, int block, __bf16 *ring) {
    constexpr int BM = kTileRows, BN = D == 256 ? 32 : 64, NS = kTileStages<D>;
    constexpr int NB = BN / 32, DC = D / 16, DB = D / 32, CPR = D / 8;
    constexpr int TILE = BN * D, UPW = TILE / 8 / 64 / 4, LPS = 2 * UPW, KPW = BN / 4;
    static_assert(UPW == 2 || UPW == 4, "loads go out four at a time");
    const int entry = over_kv_heads(p, block), kvh = block - entry * p.hkv;
    int steps = 0;
    const TileItem t = find_item<SPLIT>(p, entry, steps);
    if (!t.valid) return;
    int klo, khi;
    keys_of(p, t.off, t.lk, t.row0, min(t.rows, t.row0 + BM), klo, khi);
    const bool split = SPLIT && khi - klo > 64 * steps;
    if constexpr (SPLIT) {
        if (t.chunk > 0 && khi - klo <= 64 * t.chunk * steps) return;  // the tile reaches less than others
        klo += 64 * t.chunk * steps;
        khi = min(khi, klo + 64 * steps);
    }
    const int ntiles = khi > klo ? (khi - klo + BN - 1) / BN : 0;

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 31, kg = lane >> 5;
    const int r0 = t.row0 + 32 * wave, row = r0 + col;
    const bool wave_active = r0 < t.rows;
    const int token = token_of(p, row), head = kvh * p.group + row - token * p.group;
    const int pos = t.off + token;  // the row's key position
    // Key positions of the wave's first row and past its last.
    const int p0 = t.off + token_of(p, r0), p1 = t.off + token_of(p, min(t.rows, r0 + 32) - 1) + 1;

    const PageIds table = page_ids_of(p, t.seq);
    // Whether some page of the workgroup's keys is unmapped (its blocks then look again).
    bool holes = false;
    if (ntiles > 0)
        for (int i = page_of(p, klo) + tid; i <= page_of(p, khi - 1); i += 256)
            holes |= (uint32_t)table[i] >= (uint32_t)p.n_pages;
    const bool any_hole = __syncthreads_or(holes);

    // Wave-load j fills units [(wave * UPW + j) * 64, +64) of a tile: unit u holds key u / CPR, global
    // 16-byte column (u % CPR) ^ swz(key). Offsets are from the wave's first key of the step.
    const int k_row = (int)p.k_st * 2, v_row = (int)p.v_st * 2;
    int koff[UPW], voff[UPW];
#pragma unroll
    for (int j = 0; j < UPW; ++j) {
        const int u = (wave * UPW + j) * 64 + lane;
        const int key = u / CPR, ch = (u % CPR) ^ unit_swz<CPR>(key);
        koff[j] = (key - wave * KPW) * k_row + ch * 16;
        voff[j] = (key - wave * KPW) * v_row + ch * 16;
    }
    const uint32_t ring_base = uniform((int)lds_addr(ring));
    const char *k_head = reinterpret_cast<const char *>(p.k + kvh * p.k_sh);
    const char *v_head = reinterpret_cast<const char *>(p.v + kvh * p.v_sh);
    const uint64_t k_page = 2 * p.k_sp, v_page = 2 * p.v_sp;
    auto page_id = [&](int step) { return table[min(page_of(p, klo + step * BN + wave * KPW), p.max_pages - 1)]; };
    auto issue = [&](int stage, int step, int id) {
        const int key0 = klo + step * BN + wave * KPW, slot = key0 - page_of(p, key0) * p.page;
        const bool mapped = (uint32_t)id < (uint32_t)p.n_pages;
        const int rows = mapped ? min(p.page - slot, t.lk - key0) : 0;
        const __amdgpu_buffer_rsrc_t k_rs = page_rows(k_head, mapped ? id : 0, k_page, slot, k_row, rows, D);
        const __amdgpu_buffer_rsrc_t v_rs = page_rows(v_head, mapped ? id : 0, v_page, slot, v_row, rows, D);
        const uint32_t kb = ring_base + stage * (4 * TILE) + wave * UPW * 1024, vb = kb + 2 * TILE;
        if constexpr (UPW == 2) {
            const uint32_t l4[4] = {kb, kb + 1024, vb, vb + 1024};
            const int o4[4] = {koff[0], koff[1], voff[0], voff[1]};
            dma16x4(l4, o4, k_rs, v_rs);
        } else {
            const uint32_t lk[4] = {kb, kb + 1024, kb + 2048, kb + 3072};
            const uint32_t lv[4] = {vb, vb + 1024, vb + 2048, vb + 3072};
            const int ok[4] = {koff[0], koff[1], koff[UPW - 2], koff[UPW - 1]};
            const int ov[4] = {voff[0], voff[1], voff[UPW - 2], voff[UPW - 1]};
            dma16x4(lk, ok, k_rs, k_rs);
            dma16x4(lv, ov, v_rs, v_rs);
        }
    };

    // The query fragments, straight into registers: lane (col, kg) holds dims 16 c + 8 kg of its row.
    bf16x8 qf[DC];
    {
        const __bf16 *src = p.q + (int64_t)(t.start + token) * p.q_st + (int64_t)head * p.q_sh + 8 * kg;
#pragma unroll
        for (int c = 0; c < DC; ++c) qf[c] = row < t.rows ? ld_g16(src + 16 * c) : bf16x8{};
    }
    // Place of the operands' first chunk in a stage: chunk c of K is 16 c elements on, block db of V^T 32 db,
    // by exclusive or (the swizzle exchanges whole units of a row).
    const int vkey = 4 * kg + ((lane & 15) >> 2), vdim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    int kbase = col * D + (kg ^ unit_swz<CPR>(col)) * 8;
    int vbase0 = vkey * D + ((vdim >> 3) ^ unit_swz<CPR>(vkey)) * 8 + (vdim & 4);
    int vbase1 = (vkey + 8) * D + ((vdim >> 3) ^ unit_swz<CPR>(vkey + 8)) * 8 + (vdim & 4);

    f32x16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[db][j] = 0.0f;
    float m = kNegInf, ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const float c2 = p.c;
    auto values = [&](const __bf16 *keys, int db) {  // V^T of 16 keys, dims 32 db ..
        const bf16x4 lo = tr16(keys + (vbase0 ^ (32 * db))), hi = tr16(keys + (vbase1 ^ (32 * db)));
        return bf16x8(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto row_max = [](const auto &s) {
        float mp[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
        for (const f32x16 &x : s)
#pragma unroll
            for (int j = 0; j < 16; ++j) mp[j & 3] = fmaxf(mp[j & 3], x[j]);
        return fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3]));
    };
    // The maximum is raised only when a row exceeds it by 2^8: the exponentials stay in range and most steps
    // skip the rescale. The two lanes of a row share m.
    auto raise = [&](float mx) {
        if (!wave_any(mx * c2 > m + 8.0f)) return;
        const float mnew = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)) * c2);
        const float alpha = mnew == kNegInf ? 1.0f : exp2_fast(m - mnew);
        m = mnew;
#pragma unroll
        for (int i = 0; i < 4; ++i) ls[i] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[db][j] *= alpha;
    };
    // Steps of keys that all of the wave's rows reach and that lie in pages: [whole_from, whole_to).
    const int whole_from = p.wl >= 0 ? p1 - 1 - p.wl : 0;
    const int whole_to = any_hole ? 0 : p.wr < 0 || khi - 1 - p0 <= p.wr ? khi : p0 + 1 + p.wr;

    int next_id = 0;
    if (ntiles > 0) {
#pragma unroll
        for (int s = 0; s < NS - 1; ++s)
            if (s < ntiles) issue(s, s, page_id(s));
        next_id = page_id(NS - 1);
    }
    // The query rows' wait, here once: at their first use it would stand in the loop, and wait for the
    // loads ahead in every step.
#pragma unroll
    for (int c = 0; c < DC; ++c) asm volatile("" : "+v"(qf[c]));
    auto arrive = [&](int step) {
        // The step's loads are complete once at most the later steps' are in flight.
        const int later = min(ntiles, step + NS - 1) - step - 1;
        if (NS >= 3 && later >= 1) wait_vmcnt<LPS>();
        else wait_vmcnt<0>();
        __syncthreads();
        if (step + NS - 1 < ntiles) {  // into the stage that all waves have left
            issue((step + NS - 1) % NS, step + NS - 1, next_id);
            next_id = page_id(step + NS);
        }
    };
    auto scores = [&](const __bf16 *keys) {  // of 32 keys
        f32x16 acc;
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = 0.0f;
#pragma unroll
        for (int c = 0; c < DC; ++c) acc = mfma32(ld_s16(keys + (kbase ^ (16 * c))), qf[c], acc);
        return acc;
    };
    for (int step = 0; step < ntiles;) {
        // A run of steps that need no mask: nothing but loads, products and the softmax.
        const int first = klo + step * BN;
        const int run_end = wave_active && first >= whole_from ? min(ntiles, step + max(0, whole_to - first) / BN) : step;
        for (; step < run_end; ++step) {
            arrive(step);
            if constexpr (D == 256) asm volatile("" : "+v"(kbase), "+v"(vbase0), "+v"(vbase1));
            const __bf16 *kt = ring + step % NS * (2 * TILE), *vt = kt + TILE;
            f32x16 s[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b] = scores(kt + 32 * b * D);
            raise(row_max(s));
            const float muse = m == kNegInf ? 0.0f : m;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                // At head_dim 64 a block's exponentials all at once, at 128 and 256 each half's before its products
                // (4,096 rows: 8:2 heads of 256 518 -> 490 us, 32:8 of 128 922 -> 919, 12 of 64 241 -> 246).
                constexpr int PART = D == 64 ? 16 : 8;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 8 * h; j < 8 * h + PART && (PART == 8 || h == 0); ++j)
                        s[b][j] = exp2_fast(fmaf(s[b][j], c2, -muse));
                    const bf16x8 pb = to_bf16x8(s[b], 8 * h);
#pragma unroll
                    for (int i = 0; i < 4; ++i) ls[i] = sum2(pb, i, ls[i]);
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db] = mfma32(values(vt + (32 * b + 16 * h) * D, db), pb, o[db]);
                }
            }
        }
        if (step >= ntiles) break;
        arrive(step);
        if (wave_active) {
            const __bf16 *kt = ring + step % NS * (2 * TILE), *vt = kt + TILE;
            const int kt0 = klo + step * BN;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int kb0 = kt0 + 32 * b;
                if (!block_live(kb0, khi, p0, p1, p.wl, p.wr)) continue;
                f32x16 s[1] = {scores(kt + 32 * b * D)};
                uint32_t km = key_mask(kb0, kg, pos, khi, p.wl, p.wr);
                if (any_hole) {
                    const uint32_t low = (1u << (16 - 4 * kg)) - 1u;  // bits of the block's first 16 keys
                    km &= (mapped16(p, table, kb0) ? low : 0u) | (mapped16(p, table, kb0 + 16) ? ~low : 0u);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) s[0][j] = mask_score(s[0][j], km, acc_key(j, 0));
                raise(row_max(s));
                const float muse = m == kNegInf ? 0.0f : m;
#pragma unroll
                for (int j = 0; j < 16; ++j) s[0][j] = exp2_fast(fmaf(s[0][j], c2, -muse));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bf16x8 pb = to_bf16x8(s[0], 8 * h);
#pragma unroll
                    for (int i = 0; i < 4; ++i) ls[i] = sum2(pb, i, ls[i]);
                    const __bf16 *vh = vt + (32 * b + 16 * h) * D;
                    uint32_t bad = 0;
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        bf16x8 va = values(vh, db);
                        bad |= clean8(va);
                        o[db] = mfma32(va, pb, o[db]);
                    }
                    if (!wave_any(bad != 0)) continue;
#pragma unroll 1
                    for (int key = 0; key < 16; ++key) {
                        const bool reach = reaches(p, pos, kb0 + 16 * h + key, khi);
#pragma unroll
                        for (int q = 0; q < 4 * DB; ++q) {  // dims 8 q + 4 kg ..
                            const bf16x4 v4 = *reinterpret_cast<const bf16x4 *>(vh + key * D + (q ^ unit_swz<CPR>(key)) * 8 + 4 * kg);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[q >> 2][4 * (q & 3) + i] += reach ? only_nonfinite(v4[i]) : 0.0f;
                        }
                    }
                }
            }
        }
        ++step;
    }
    if (!wave_active) return;
    const float lsum = (ls[0] + ls[1]) + (ls[2] + ls[3]);
    const float l = lsum + __shfl_xor(lsum, 32);
    if (split) {
        if (row >= t.rows) return;
        const int64_t slot = tile_slot(p, t.slot, kvh) + 32 * wave + col;
        float *dst = p.part_o + slot * D + 4 * kg;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj)
                *reinterpret_cast<f32x4 *>(dst + 32 * db + 8 * jj) =
                    f32x4{o[db][4 * jj], o[db][4 * jj + 1], o[db][4 * jj + 2], o[db][4 * jj + 3]};
        if (kg == 0) {
            p.part_ml[2 * slot] = m;
            p.part_ml[2 * slot + 1] = l;
        }
        return;
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    // The output from the tile's first token on: a resource of its own tokens, whatever the sequence's length.
    const int first = token_of(p, t.row0), last = token_of(p, min(t.rows, t.row0 + BM) - 1);
    const __amdgpu_buffer_rsrc_t o_rs = make_rsrc(
        p.o + (int64_t)(t.start + first) * p.o_st, (uint32_t)(((int64_t)(last - first) * p.o_st + (p.hq - 1) * p.o_sh + D) * 2));
    const int ooff = row < t.rows ? (int)(((token - first) * p.o_st + head * p.o_sh) * 2) : kVoidOffset;
    store_block<DB, false>(o, inv, kg, o_rs, ooff, o_rs, 0);
}

template <int D, bool SPLIT>
__global__ __launch_bounds__(256, 2) void paged_tile_kernel(PagedParams p) {
    __shared__ __attribute__((aligned(16))) __bf16 ring[kTileLds<D>];
    tile_item<D, SPLIT>(p, blockIdx.x, ring);
}

// ----------------------------------------------------------------------------- few rows

// Calls of at most 32 rows per sequence and kv head (single decoded tokens, a few drafted ones) last as long as
// reading their keys once, if all waves read to the end. The keys of one kv head, all sequences in a row, are
// cut into steps of 32 and dealt in equal runs to the head's waves: a run may end one sequence and begin the
// next, so lengths however unequal leave no wave idle, and a wave begins at most one or two sequences. (Equal
// chunks of each sequence, two waves each: 64 sequences of U{512..8192} keys left 10 % to the last to end.)
// Bound by HBM: those 64, at 32:8 heads of 128, 1,160 MB in 212 us and 7 for the parts; three of up to 131,072
// keys at 8:2 of 256 567 MB in 99 us and 7 (5.5 and 5.7 TB/s; reads alone reach 6.1).
constexpr int kRunSteps = 2;  // at least, per wave

struct RowLanes {
    Lanes seq;
    int base, n, upto, all;  // steps, their inclusive sum over the lanes, their total
};

__device__ __forceinline__ RowLanes row_lanes(const PagedParams &p, int base) {
    RowLanes r;
    r.base = base;
    r.seq = lanes_from(p, base);
    r.n = 0;
    if (r.seq.rows > 0 && r.seq.rows <= p.few) {
        int klo, khi;
        keys_of(p, r.seq.lk - token_of(p, r.seq.rows), r.seq.lk, 0, r.seq.rows, klo, khi);
        r.n = max(1, (khi - klo + 31) >> 5);  // a sequence without a key in reach still has rows to write
    }
    r.upto = wave_scan(r.n);
    r.all = __builtin_amdgcn_readlane(r.upto, 63);
    return r;
}

// Steps of a wave's run: all sequences' steps over the head's waves.
__device__ __forceinline__ int row_run(const PagedParams &p, int total) {
    return max(kRunSteps, (total + p.workers - 1) / p.workers);
}

// Place of a part: a wave writes at most two, of the sequence that began before its run and of the one
// that goes on past it.
__device__ __forceinline__ int64_t row_slot(const PagedParams &p, int wave, int which) {
    return ((int64_t)wave * 2 + which) * p.few;
}

// One wave, with LDS stages of its own: no barrier, a step waits for the wave's own loads. Products on
// v_mfma_f32_16x16x32_bf16, lane l: c16 = l % 16, g4 = l / 16:
//  * S^T = K . Q^T per 16 keys: A = key c16 by dims 32 c + 8 g4 .., B = the lane's row; lane l then holds, for
//    row c16, keys 4 g4 + i.
//  * O^T = V^T . P^T per 16 dims: B = the lane's own 8 probabilities, k-slot 8 g4 + i standing for key
//    4 g4 + i and 8 g4 + 4 + i for key 16 + 4 g4 + i; A = V^T for the same keys by two transposing reads;
//    lane l accumulates dims 16 db + 4 g4 + i of row c16.
// The steps of one wave over a sequence's keys: what it adds up for each row.
template <int D, int NR>
struct RowSums {
    f32x4 o[NR][D / 16];
    float m[NR], l[NR];
};

struct RowWork {
    int seq, start, nrows, lk, off, khi;  // the sequence: its rows, keys, key position of its first row
    int key_first, steps;                 // the wave's part of its keys
};

template <int D, int NR, int NS>
__device__ __forceinline__ void row_steps(const PagedParams &p, int kvh, const RowWork &w, __bf16 *ring, RowSums<D, NR> &sums) {
    constexpr int BN = 32, DC = D / 32, DB = D / 16, CPR = D / 8;
    constexpr int TILE = BN * D;  // elements of a step's K (or V)
    constexpr int LH = CPR / 4;   // 1 KB loads of 16 keys
    constexpr int LPS = 4 * LH;   // loads of a step
    static_assert(LH == 2 || LH % 4 == 0, "loads go out four at a time");
    const int lane = threadIdx.x & 63, c16 = lane & 15, g4 = lane >> 4;
    const int start = w.start, nrows = w.nrows, lk = w.lk, off = w.off, khi = w.khi, key_first = w.key_first, steps = w.steps;
    const int k_row = (int)p.k_st * 2, v_row = (int)p.v_st * 2;
    int koff[LH], voff[LH];
#pragma unroll
    for (int j = 0; j < LH; ++j) {
        const int u = j * 64 + lane, key = u / CPR, ch = (u % CPR) ^ unit_swz<CPR>(key);
        koff[j] = key * k_row + ch * 16;
        voff[j] = key * v_row + ch * 16;
    }
    // Place of the operands' first chunk in a stage; the swizzle exchanges whole units and depends on the
    // key's low four bits alone, so chunk c is 32 c elements on by exclusive or, and 16 keys on by sum.
    const int vkey = 4 * g4 + (c16 >> 2), vdim = 4 * (c16 & 3);
    const int kbase = c16 * D + (g4 ^ unit_swz<CPR>(c16)) * 8;
    const int vbase = vkey * D + ((vdim >> 3) ^ unit_swz<CPR>(vkey)) * 8 + (vdim & 4);
    const uint32_t ring_base = uniform((int)lds_addr(ring));
    const char *k_head = reinterpret_cast<const char *>(p.k + kvh * p.k_sh);
    const char *v_head = reinterpret_cast<const char *>(p.v + kvh * p.v_sh);
    const uint64_t k_page = 2 * p.k_sp, v_page = 2 * p.v_sp;
    const float c2 = p.c;

    const PageIds table = page_ids_of(p, w.seq);
    // The ids of the pages that hold a step's two halves.
    auto page_ids = [&](int step) {
        const int key = key_first + 32 * step, top = p.max_pages - 1;
        if (top < 0) return int2{-1, -1};
        return int2{table[min(page_of(p, key), top)], table[min(page_of(p, key + 16), top)]};
    };
    auto mapped = [&](int id) { return (uint32_t)id < (uint32_t)p.n_pages; };
    auto issue = [&](int stage, int step, int2 ids) {
        const uint32_t base = ring_base + stage * (4 * TILE);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int key0 = key_first + 32 * step + 16 * h, slot = key0 - page_of(p, key0) * p.page;
            const int id = h ? ids.y : ids.x;
            const int rows = mapped(id) ? min(p.page - slot, lk - key0) : 0;
            const __amdgpu_buffer_rsrc_t k_rs = page_rows(k_head, mapped(id) ? id : 0, k_page, slot, k_row, rows, D);
            const __amdgpu_buffer_rsrc_t v_rs = page_rows(v_head, mapped(id) ? id : 0, v_page, slot, v_row, rows, D);
            const uint32_t kb = base + h * LH * 1024, vb = kb + 2 * TILE;
            if constexpr (LH == 2) {
                const uint32_t l4[4] = {kb, kb + 1024, vb, vb + 1024};
                const int o4[4] = {koff[0], koff[1], voff[0], voff[1]};
                dma16x4(l4, o4, k_rs, v_rs);
            } else {
#pragma unroll
                for (int j = 0; j < LH; j += 4) {
                    const uint32_t l = kb + j * 1024, l4[4] = {l, l + 1024, l + 2048, l + 3072};
                    const int o4[4] = {koff[j], koff[j + 1], koff[j + 2], koff[j + 3]};
                    dma16x4(l4, o4, k_rs, k_rs);
                }
#pragma unroll
                for (int j = 0; j < LH; j += 4) {
                    const uint32_t l = vb + j * 1024, l4[4] = {l, l + 1024, l + 2048, l + 3072};
                    const int o4[4] = {voff[j], voff[j + 1], voff[j + 2], voff[j + 3]};
                    dma16x4(l4, o4, v_rs, v_rs);
                }
            }
        }
    };

    // Query fragments: lane (c16, g4) holds dims 32 c + 8 g4 .. of row c16 of each block.
    int pos[NR];
    bf16x8 qf[NR][DC];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int row = 16 * r + c16, token = token_of(p, row), head = kvh * p.group + row - token * p.group;
        pos[r] = off + token;
        const __bf16 *src = p.q + (int64_t)(start + token) * p.q_st + (int64_t)head * p.q_sh + 8 * g4;
#pragma unroll
        for (int c = 0; c < DC; ++c) qf[r][c] = row < nrows ? ld_g16(src + 32 * c) : bf16x8{};
    }
    const int p0 = off, p1 = off + token_of(p, nrows - 1) + 1;  // key positions of the first row, past the last

    auto &o = sums.o;
    auto &m = sums.m;
    auto &ls = sums.l;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int db = 0; db < DB; ++db) o[r][db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[r] = kNegInf;
        ls[r] = 0.0f;
    }
    int2 held[NS];  // page ids of the steps in the ring, and of the next to issue
#pragma unroll
    for (int s = 0; s < NS; ++s) held[s] = page_ids(s);
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // the sequence before has read its stages
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
        if (s < steps) issue(s, s, held[s]);
    // The query rows' wait, here once: at their first use it would stand in the loop, and wait for the
    // loads ahead in every step.
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int c = 0; c < DC; ++c) asm volatile("" : "+v"(qf[r][c]));
    for (int step = 0; step < steps; ++step) {
        // The stage of the step before is free once its reads are done; a step's loads are complete once at
        // most the later steps' are in flight.
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
        const int stage = step % NS, ahead = step + NS - 1;
        if (ahead < steps) issue(ahead % NS, ahead, held[NS - 1]);
        const int later = min(steps, ahead + 1) - step - 1;
        if (NS >= 4 && later >= 3) wait_vmcnt<NS >= 4 ? 3 * LPS : 0>();
        else if (NS >= 3 && later >= 2) wait_vmcnt<2 * LPS>();
        else if (later >= 1) wait_vmcnt<LPS>();
        else wait_vmcnt<0>();
        const int2 ids = held[0];
#pragma unroll
        for (int s = 0; s < NS - 1; ++s) held[s] = held[s + 1];
        held[NS - 1] = page_ids(step + NS);
        const __bf16 *kt = ring + stage * (2 * TILE), *vt = kt + TILE;
        const int kt0 = key_first + 32 * step;
        const bool whole = mapped(ids.x) && mapped(ids.y) && block_full(kt0, khi, p0, p1, p.wl, p.wr);
        f32x4 sc[NR][2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int r = 0; r < NR; ++r) sc[r][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const bf16x8 ka = ld_s16(kt + 16 * b * D + (kbase ^ (32 * c)));
#pragma unroll
                for (int r = 0; r < NR; ++r)
                    sc[r][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, qf[r][c], sc[r][b], 0, 0, 0);
            }
        }
        bf16x8 pb[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            if (!whole) {
                uint32_t km = key_mask(kt0, g4, pos[r], khi, p.wl, p.wr);  // bit x: key kt0 + 4 g4 + x
                const uint32_t low = (1u << (16 - 4 * g4)) - 1u;          // of the step's first 16 keys
                km &= (mapped(ids.x) ? low : 0u) | (mapped(ids.y) ? ~low : 0u);
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[r][b][i] = mask_score(sc[r][b][i], km, 16 * b + i);
            }
            const f32x4 &a = sc[r][0], &z = sc[r][1];
            const float mx =
                fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])));
            // Raised only when a row exceeds it by 2^8; the four lanes of a row share m.
            if (wave_any(mx * c2 > m[r] + 8.0f)) {
                float top = fmaxf(mx, __shfl_xor(mx, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float mnew = fmaxf(m[r], top * c2);
                const float alpha = mnew == kNegInf ? 1.0f : exp2_fast(m[r] - mnew);
                m[r] = mnew;
                ls[r] *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db) o[r][db] *= alpha;
            }
            const float muse = m[r] == kNegInf ? 0.0f : m[r];
#pragma unroll
            for (int i = 0; i < 8; ++i) pb[r][i] = (__bf16)exp2_fast(fmaf(sc[r][i >> 2][i & 3], c2, -muse));
#pragma unroll
            for (int i = 0; i < 4; ++i) ls[r] = sum2(pb[r], i, ls[r]);
        }
        auto values = [&](int db) {
            const __bf16 *at = vt + (vbase ^ (16 * db));
            const bf16x4 lo = tr16(at), hi = tr16(at + 16 * D);
            return bf16x8(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        uint32_t bad = 0;
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            bf16x8 va = values(db);
            if (!whole) bad |= clean8(va);
#pragma unroll
            for (int r = 0; r < NR; ++r) o[r][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb[r], o[r][db], 0, 0, 0);
        }
        if (wave_any(bad != 0)) {
#pragma unroll 1
            for (int key = 0; key < BN; ++key) {
#pragma unroll
                for (int db = 0; db < DB; ++db) {  // dims 16 db + 4 g4 ..
                    const int unit = (2 * db + (g4 >> 1)) ^ unit_swz<CPR>(key);
                    const bf16x4 v4 = *reinterpret_cast<const bf16x4 *>(vt + key * D + unit * 8 + 4 * (g4 & 1));
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const bool reach = reaches(p, pos[r], kt0 + key, khi);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[r][db][i] += reach ? only_nonfinite(v4[i]) : 0.0f;
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        ls[r] += __shfl_xor(ls[r], 16);
        ls[r] += __shfl_xor(ls[r], 32);
    }
}

template <int D, int NR, int NS>
__device__ __forceinline__ void row_runs(const PagedParams &p, int wave, __bf16 *ring) {
    constexpr int DB = D / 16;
    const int worker = over_kv_heads(p, wave), kvh = wave - worker * p.hkv;
    const int lane = threadIdx.x & 63, c16 = lane & 15, g4 = lane >> 4;
    RowLanes seqs = row_lanes(p, 0);
    int total = seqs.all;
    for (int base = 64; base < p.n_seq; base += 64) total += row_lanes(p, base).all;
    const int run = row_run(p, total), first = worker * run;
    if (first >= total) return;
    const int last = min(total, first + run);

    int before = 0;  // steps of the sequences before seqs.base
    for (int x = first; x < last;) {
        while (before + seqs.all <= x) {
            before += seqs.all;
            seqs = row_lanes(p, seqs.base + 64);
        }
        const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + seqs.upto > x));
        const int begin = before + __builtin_amdgcn_readlane(seqs.upto - seqs.n, who);
        const int end = before + __builtin_amdgcn_readlane(seqs.upto, who);
        RowWork w;
        w.seq = seqs.base + who;
        w.start = __builtin_amdgcn_readlane(seqs.seq.start, who);
        w.nrows = __builtin_amdgcn_readlane(seqs.seq.rows, who);
        w.lk = __builtin_amdgcn_readlane(seqs.seq.lk, who);
        w.off = w.lk - token_of(p, w.nrows);
        keys_of(p, w.off, w.lk, 0, w.nrows, w.key_first, w.khi);
        w.key_first += 32 * (x - begin);
        w.steps = min(last, end) - x;
        const bool whole_row = begin >= first && end <= last;  // no other wave has keys of these rows
        const int slot_of = begin < first ? 0 : 1;
        x += w.steps;
        RowSums<D, NR> sums;
        row_steps<D, NR, NS>(p, kvh, w, ring, sums);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = 16 * r + c16;
            if (row >= w.nrows) continue;
            if (whole_row) {
                const int token = token_of(p, row), head = kvh * p.group + row - token * p.group;
                const float l = sums.l[r], inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
                __bf16 *dst = p.o + (int64_t)(w.start + token) * p.o_st + (int64_t)head * p.o_sh + 4 * g4;
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    const f32x4 &o = sums.o[r][db];
                    *reinterpret_cast<bf16x4 *>(dst + 16 * db) =
                        round4<false>(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv, bf16x4{});
                }
            } else {
                const int64_t slot = row_slot(p, wave, slot_of) + row;
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    *reinterpret_cast<f32x4 *>(p.part_o + slot * D + 16 * db + 4 * g4) = sums.o[r][db];
                if (g4 == 0) {
                    p.part_ml[2 * slot] = sums.m[r];
                    p.part_ml[2 * slot + 1] = sums.l[r];
                }
            }
        }
    }
}

template <int D, int NR, int NS>
__global__ __launch_bounds__(64) void paged_row_kernel(PagedParams p) {
    __shared__ __attribute__((aligned(16))) __bf16 ring[NS * 2 * 32 * D];
    row_runs<D, NR, NS>(p, blockIdx.x, ring);
}

// Small calls: a workgroup per sequence and kv head, its waves' sums added through LDS. No parts and no second
// launch, at the price of one CU's rate for all of a sequence's keys. Bound by latency, of the launch, the
// bounds, the page ids and each wave's steps in turn: four sequences of U{100..600} keys at 32:8 heads of 128
// 9.3 us (12.2 as runs; three waves of three stages 9.6), one of 64 keys 5.8.
template <int D>
constexpr int kGroupWaves = D == 256 ? 2 : 4;

template <int D, int NR>
__global__ __launch_bounds__(64 * kGroupWaves<D>) void paged_group_kernel(PagedParams p) {
    constexpr int NW = kGroupWaves<D>, BM = 16 * NR, DB = D / 16, kRing = 2 * 2 * 32 * D;
    __shared__ __attribute__((aligned(16))) __bf16 ring[NW * kRing];
    __shared__ float stat[NW][2][BM];
    static_assert(sizeof(ring) >= (size_t)NW * BM * D * 4, "the waves' sums fit the stages");
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), c16 = lane & 15, g4 = lane >> 4;
    const int seq = over_kv_heads(p, blockIdx.x), kvh = blockIdx.x - seq * p.hkv;
    RowWork w;
    w.seq = seq;
    w.start = p.cu[seq];
    const int L = p.cu[seq + 1] - w.start;
    w.lk = p.lens[seq];
    if (!served(p, w.start, L, w.lk)) return;
    w.nrows = L * p.group;
    w.off = w.lk - L;
    int klo;
    keys_of(p, w.off, w.lk, 0, w.nrows, klo, w.khi);
    const int steps = max(0, (w.khi - klo + 31) >> 5), per = (steps + NW - 1) / NW;
    w.key_first = klo + 32 * per * wave;
    w.steps = min(per, max(0, steps - per * wave));
    RowSums<D, NR> sums;
    row_steps<D, NR, 2>(p, kvh, w, ring + wave * kRing, sums);
#pragma unroll
    for (int r = 0; r < NR; ++r)
        if (g4 == 0) {
            stat[wave][0][16 * r + c16] = sums.m[r];
            stat[wave][1][16 * r + c16] = sums.l[r];
        }
    __syncthreads();
    // A row's largest maximum and the inverse of its sum, and the weight of sums at maximum m.
    auto weight = [](float m, float mx) { return m == kNegInf ? 0.0f : exp2_fast(m - mx); };
    auto normaliser = [&](int row, float &mx) {
        mx = stat[0][0][row];
#pragma unroll
        for (int j = 1; j < NW; ++j) mx = fmaxf(mx, stat[j][0][row]);
        float l = 0.0f;
#pragma unroll
        for (int j = 0; j < NW; ++j) l = fmaf(stat[j][1][row], weight(stat[j][0][row], mx), l);
        return l > 0.0f || l != l ? 1.0f / l : 0.0f;
    };
    // Where a thread adds more than two pieces, the waves weigh their own sums first (12 sequences of 8 drafted
    // tokens at 8:2 heads of 256 15.0 against 16.8 us), else each piece is weighed where it is added (four of one
    // token at 32:8 of 128 9.3 against 9.5).
    constexpr bool kFirst = BM * (D / 4) > 2 * 64 * NW;
    float *all = reinterpret_cast<float *>(ring);  // [NW][BM][D]
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int row = 16 * r + c16;
        float mine = 1.0f;
        if constexpr (kFirst) {
            float mx;
            mine = normaliser(row, mx);
            mine *= weight(sums.m[r], mx);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
            *reinterpret_cast<f32x4 *>(all + (wave * BM + row) * D + 16 * db + 4 * g4) = sums.o[r][db] * mine;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < w.nrows * (D / 4); i += 64 * NW) {
        const int row = i / (D / 4), dim = 4 * (i - row * (D / 4));
        float mx, inv = 1.0f;
        if constexpr (!kFirst) inv = normaliser(row, mx);
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const f32x4 y = *reinterpret_cast<const f32x4 *>(all + (j * BM + row) * D + dim);
            if constexpr (kFirst) x += y;
            else x += y * weight(stat[j][0][row], mx);
        }
        const int token = token_of(p, row), head = kvh * p.group + row - token * p.group;
        *reinterpret_cast<bf16x4 *>(p.o + (int64_t)(w.start + token) * p.o_st + (int64_t)head * p.o_sh + dim) =
            round4<false>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv, bf16x4{});
    }
}

// ----------------------------------------------------------------------------- both at once

// A call of short and long sequences: the first `row_groups` workgroups, one per CU, run the short ones' rows with
// as many waves as have their two stages in a tile's LDS, the others the long ones' tiles beside them, so that
// what waits for memory and what waits for products share the CUs (40 decoding users and two chunks of 2,048
// rows at 32:8 heads of 128 793 us, one after the other 844).
template <int D>
constexpr int kRowWaves = D == 64 ? 4 : D == 128 ? 2 : 1;

template <int D, bool SPLIT>
__global__ __launch_bounds__(256, 2) void paged_both_kernel(PagedParams p, int row_groups) {
    constexpr int kRing = 2 * 2 * 32 * D, kRows = kRowWaves<D> * kRing;
    __shared__ __attribute__((aligned(16))) __bf16 ring[kRows > kTileLds<D> ? kRows : kTileLds<D>];
    if ((int)blockIdx.x >= row_groups) return tile_item<D, SPLIT>(p, blockIdx.x - row_groups, ring);
    const int wave = uniform(threadIdx.x >> 6), index = blockIdx.x * kRowWaves<D> + wave;
    if (wave < kRowWaves<D> && index < p.workers * p.hkv) row_runs<D, 1, 2>(p, index, ring + wave * kRing);
}

// ----------------------------------------------------------------------------- the parts' sums

// Adds the parts of split rows, weighed against the row's largest maximum, in a fixed order: the result does
// not depend on which wave finished first. Rows of one part are already written.

// Where a packed row of one query head has its parts: count (0 or 1: nothing to add), the first's slot, and the
// others' base and step: part i > 0 is slot rest + i * step.
struct RowParts {
    int count;
    int64_t first, rest, step;
};

// A packed row's sequence and where its parts lie, the same for all query heads. RUNS: sequences of few rows
// have parts; TILES: the others have.
struct RowPlace {
    int token, rows, lk;                    // token < 0: a row that the call does not serve
    int begin, end, run;                    // steps of its sequence, and of a wave's run
    int item0, tiles, steps;                // its first item that leaves parts, its tiles, the steps of a chunk
};

template <bool RUNS, bool TILES>
__device__ __forceinline__ RowPlace row_place(const PagedParams &p, int row) {
    RowPlace r;
    r.token = -1;
    r.rows = r.lk = r.begin = r.end = r.item0 = r.tiles = r.steps = 0;
    if constexpr (TILES) r.steps = chunk_steps(p, tile_lanes(p, 0));
    int total = 0, items = 0;
    for (int base = 0; base < p.n_seq; base += 64) {
        const TileLanes t = tile_lanes(p, base);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(t.seq.rows > 0 && t.seq.start <= row &&
                                                         row < t.seq.start + token_of(p, t.seq.rows));
        const bool here = hit && r.token < 0;
        const int who = here ? __builtin_ctzll(hit) : 0;
        if (here) {
            r.token = row - __builtin_amdgcn_readlane(t.seq.start, who);
            r.rows = __builtin_amdgcn_readlane(t.seq.rows, who);
            r.lk = __builtin_amdgcn_readlane(t.seq.lk, who);
        }
        if constexpr (RUNS) {
            const RowLanes seqs = row_lanes(p, base);
            if (here) {
                r.begin = total + __builtin_amdgcn_readlane(seqs.upto - seqs.n, who);
                r.end = total + __builtin_amdgcn_readlane(seqs.upto, who);
            }
            total += seqs.all;
        }
        if constexpr (TILES) {
            const int n = split_items(t, r.steps), upto = wave_scan(n);
            if (here) {
                r.item0 = items + __builtin_amdgcn_readlane(upto - n, who);
                r.tiles = __builtin_amdgcn_readlane(t.tiles, who);
            }
            items += __builtin_amdgcn_readlane(upto, 63);
        } else if (!RUNS || (here && r.rows > p.few)) {
            break;  // nothing more to know
        }
    }
    r.run = row_run(p, total);
    return r;
}

template <bool RUNS, bool TILES>
__device__ __forceinline__ RowParts parts_of(const PagedParams &p, const RowPlace &r, int qh) {
    RowParts s;
    s.count = 0;
    s.first = s.rest = s.step = 0;
    const int kvh = token_of(p, qh), at = r.token * p.group + qh - kvh * p.group;  // row of the sequence
    if (r.token < 0) return s;
    if (RUNS && r.rows <= p.few) {
        const int w0 = r.begin / r.run;
        s.count = (r.end - 1) / r.run - w0 + 1;
        s.first = row_slot(p, w0 * p.hkv + kvh, 1) + at;
        s.rest = row_slot(p, w0 * p.hkv + kvh, 0) + at;
        s.step = row_slot(p, p.hkv, 0);
    } else if (TILES && r.rows > p.few) {
        const int tile = at / kTileRows;
        int klo, khi;
        keys_of(p, r.lk - token_of(p, r.rows), r.lk, tile * kTileRows, min(r.rows, (tile + 1) * kTileRows), klo, khi);
        s.count = max(0, khi - klo + 64 * r.steps - 1) / (64 * r.steps);
        s.first = s.rest = tile_slot(p, r.item0 + tile, kvh) + at - tile * kTileRows;
        s.step = (int64_t)r.tiles * p.hkv * kTileRows;
    }
    return s;
}

__device__ __forceinline__ int64_t part_at(const RowParts &r, int i) { return i == 0 ? r.first : r.rest + i * r.step; }

__device__ __forceinline__ void store_merged(const PagedParams &p, int row, int qh, int dim, const f32x4 &o, float l) {
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    *reinterpret_cast<bf16x4 *>(p.o + (int64_t)row * p.o_st + (int64_t)qh * p.o_sh + dim) =
        round4<false>(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv, bf16x4{});
}

// Many rows: a wave per row and 64 / (D / 4) query heads, D / 4 lanes each. No LDS and no barrier, so that the
// chip's waves are on their loads (a workgroup per row and head: 2,048 rows of 12 heads of 64 in 6 parts
// 47 us, this 16).
template <int D, bool RUNS, bool TILES>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p) {
    constexpr int LPR = D / 4, HEADS = 64 / LPR, AHEAD = 4;
    const int lane = threadIdx.x & 63, sub = lane % LPR, dim = 4 * sub, per = (p.hq + HEADS - 1) / HEADS;
    const int64_t item = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
    if (item >= (int64_t)p.total_q * per) return;
    const int row = (int)(item / per), qh = (int)(item - (int64_t)row * per) * HEADS + lane / LPR;
    const RowPlace place = row_place<RUNS, TILES>(p, row);
    RowParts parts = parts_of<RUNS, TILES>(p, place, min(qh, p.hq - 1));
    if (qh >= p.hq) parts.count = 0;
    if (!wave_any(parts.count > 1)) return;
    const float2 *stats = reinterpret_cast<const float2 *>(p.part_ml);
    float mx = kNegInf;
    for (int i = sub; i < parts.count; i += LPR) mx = fmaxf(mx, stats[part_at(parts, i)].x);
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    float l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int base = 0; wave_any(base < parts.count); base += LPR) {
        const int n = min(LPR, parts.count - base);
        const float2 ml = sub < n ? stats[part_at(parts, base + sub)] : float2{kNegInf, 0.0f};
        const float w = ml.x == kNegInf ? 0.0f : exp2_fast(ml.x - mx);
        l = fmaf(ml.y, w, l);
        for (int c0 = 0; wave_any(c0 < n); c0 += AHEAD) {
            f32x4 x[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (c0 + u < n) x[u] = *reinterpret_cast<const f32x4 *>(p.part_o + part_at(parts, base + c0 + u) * D + dim);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const float wc = __shfl(w, ((lane / LPR) * LPR + c0 + u) & 63);  // every lane takes part
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = c0 + u < n ? fmaf(x[u][i], wc, o[i]) : o[i];
            }
        }
    }
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) l += __shfl_xor(l, d);
    if (parts.count > 1) store_merged(p, row, qh, dim, o, l);
}

// Few rows, which may have many parts: 64 dims of a (row, query head) have a workgroup of their own, its
// sixteen groups of lanes taking the parts in turn.
constexpr int kMaxParts = 2048;

template <int D, bool RUNS, bool TILES>
__global__ __launch_bounds__(256) void paged_merge_long_kernel(PagedParams p) {
    __shared__ float weight[kMaxParts];
    __shared__ float red[2][4];
    __shared__ __attribute__((aligned(16))) float sums[16][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int row = blockIdx.x, qh = blockIdx.y;
    const RowParts parts = parts_of<RUNS, TILES>(p, row_place<RUNS, TILES>(p, row), qh);
    const int count = min(parts.count, kMaxParts);
    if (count <= 1) return;
    const float2 *stats = reinterpret_cast<const float2 *>(p.part_ml);
    float mx = kNegInf;
    for (int i = tid; i < count; i += 256) mx = fmaxf(mx, weight[i] = stats[part_at(parts, i)].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    if (lane == 0) red[0][wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float l = 0.0f;
    for (int i = tid; i < count; i += 256) {
        const float w = weight[i] == kNegInf ? 0.0f : exp2_fast(weight[i] - mx);
        weight[i] = w;
        l = fmaf(stats[part_at(parts, i)].y, w, l);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const int g = tid >> 4, at = 4 * (tid & 15), dim = 64 * blockIdx.z + at;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int c = g; c < count; c += 16) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(p.part_o + part_at(parts, c) * D + dim);
        const float wc = weight[c];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(x[i], wc, o[i]);
    }
    *reinterpret_cast<f32x4 *>(&sums[g][at]) = o;
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) o += *reinterpret_cast<const f32x4 *>(&sums[i][at]);
    store_merged(p, row, qh, dim, o, l);
}

}  // namespace pe
