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
    uint32_t page_mul, page_shift;  // n / page = (n * page_mul >> 32) >> page_shift for 0 <= n < 2^31
    int32_t wl, wr;                 // window (-1: unbounded); causal folded into wr = 0
    int32_t max_seqlen, max_seqlen_k;
    int32_t one_tile;               // 1: every sequence has at most one query tile, its own
    int32_t chunk;                  // keys per workgroup along grid y
    int32_t total_q;
    float c;                        // softmax_scale * log2(e)
    float *part_o, *part_ml;        // split calls: [chunks][total_q][hq][D] and [..][2], fp32
};

__device__ __forceinline__ int page_of(const PagedParams &p, int key) {
    return (int)(__umulhi((uint32_t)key, p.page_mul) >> p.page_shift);
}

// The page table as constant memory: a wave's uniform entry is then a scalar load, which the waits for its
// vector loads do not see (as ordinary memory, which the direct-to-LDS loads might change for all the
// compiler knows, it is a vector load behind every load in flight).
typedef const __attribute__((address_space(4))) int32_t *PageIds;

__device__ __forceinline__ PageIds page_ids_of(const PagedParams &p, int seq) {
    return (PageIds)(uintptr_t)(p.table + (int64_t)seq * p.table_st);
}

// A query tile of `bm` rows: sequence, first row, rows of the sequence, key position of its token 0.
struct PagedTile {
    int seq, row0, rows, start, lk, off;
    bool valid;
};

// The sequence's bounds, and whether the call serves it (else its rows are left unwritten).
__device__ __forceinline__ void load_bounds(const PagedParams &p, PagedTile &t) {
    t.start = uniform(p.cu[t.seq]);
    const int L = uniform(p.cu[t.seq + 1]) - t.start;
    t.lk = uniform(p.lens[t.seq]);
    t.off = t.lk - L;
    t.rows = L * p.group;
    t.valid = L > 0 && L <= p.max_seqlen && t.lk >= 0 && t.lk <= p.max_seqlen_k &&
              t.lk <= (int64_t)p.max_pages * p.page && t.start >= 0 && (int64_t)t.start + L <= p.total_q;
}

// Tile `entry` of the call. Every wave finds it from the bounds: 64 sequences at a time, one per lane,
// their tiles numbered by a scan.
__device__ __forceinline__ PagedTile find_tile(const PagedParams &p, int entry, int bm) {
    PagedTile t;
    t.valid = false;
    t.seq = entry;
    t.row0 = 0;
    if (!p.one_tile) {
        const int lane = threadIdx.x & 63;
        for (int base = 0;; base += 64) {
            if (base >= p.n_seq) return t;
            const int s = base + lane;
            int n = 0;
            if (s < p.n_seq) {
                const int L = p.cu[s + 1] - p.cu[s];
                if (L > 0 && L <= p.max_seqlen) n = (int)(((int64_t)L * p.group + bm - 1) / bm);
            }
            const int upto = wave_scan(n), all = __builtin_amdgcn_readlane(upto, 63);
            if (entry < all) {
                const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > entry));
                t.seq = base + who;
                t.row0 = (entry - __builtin_amdgcn_readlane(upto - n, who)) * bm;
                break;
            }
            entry -= all;
        }
    }
    load_bounds(p, t);
    t.valid = t.valid && t.row0 < t.rows;
    return t;
}

// Keys [klo, khi) that some of the tile's rows reach by position, klo on a multiple of 64.
__device__ __forceinline__ void tile_keys(const PagedParams &p, const PagedTile &t, int bm, int &klo, int &khi) {
    const int t0 = t.row0 / p.group, t1 = (min(t.rows, t.row0 + bm) - 1) / p.group;
    klo = p.wl >= 0 ? max(0, t.off + t0 - p.wl) & ~63 : 0;
    khi = t.lk;
    if (p.wr >= 0) khi = (int)max((int64_t)0, min((int64_t)t.lk, (int64_t)t.off + t1 + 1 + p.wr));
}

__device__ __forceinline__ int tile_chunks(const PagedParams &p, int klo, int khi) {
    return max(1, (khi - klo + p.chunk - 1) / p.chunk);
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

// Place of a row's share of one chunk, to be added to the other chunks' by paged_merge_kernel.
__device__ __forceinline__ int64_t paged_slot(const PagedParams &p, int chunk, int row, int head) {
    return ((int64_t)chunk * p.total_q + row) * p.hq + head;
}

// The 16 keys from `key` on (a multiple of 16) lie in a mapped page.
__device__ __forceinline__ bool mapped16(const PagedParams &p, PageIds table, int key) {
    return (uint32_t)table[min(page_of(p, key), p.max_pages - 1)] < (uint32_t)p.n_pages;
}

// Tiles of 128 rows, four waves of 32, over keys that all of them read from LDS: chunks of prompts,
// and any call. Two stages of 64 keys (32 at head_dim 256), filled by direct global-to-LDS loads of the
// next while the waves work on one: 64 KB, two workgroups per CU (head_dim 64: three stages, 48 KB).
template <int D, bool SPLIT>
__global__ __launch_bounds__(256) void paged_tile_kernel(PagedParams p) {
    constexpr int BM = 128, BN = D == 256 ? 32 : 64, NS = D == 64 ? 3 : 2;
    constexpr int NB = BN / 32, DC = D / 16, DB = D / 32, CPR = D / 8;
    constexpr int TILE = BN * D, UPW = TILE / 8 / 64 / 4, LPS = 2 * UPW, KPW = BN / 4;
    static_assert(UPW == 2 || UPW == 4, "loads go out four at a time");
    __shared__ __attribute__((aligned(16))) __bf16 ring[NS][2][TILE];

    const int entry = blockIdx.x / p.hkv, kvh = blockIdx.x - entry * p.hkv;
    const PagedTile t = find_tile(p, entry, BM);
    if (!t.valid) return;
    int klo, khi;
    tile_keys(p, t, BM, klo, khi);
    const int chunks = SPLIT ? tile_chunks(p, klo, khi) : 1;
    if constexpr (SPLIT) {
        if ((int)blockIdx.y >= chunks) return;
        klo += blockIdx.y * p.chunk;
        khi = min(khi, klo + p.chunk);
    }
    const int ntiles = khi > klo ? (khi - klo + BN - 1) / BN : 0;

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 31, kg = lane >> 5;
    const int r0 = t.row0 + 32 * wave, row = r0 + col;
    const bool wave_active = r0 < t.rows;
    const int token = row / p.group, head = kvh * p.group + row - token * p.group;
    const int pos = t.off + token;  // the row's key position
    // Key positions of the wave's first row and past its last.
    const int p0 = t.off + r0 / p.group, p1 = t.off + (min(t.rows, r0 + 32) - 1) / p.group + 1;

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
        const int key = u / CPR, ch = (u % CPR) ^ swz<CPR>(key);
        koff[j] = (key - wave * KPW) * k_row + ch * 16;
        voff[j] = (key - wave * KPW) * v_row + ch * 16;
    }
    const uint32_t ring_base = uniform((int)lds_addr(&ring[0][0][0]));
    auto page_id = [&](int step) { return table[min(page_of(p, klo + step * BN + wave * KPW), p.max_pages - 1)]; };
    auto issue = [&](int stage, int step, int id) {
        const int key0 = klo + step * BN + wave * KPW, slot = key0 - page_of(p, key0) * p.page;
        const bool mapped = (uint32_t)id < (uint32_t)p.n_pages;
        const int rows = mapped ? min(p.page - slot, t.lk - key0) : 0;
        const int64_t page = mapped ? id : 0;
        const __amdgpu_buffer_rsrc_t k_rs =
            make_rsrc(p.k + page * p.k_sp + slot * p.k_st + kvh * p.k_sh, rows_bytes(rows, p.k_st, D));
        const __amdgpu_buffer_rsrc_t v_rs =
            make_rsrc(p.v + page * p.v_sp + slot * p.v_st + kvh * p.v_sh, rows_bytes(rows, p.v_st, D));
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
    const int kbase = col * D + (kg ^ swz<CPR>(col)) * 8;
    const int vbase0 = vkey * D + ((vdim >> 3) ^ swz<CPR>(vkey)) * 8 + (vdim & 4);
    const int vbase1 = (vkey + 8) * D + ((vdim >> 3) ^ swz<CPR>(vkey + 8)) * 8 + (vdim & 4);

    f32x16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[db][j] = 0.0f;
    float m = kNegInf, ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const float c2 = p.c;

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
    for (int step = 0; step < ntiles; ++step) {
        // The step's loads are complete once at most the later steps' are in flight.
        const int later = min(ntiles, step + NS - 1) - step - 1;
        if (NS >= 3 && later >= 1) wait_vmcnt<LPS>();
        else wait_vmcnt<0>();
        __syncthreads();
        if (step + NS - 1 < ntiles) {  // into the stage that all waves have left
            issue((step + NS - 1) % NS, step + NS - 1, next_id);
            next_id = page_id(step + NS);
        }
        if (!wave_active) continue;
        const __bf16 *kt = &ring[step % NS][0][0], *vt = &ring[step % NS][1][0];
        const int kt0 = klo + step * BN;
        f32x16 s[NB];
        bool live[NB], whole[NB];
        float mp[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int kb0 = kt0 + 32 * b;
            live[b] = block_live(kb0, khi, p0, p1, p.wl, p.wr);
            whole[b] = true;
            if (live[b]) {
                f32x16 acc;
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[j] = 0.0f;
#pragma unroll
                for (int c = 0; c < DC; ++c) acc = mfma32(ld_s16(kt + 32 * b * D + (kbase ^ (16 * c))), qf[c], acc);
                whole[b] = block_full(kb0, khi, p0, p1, p.wl, p.wr);
                if (!whole[b] || any_hole) {
                    uint32_t km = key_mask(kb0, kg, pos, khi, p.wl, p.wr);
                    if (any_hole) {
                        const uint32_t low = (1u << (16 - 4 * kg)) - 1u;  // bits of the block's first 16 keys
                        km &= (mapped16(p, table, kb0) ? low : 0u) | (mapped16(p, table, kb0 + 16) ? ~low : 0u);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[j] = mask_score(acc[j], km, acc_key(j, 0));
                }
                s[b] = acc;
#pragma unroll
                for (int j = 0; j < 16; ++j) mp[j & 3] = fmaxf(mp[j & 3], acc[j]);
            }
        }
        // The maximum is raised only when a row exceeds it by 2^8: the exponentials stay in range and
        // most tiles skip the rescale. The two lanes of a row share m.
        const float mx = fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3]));
        if (wave_any(mx * c2 > m + 8.0f)) {
            const float mnew = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)) * c2);
            const float alpha = mnew == kNegInf ? 1.0f : exp2_fast(m - mnew);
            m = mnew;
#pragma unroll
            for (int i = 0; i < 4; ++i) ls[i] *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[db][j] *= alpha;
        }
        const float muse = m == kNegInf ? 0.0f : m;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (!live[b]) continue;
#pragma unroll
            for (int j = 0; j < 16; ++j) s[b][j] = exp2_fast(fmaf(s[b][j], c2, -muse));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bf16x8 pb = to_bf16x8(s[b], 8 * h);
#pragma unroll
                for (int i = 0; i < 4; ++i) ls[i] = sum2(pb, i, ls[i]);
                const __bf16 *vh = vt + (32 * b + 16 * h) * D;
                auto values = [&](int db) {
                    const bf16x4 lo = tr16(vh + (vbase0 ^ (32 * db))), hi = tr16(vh + (vbase1 ^ (32 * db)));
                    return bf16x8(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                uint32_t bad = 0;
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    bf16x8 va = values(db);
                    if (!whole[b]) bad |= clean8(va);
                    o[db] = mfma32(va, pb, o[db]);
                }
                if (!wave_any(bad != 0)) continue;
#pragma unroll 1
                for (int key = 0; key < 16; ++key) {
                    const bool reach = reaches(p, pos, kt0 + 32 * b + 16 * h + key, khi);
#pragma unroll
                    for (int q = 0; q < 4 * DB; ++q) {  // dims 8 q + 4 kg ..
                        const bf16x4 v4 = *reinterpret_cast<const bf16x4 *>(vh + key * D + (q ^ swz<CPR>(key)) * 8 + 4 * kg);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[q >> 2][4 * (q & 3) + i] += reach ? only_nonfinite(v4[i]) : 0.0f;
                    }
                }
            }
        }
    }
    if (!wave_active) return;
    const float lsum = (ls[0] + ls[1]) + (ls[2] + ls[3]);
    const float l = lsum + __shfl_xor(lsum, 32);
    if (SPLIT && chunks > 1) {
        if (row >= t.rows) return;
        const int64_t slot = paged_slot(p, blockIdx.y, t.start + token, head);
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
    const __amdgpu_buffer_rsrc_t o_rs =
        make_rsrc(p.o + (int64_t)t.start * p.o_st,
                  (uint32_t)(((int64_t)(t.rows / p.group - 1) * p.o_st + (p.hq - 1) * p.o_sh + D) * 2));
    const int ooff = row < t.rows ? (int)((token * p.o_st + head * p.o_sh) * 2) : kVoidOffset;
    store_block<DB, false>(o, inv, kg, o_rs, ooff, o_rs, 0);
}

// Tiles of 16 NR rows: single decoded tokens, a few drafted ones. There is one row tile per (sequence, kv
// head) or little more, and the time is that of reading its keys once, so the waves share nothing: each takes
// every NW-th 32-key step of the workgroup's chunk through stages of its own (no barrier; a step waits for the
// wave's own loads), and the waves' sums are added at the end. Products on v_mfma_f32_16x16x32_bf16, lane l:
// c16 = l % 16, g4 = l / 16:
//  * S^T = K . Q^T per 16 keys: A = key c16 by dims 32 c + 8 g4 .., B = the lane's row; lane l then holds, for
//    row c16, keys 4 g4 + i.
//  * O^T = V^T . P^T per 16 dims: B = the lane's own 8 probabilities, k-slot 8 g4 + i standing for key
//    4 g4 + i and 8 g4 + 4 + i for key 16 + 4 g4 + i; A = V^T for the same keys by two transposing reads;
//    lane l accumulates dims 16 db + 4 g4 + i of row c16.
template <int D, int NR, int NW, int NS, bool SPLIT>
__global__ __launch_bounds__(64 * NW) void paged_row_kernel(PagedParams p) {
    constexpr int BM = 16 * NR, BN = 32, DC = D / 32, DB = D / 16, CPR = D / 8;
    constexpr int TILE = BN * D;           // elements of a step's K (or V)
    constexpr int LH = CPR / 4;            // 1 KB loads of 16 keys
    constexpr int LPS = 4 * LH;            // loads of a step
    static_assert(LH == 2 || LH % 4 == 0, "loads go out four at a time");
    __shared__ __attribute__((aligned(16))) __bf16 ring[NW][NS][2][TILE];
    static_assert(sizeof(ring) >= (size_t)NW * BM * D * 4, "the waves' sums fit the ring");
    __shared__ float stat[NW][2][BM];

    const int entry = blockIdx.x / p.hkv, kvh = blockIdx.x - entry * p.hkv;
    const PagedTile t = find_tile(p, entry, BM);
    if (!t.valid) return;
    int klo, khi;
    tile_keys(p, t, BM, klo, khi);
    const int chunks = SPLIT ? tile_chunks(p, klo, khi) : 1;
    if constexpr (SPLIT) {
        if ((int)blockIdx.y >= chunks) return;
        klo += blockIdx.y * p.chunk;
        khi = min(khi, klo + p.chunk);
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    const int all = khi > klo ? (khi - klo + BN - 1) / BN : 0;       // steps of the workgroup
    const int steps = all > wave ? (all - wave + NW - 1) / NW : 0;  // and of the wave
    const PageIds table = page_ids_of(p, t.seq);

    const int k_row = (int)p.k_st * 2, v_row = (int)p.v_st * 2;
    int koff[LH], voff[LH];
#pragma unroll
    for (int j = 0; j < LH; ++j) {
        const int u = j * 64 + lane, key = u / CPR, ch = (u % CPR) ^ swz<CPR>(key);
        koff[j] = key * k_row + ch * 16;
        voff[j] = key * v_row + ch * 16;
    }
    const uint32_t ring_base = uniform((int)lds_addr(&ring[wave][0][0][0]));
    auto key_of = [&](int step) { return klo + (step * NW + wave) * BN; };
    // The ids of the pages that hold a step's two halves.
    auto page_ids = [&](int step) {
        const int key = key_of(step), last = p.max_pages - 1;
        return int2{table[min(page_of(p, key), last)], table[min(page_of(p, key + 16), last)]};
    };
    auto mapped = [&](int id) { return (uint32_t)id < (uint32_t)p.n_pages; };
    auto issue = [&](int stage, int step, int2 ids) {
        const uint32_t base = ring_base + stage * (4 * TILE);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int key0 = key_of(step) + 16 * h, slot = key0 - page_of(p, key0) * p.page, id = h ? ids.y : ids.x;
            const int rows = mapped(id) ? max(0, min(p.page - slot, t.lk - key0)) : 0;
            const int64_t page = mapped(id) ? id : 0;
            const __amdgpu_buffer_rsrc_t k_rs =
                make_rsrc(p.k + page * p.k_sp + slot * p.k_st + kvh * p.k_sh, rows_bytes(rows, p.k_st, D));
            const __amdgpu_buffer_rsrc_t v_rs =
                make_rsrc(p.v + page * p.v_sp + slot * p.v_st + kvh * p.v_sh, rows_bytes(rows, p.v_st, D));
            const uint32_t kb = base + h * LH * 1024, vb = kb + 2 * TILE;
            if constexpr (LH == 2) {
                const uint32_t l4[4] = {kb, kb + 1024, vb, vb + 1024};
                const int o4[4] = {koff[0], koff[1], voff[0], voff[1]};
                dma16x4(l4, o4, k_rs, v_rs);
            } else {
#pragma unroll
                for (int j = 0; j < LH; j += 4) {
                    const uint32_t lk[4] = {kb + j * 1024, kb + j * 1024 + 1024, kb + j * 1024 + 2048, kb + j * 1024 + 3072};
                    const int ok[4] = {koff[j], koff[j + 1], koff[j + 2], koff[j + 3]};
                    dma16x4(lk, ok, k_rs, k_rs);
                }
#pragma unroll
                for (int j = 0; j < LH; j += 4) {
                    const uint32_t lv[4] = {vb + j * 1024, vb + j * 1024 + 1024, vb + j * 1024 + 2048, vb + j * 1024 + 3072};
                    const int ov[4] = {voff[j], voff[j + 1], voff[j + 2], voff[j + 3]};
                    dma16x4(lv, ov, v_rs, v_rs);
                }
            }
        }
    };

    // Query fragments: lane (c16, g4) holds dims 32 c + 8 g4 .. of row c16 of each block.
    int pos[NR];
    bf16x8 qf[NR][DC];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int row = t.row0 + 16 * r + c16, token = row / p.group, head = kvh * p.group + row - token * p.group;
        pos[r] = t.off + token;
        const __bf16 *src = p.q + (int64_t)(t.start + token) * p.q_st + (int64_t)head * p.q_sh + 8 * g4;
#pragma unroll
        for (int c = 0; c < DC; ++c) qf[r][c] = row < t.rows ? ld_g16(src + 32 * c) : bf16x8{};
    }
    // Key positions of the tile's first row and past its last.
    const int p0 = t.off + t.row0 / p.group, p1 = t.off + (min(t.rows, t.row0 + BM) - 1) / p.group + 1;
    // Place of the operands' first chunk in a stage; the swizzle exchanges whole units and depends on the
    // key's low four bits alone, so chunk c is 32 c elements on by exclusive or, and 16 keys on by sum.
    const int vkey = 4 * g4 + (c16 >> 2), vdim = 4 * (c16 & 3);
    const int kbase = c16 * D + (g4 ^ swz<CPR>(c16)) * 8;
    const int vbase = vkey * D + ((vdim >> 3) ^ swz<CPR>(vkey)) * 8 + (vdim & 4);

    f32x4 o[NR][DB];
    float m[NR], ls[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int db = 0; db < DB; ++db) o[r][db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[r] = kNegInf;
        ls[r] = 0.0f;
    }
    const float c2 = p.c;

    int2 held[NS];  // page ids of the steps in the ring, and of the next to issue
    if (steps > 0) {
#pragma unroll
        for (int s = 0; s < NS; ++s) held[s] = page_ids(s);
#pragma unroll
        for (int s = 0; s < NS - 1; ++s)
            if (s < steps) issue(s, s, held[s]);
    }
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
        if (NS >= 3 && later >= 2) wait_vmcnt<2 * LPS>();
        else if (later >= 1) wait_vmcnt<LPS>();
        else wait_vmcnt<0>();
        const int2 ids = held[0];
#pragma unroll
        for (int s = 0; s < NS - 1; ++s) held[s] = held[s + 1];
        held[NS - 1] = page_ids(step + NS);
        const __bf16 *kt = &ring[wave][stage][0][0], *vt = &ring[wave][stage][1][0];
        const int kt0 = key_of(step);
        const bool gap = !mapped(ids.x) || !mapped(ids.y);
        const bool whole = !gap && block_full(kt0, khi, p0, p1, p.wl, p.wr);
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
                const uint32_t low = (1u << (16 - 4 * g4)) - 1u;
                km &= (mapped(ids.x) ? low : 0u) | (mapped(ids.y) ? ~low : 0u);
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[r][b][i] = mask_score(sc[r][b][i], km, 16 * b + i);
            }
            const f32x4 &a = sc[r][0], &z = sc[r][1];
            const float mx = fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])));
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
                    const int unit = (2 * db + (g4 >> 1)) ^ swz<CPR>(key);
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

    // The waves' sums through LDS, then one thread per four dims of a row weighs and adds them.
    __syncthreads();
    float *sums = reinterpret_cast<float *>(&ring[0][0][0][0]);  // [NW][BM][D]
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        float l = ls[r] + __shfl_xor(ls[r], 16);
        l += __shfl_xor(l, 32);
        if (g4 == 0) {
            stat[wave][0][16 * r + c16] = m[r];
            stat[wave][1][16 * r + c16] = l;
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
            *reinterpret_cast<f32x4 *>(sums + (wave * BM + 16 * r + c16) * D + 16 * db + 4 * g4) = o[r][db];
    }
    __syncthreads();
    const int rows = min(BM, t.rows - t.row0);
    for (int i = tid; i < rows * (D / 4); i += 64 * NW) {
        const int r = i / (D / 4), dim = 4 * (i - r * (D / 4));
        float mx = stat[0][0][r];
#pragma unroll
        for (int w = 1; w < NW; ++w) mx = fmaxf(mx, stat[w][0][r]);
        float l = 0.0f;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float weight = stat[w][0][r] == kNegInf ? 0.0f : exp2_fast(stat[w][0][r] - mx);
            l = fmaf(stat[w][1][r], weight, l);
            const f32x4 y = *reinterpret_cast<const f32x4 *>(sums + (w * BM + r) * D + dim);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = fmaf(y[j], weight, x[j]);
        }
        const int row = t.row0 + r, token = row / p.group, head = kvh * p.group + row - token * p.group;
        if (SPLIT && chunks > 1) {
            const int64_t slot = paged_slot(p, blockIdx.y, t.start + token, head);
            *reinterpret_cast<f32x4 *>(p.part_o + slot * D + dim) = x;
            if (dim == 0) {
                p.part_ml[2 * slot] = mx;
                p.part_ml[2 * slot + 1] = l;
            }
        } else {
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            *reinterpret_cast<bf16x4 *>(p.o + (int64_t)(t.start + token) * p.o_st + (int64_t)head * p.o_sh + dim) =
                round4<false>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv, bf16x4{});
        }
    }
}

// Adds the chunks of split rows: one workgroup per (query row, head). The chunks' maxima and sums (at
// most kMaxChunks) are read at once and turned into weights in LDS; then groups of D / 4 lanes take the
// chunks in turn and their sums are added in a fixed order, so the result does not depend on which
// workgroup finished first.
constexpr int kMaxChunks = 1024;

template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p, int bm, int max_chunks) {
    constexpr int LPR = D / 4, GROUPS = 256 / LPR;
    __shared__ float weight[kMaxChunks];
    __shared__ float red[2][4];
    __shared__ __attribute__((aligned(16))) float sums[GROUPS][D];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int row = blockIdx.x, qh = blockIdx.y;  // packed token, query head
    PagedTile t;
    t.seq = -1;
    for (int base = 0; base < p.n_seq; base += 64) {
        const int s = base + lane;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(s < p.n_seq && p.cu[s] <= row && row < p.cu[s + 1]);
        if (hit) {
            t.seq = base + __builtin_ctzll(hit);
            break;
        }
    }
    if (t.seq < 0) return;
    load_bounds(p, t);
    if (!t.valid) return;
    t.row0 = ((row - t.start) * p.group + qh % p.group) / bm * bm;
    int klo, khi;
    tile_keys(p, t, bm, klo, khi);
    const int chunks = min(max_chunks, tile_chunks(p, klo, khi));
    if (chunks <= 1) return;  // written by its one workgroup
    const int64_t slot0 = paged_slot(p, 0, row, qh), stride = paged_slot(p, 1, 0, 0);
    float2 ml[kMaxChunks / 256];
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < kMaxChunks / 256; ++i) {
        ml[i] = float2{kNegInf, 0.0f};
        if (tid + 256 * i < chunks) ml[i] = reinterpret_cast<const float2 *>(p.part_ml)[slot0 + (tid + 256 * i) * stride];
        mx = fmaxf(mx, ml[i].x);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    if (lane == 0) red[0][wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxChunks / 256; ++i) {
        const float w = ml[i].x == kNegInf ? 0.0f : exp2_fast(ml[i].x - mx);
        weight[tid + 256 * i] = w;
        l = fmaf(ml[i].y, w, l);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const int g = tid / LPR, dim = 4 * (tid % LPR);
    const float *src = p.part_o + slot0 * D + dim;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int c = g; c < chunks; c += GROUPS) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(src + c * stride * D);
        const float wc = weight[c];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(x[i], wc, o[i]);
    }
    *reinterpret_cast<f32x4 *>(&sums[g][dim]) = o;
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) o += *reinterpret_cast<const f32x4 *>(&sums[i][dim]);
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const bf16x4 y = round4<false>(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv, bf16x4{});
    *reinterpret_cast<bf16x4 *>(p.o + (int64_t)row * p.o_st + (int64_t)qh * p.o_sh + dim) = y;
}

}  // namespace pe
