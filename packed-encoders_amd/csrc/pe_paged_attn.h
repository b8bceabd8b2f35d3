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

// 0x8000 bits set for the halves of a bf16 pair that are infinite or NaN.
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

__device__ __forceinline__ uint32_t nonfinite8(const bf16x8 &x) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 u = __builtin_bit_cast(u32x4, x);
    return nonfinite2(u[0]) | nonfinite2(u[1]) | nonfinite2(u[2]) | nonfinite2(u[3]);
}

// Element 0 of x where `keep`, zero elsewhere and in the others.
__device__ __forceinline__ bf16x8 only_first(const bf16x8 &x, bool keep) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 u = __builtin_bit_cast(u32x4, x);
    return __builtin_bit_cast(bf16x8, u32x4{keep ? u[0] & 0xffffu : 0u, 0u, 0u, 0u});
}

__device__ __forceinline__ bf16x8 next_first(const bf16x8 &x) {
    return __builtin_shufflevector(x, x, 1, 2, 3, 4, 5, 6, 7, 0);
}

// Place of a row's share of one chunk, to be added to the other chunks' by paged_merge_kernel.
__device__ __forceinline__ int64_t paged_slot(const PagedParams &p, int chunk, int row, int head) {
    return ((int64_t)chunk * p.total_q + row) * p.hq + head;
}

// The 16 keys from `key` on (a multiple of 16) lie in a mapped page.
__device__ __forceinline__ bool mapped16(const PagedParams &p, const int32_t *table, int key) {
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

    const int32_t *table = p.table + (int64_t)t.seq * p.table_st;
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
    int kbase_c[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) kbase_c[c] = col * D + ((2 * c + kg) ^ swz<CPR>(col)) * 8;
    const int vi = lane & 15, vg = lane >> 4;
    const int vkey0 = 4 * (vg >> 1) + (vi >> 2);
    const int vdim0 = 16 * (vg & 1) + 4 * (vi & 3);
    int vbase[2][DB];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const int key = 8 * half + vkey0, dim = 32 * db + vdim0;
            vbase[half][db] = key * D + (((dim >> 3) ^ swz<CPR>(key)) * 8) + (dim & 4);
        }

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
                for (int c = 0; c < DC; ++c) acc = mfma32(ld_s16(kt + 32 * b * D + kbase_c[c]), qf[c], acc);
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
                bf16x8 pb = to_bf16x8(s[b], 8 * h);
#pragma unroll
                for (int i = 0; i < 4; ++i) ls[i] = sum2(pb, i, ls[i]);
                const __bf16 *vh = vt + (32 * b + 16 * h) * D;
                auto values = [&](int db) {
                    const bf16x4 lo = tr16(vh + vbase[0][db]), hi = tr16(vh + vbase[1][db]);
                    return bf16x8(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                bool apart = false;
                if (!whole[b]) {
                    uint32_t bad = 0;
#pragma unroll
                    for (int db = 0; db < DB; ++db) bad |= nonfinite8(values(db));
                    apart = wave_any(bad != 0);
                }
                if (!apart) {
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db] = mfma32(values(db), pb, o[db]);
                    continue;
                }
                // A masked key may hold an infinity or NaN, whose product with a zero probability is NaN:
                // one key at a time, and only the rows that reach it take the sum. Element e of the
                // operands is key 16 h + 8 (e / 4) + 4 kg + e % 4; eight turns bring pb back.
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    bf16x8 va = values(db);
#pragma unroll 1
                    for (int e = 0; e < 8; ++e) {
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const int key = kt0 + 32 * b + 16 * h + 8 * (e >> 2) + 4 * g + (e & 3);
                            const bool reach = key < khi && (p.wl < 0 || pos - key <= p.wl) &&
                                               (p.wr < 0 || key - pos <= p.wr);
                            const f32x16 sum = mfma32(only_first(va, kg == g), only_first(pb, kg == g), o[db]);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[db][j] = reach ? sum[j] : o[db][j];
                        }
                        pb = next_first(pb);
                        va = next_first(va);
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

// Adds the chunks of split rows: one workgroup per (query row, head). The chunks' maxima and sums (at
// most 256) are read at once, one per thread, and turned into weights in LDS; then groups of D / 4
// lanes take the chunks in turn and their sums are added in a fixed order, so the result does not
// depend on which workgroup finished first.
template <int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p, int bm, int max_chunks) {
    constexpr int LPR = D / 4, GROUPS = 256 / LPR;
    __shared__ float weight[256];
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
    const float2 ml = tid < chunks ? reinterpret_cast<const float2 *>(p.part_ml)[slot0 + tid * stride]
                                   : float2{kNegInf, 0.0f};
    float mx = ml.x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    if (lane == 0) red[0][wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float w = ml.x == kNegInf ? 0.0f : exp2_fast(ml.x - mx);
    weight[tid] = w;
    float l = ml.y * w;
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
