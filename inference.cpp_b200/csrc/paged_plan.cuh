// What the kernels of ib_attention_paged share: how the work of a batch is cut, and small
// pieces of arithmetic.
#pragma once
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "paged.cuh"

namespace ib {

// ---- cutting a batch into pieces ---------------------------------------------------------
// Sequences with rows in [min_rows, max_rows] take part, in tiles of R rows and key tiles of KT
// positions, in n_pieces pieces of at least `least` positions of one token.
struct CutRule {
    int R, KT, min_rows, max_rows, n_pieces, least;
    int filled = 0; // parts: at least so many positions where there is one for each SM (0: `least`)
    int fixed = 0;  // positions that beginning a tile costs as much as (pieces)
    // trees: every tile of a sequence costs the same, whole key tiles; none is cut so that a side has
    // fewer than `least` positions, nor one of fewer than `uncut`
    bool flat = false;
    int uncut = 0;
    bool split = false;  // tcgen05: one query tile, its key tiles shared out (paged_tensor.cu)
    __device__ __forceinline__ int slope() const { return flat ? 0 : R; }
};

// Work is counted in rows x positions, roughly: tile i of a sequence whose first new token is
// at `start` counts G start + (i + 1) R, which has a closed sum over tiles.
struct SeqWork {
    SeqInfo s;
    long long per_head, all;  // per kv head; 0: the sequence does not take part
};

constexpr unsigned long long kMostWork = 1ull << 62;  // sums of what device memory says saturate
__device__ __forceinline__ long long add_work(long long a, long long b) {
    return (long long)min((unsigned long long)a + (unsigned long long)b, kMostWork);
}

// What a tile of a sequence costs before the rows' own positions.
__device__ __forceinline__ long long start_work(const CutRule& rule, const SeqInfo& s, int G) {
    const int seen = rule.flat ? (max(s.L, 0) + rule.KT - 1) / rule.KT * rule.KT : max(s.L - s.n, 0);
    return (long long)G * (seen + rule.fixed);
}

// flat: the key tile of nkt at which a cut `x` into a tile's work falls.  What beginning a tile costs is
// half on either side of it.  A cut close to an end falls on the end: the side that is left begins
// no tile and has nothing to be joined.  Two kernels have to agree, so every step is rounded by itself.
__device__ __forceinline__ int flat_cut(const CutRule& rule, long long x, int G, int nkt) {
    const float per = __fdividef(1.f, (float)(G * rule.KT));
    const int kt = __float2int_rn(__fsub_rn(__fmul_rn((float)x, per),
                                            __fdividef((float)(rule.fixed / 2), (float)rule.KT)));
    if (nkt * rule.KT < rule.uncut) return 2 * kt < nkt ? 0 : nkt;
    const int few = (rule.least + rule.KT - 1) / rule.KT;
    return kt < few ? 0 : nkt - kt < few ? nkt : kt;
}
// The key tiles that a tile's rows see.
__device__ __forceinline__ int seen_tiles(const CutRule& rule, int start, int row0, int rows, int G) {
    return (max(0, start + (row0 + rows - 1) / G + 1) + rule.KT - 1) / rule.KT;
}

__device__ __forceinline__ long long tiles_work(long long t, long long start_g, int R) {
    return t * start_g + (long long)R * (t * (t + 1) / 2);
}

__device__ __forceinline__ SeqWork seq_work(const PagedView& w, const CutRule& rule, int b) {
    SeqWork x;
    x.s = seq_info(w, b);
    const int G = w.H / w.Hkv, rows = x.s.n * G;
    const bool in = rows >= rule.min_rows && rows <= rule.max_rows;
    const int tiles = in ? (rows + rule.R - 1) / rule.R : 0;
    x.per_head = tiles_work(tiles, start_work(rule, x.s, G), rule.slope());
    // at most 2^23 tiles of at most 2^38 each (paged_check_batch)
    x.all = x.per_head * w.Hkv;
    return x;
}

// One tile, or a part of one, in a worker's piece.
struct Segment {
    SeqInfo s;
    int hk, tile, rows;
    int start;      // position of the sequence's first new token
    int kt0, kt1;   // key tiles
    int part;       // where its partial result goes, -1: it is the whole tile
    int row0;       // first row
};

struct Piece {
    long long at, end, len;  // work left to do: [at, end); of a piece
    long long base;          // where sequence b begins
    int b, no;
    SeqWork x;
};

// flat: a piece behind its first segment.
struct Following {
    long long left, start_g;  // work left to do; of a tile of the sequence
    SeqInfo s;
    int b, no, hk, tile, tiles;  // of the last segment; the sequence's tiles
};

// Piece `no` of the batch, into shared memory; found: whether there is one.  Every thread of the
// CTA (NT of them) calls it; a barrier has to follow.
template <int NT>
__device__ __forceinline__ void find_piece(const PagedView& w, const CutRule& rule, int no, Piece* out,
                                           int* found) {
    __shared__ long long sh_sum[NT / 32][2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    SeqWork x0{};
    long long work = 0, tokens = 0;
    for (int b = tid; b < w.n_seqs; b += NT) {
        const SeqWork x = seq_work(w, rule, b);
        work = add_work(work, x.all);
        tokens += x.s.n;
        if (b == tid) x0 = x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        work = add_work(work, __shfl_xor_sync(0xffffffffu, work, o));
        tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
    }
    if (lane == 0) sh_sum[warp][0] = work, sh_sum[warp][1] = tokens;
    if (tid == 0) *found = 0;
    __syncthreads();
    work = tokens = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
        work = add_work(work, sh_sum[i][0]);
        tokens += sh_sum[i][1];
    }
    if (tokens > w.n_tokens) {  // a cu_q that is not in order names rows twice: no work
        if (tid == 0) paged_fault(PAGED_BAD_LEN);
        return;
    }
    const long long len = max((work + rule.n_pieces - 1) / rule.n_pieces,
                              (long long)rule.least * (w.H / w.Hkv));
    const long long want = no * len;
    if (want >= work) return;
    long long before = 0;
    for (int b0 = 0; b0 < w.n_seqs; b0 += NT) {
        const int b = b0 + tid;
        SeqWork x = x0;
        if (b0 > 0 && b < w.n_seqs) x = seq_work(w, rule, b);
        if (b >= w.n_seqs) x.all = 0;
        long long a = x.all;  // inclusive sum
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, a, o);
            if (lane >= o) a = add_work(a, y);
        }
        __syncthreads();  // sh_sum has been read
        if (lane == 31) sh_sum[warp][0] = a;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) {
            if (i == warp) a = add_work(a, all);
            all = add_work(all, sh_sum[i][0]);
        }
        const long long a0 = add_work(before, a - x.all);
        if (want >= a0 && want < a0 + x.all) {
            *out = Piece{want, min(work, want + len), len, a0, b, no, x};
            *found = 1;
        }
        before = add_work(before, all);
        if (want < before) break;  // the same for every thread
    }
}

// The tile that work `p.at` of the piece's sequence is in.
struct TileAt {
    int hk, tile;
    long long x0, all;  // how far into its work; all of it
};
template <bool FLAT>
__device__ __forceinline__ TileAt tile_at(const PagedView& w, const CutRule& rule, const Piece& p,
                                          long long start_g) {
    TileAt t;
    const int G = w.H / w.Hkv;
    long long u = p.at - p.base;
    t.hk = min((int)__fdividef((float)u, (float)p.x.per_head), w.Hkv - 1);  // to one
    if (t.hk * p.x.per_head > u) --t.hk;
    else if ((t.hk + 1) * p.x.per_head <= u) ++t.hk;
    u -= t.hk * p.x.per_head;
    const int tiles = (p.x.s.n * G + rule.R - 1) / rule.R;
    int lo = 0;  // the last whose work begins at or before u
    if constexpr (FLAT) {
        while (lo + 1 < tiles && u >= start_g) ++lo, u -= start_g;
        t.x0 = u;
        t.all = start_g;
    } else {
        int hi = tiles;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (tiles_work(mid, start_g, rule.slope()) <= u) lo = mid;
            else hi = mid;
        }
        t.x0 = u - tiles_work(lo, start_g, rule.slope());
        t.all = start_g + (long long)(lo + 1) * rule.slope();
    }
    t.tile = lo;
    return t;
}

// The next segment of a piece; false at its end.  Called by whole warps, each for itself.
template <bool FLAT>
__device__ __forceinline__ bool next_segment(const PagedView& w, const CutRule& rule, Piece& p,
                                             Segment& g) {
    while (p.at < p.end) {
    if (p.at >= p.base + p.x.all) {  // on to the next sequence that takes part
        p.base += p.x.all;
        for (int b0 = p.b + 1;; b0 += 32) {
            if (b0 >= w.n_seqs) return false;
            const int b = b0 + (int)(threadIdx.x & 31);
            SeqWork x{};
            if (b < w.n_seqs) x = seq_work(w, rule, b);
            const unsigned has = __ballot_sync(0xffffffffu, x.all > 0);
            if (has) {
                p.b = b0 + __ffs(has) - 1;
                p.x = seq_work(w, rule, p.b);
                break;
            }
        }
    }
    const int G = w.H / w.Hkv;
    const SeqInfo& s = p.x.s;
    const long long start_g = start_work(rule, s, G);
    const TileAt t = tile_at<FLAT>(w, rule, p, start_g);
    g.s = s;
    g.start = s.L - s.n;
    g.hk = t.hk;
    g.tile = t.tile;
    g.row0 = t.tile * rule.R;
    g.rows = min(rule.R, s.n * G - g.row0);
    const long long all = t.all, x0 = t.x0;
    const long long x1 = min(all, x0 + (p.end - p.at));
    const int nkt = seen_tiles(rule, g.start, g.row0, g.rows, G);
    bool whole = x0 == 0 && x1 == all, none = false;
    if constexpr (FLAT) {
        g.kt0 = x0 == 0 ? 0 : flat_cut(rule, x0, G, nkt);
        g.kt1 = x1 == all ? nkt : flat_cut(rule, x1, G, nkt);
        // rows that see nothing are the first piece's
        none = nkt == 0 ? x0 > 0 : g.kt0 == g.kt1;
        whole = g.kt0 == 0 && g.kt1 == nkt;
    } else {
        // the same value for a piece's end and the next one's beginning, and more for more work: that
        // is all a cut needs (three integer divisions of 64 bits took a thousand cycles)
        const float per = __fdividef((float)nkt, (float)all);
        g.kt0 = x0 == 0 ? 0 : min(nkt, (int)((float)x0 * per));
        g.kt1 = x1 == all ? nkt : min(nkt, (int)((float)x1 * per));
    }
    g.part = whole ? -1 : 2 * p.no + (p.at == p.no * p.len ? 0 : 1);
    p.at += x1 - x0;
    if (!FLAT || !none) return true;
    }
    return false;
}

// flat: the segments behind a piece's first one, which begin with their tiles: little code, since each of a
// CTA's roles has its own and misses the instruction cache there.
__device__ __forceinline__ Following following(const PagedView& w, const CutRule& rule, const Piece& p,
                                               const Segment& g) {
    const int G = w.H / w.Hkv;
    return Following{p.end - p.at, start_work(rule, p.x.s, G), p.x.s, p.b, p.no, g.hk, g.tile,
                     (p.x.s.n * G + rule.R - 1) / rule.R};
}
__device__ __forceinline__ bool following_segment(const PagedView& w, const CutRule& rule, Following& p, Segment& g) {
    const int G = w.H / w.Hkv;
    while (p.left > 0) {
        if (++p.tile == p.tiles) {
            p.tile = 0;
            if (++p.hk == w.Hkv) {
                p.hk = 0;
                for (int b0 = p.b + 1;; b0 += 32) {
                    if (b0 >= w.n_seqs) return false;
                    const int b = b0 + (int)(threadIdx.x & 31);
                    const int rows = b < w.n_seqs ? seq_info(w, b).n * G : 0;
                    const unsigned has = __ballot_sync(0xffffffffu, rows >= rule.min_rows && rows <= rule.max_rows);
                    if (has) {
                        p.b = b0 + __ffs(has) - 1;
                        break;
                    }
                }
                p.s = seq_info(w, p.b);
                p.tiles = (p.s.n * G + rule.R - 1) / rule.R;
                p.start_g = start_work(rule, p.s, G);
            }
        }
        const SeqInfo& s = p.s;
        g.s = s;
        g.start = s.L - s.n;
        g.hk = p.hk;
        g.tile = p.tile;
        g.row0 = p.tile * rule.R;
        g.rows = min(rule.R, s.n * G - g.row0);
        const long long x1 = min(p.start_g, p.left);
        const int nkt = seen_tiles(rule, g.start, g.row0, g.rows, G);
        g.kt0 = 0;
        g.kt1 = x1 == p.start_g ? nkt : flat_cut(rule, x1, G, nkt);
        g.part = g.kt1 == nkt ? -1 : 2 * p.no + 1;
        p.left -= x1;
        if (g.kt1 > 0 || nkt == 0) return true;
    }
    return false;
}

// ---- or into parts of tiles ----------------------------------------------------------------
// The other way to cut, for tiles of few rows: every tile by itself into parts of equal length,
// about n_pieces parts in all, each a CTA's only work.  Where several CTAs share an SM the
// scheduler evens them out, and no CTA has to refill its pipeline on the way: 64 single tokens
// over 200..4096 positions (32 heads on 8) take 119 us this way, 141 us in equal pieces that
// run on from tile to tile.
struct Item {
    int b, hk, tile, part, n_parts, part_base;
    int kt0, kt1;  // key tiles of the part
    SeqInfo s;
};

__device__ __forceinline__ void seq_shape(const PagedView& w, const CutRule& rule,
                                          const SeqInfo& s, int& tiles, int& nkt) {
    const int rows = s.n * (w.H / w.Hkv);
    const bool in = rows >= rule.min_rows && rows <= rule.max_rows;
    tiles = in ? (rows + rule.R - 1) / rule.R : 0;
    nkt = max(1, (s.L + rule.KT - 1) / rule.KT);  // a sequence without positions: zeros
}

// Every thread of the CTA (NT threads) calls it; false when there are fewer items.  BY_TILE
// counts row tiles instead of items (the joining kernel).
template <int NT, bool BY_TILE>
__device__ __forceinline__ bool find_item(const PagedView& w, const CutRule& rule, int item,
                                          Item& out) {
    __shared__ long long sh_units[NT / 32];
    __shared__ int sh_scan[NT / 32][2];
    __shared__ Item sh_item;
    __shared__ int sh_found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    SeqInfo s0{};
    int tiles0 = 0, nkt0 = 1;
    long long units = 0;
    for (int b = tid; b < w.n_seqs; b += NT) {
        const SeqInfo s = seq_info(w, b);
        int tiles, nkt;
        seq_shape(w, rule, s, tiles, nkt);
        units += min((long long)tiles * nkt, 1ll << 40);
        if (b == tid) s0 = s, tiles0 = tiles, nkt0 = nkt;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
    if (lane == 0) sh_units[warp] = units;
    if (tid == 0) sh_found = 0;
    __syncthreads();
    units = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) units += sh_units[i];
    units = min(units, 1ll << 45) * w.Hkv;
    long long most = max((long long)(rule.least / rule.KT), (units + rule.n_pieces - 1) / rule.n_pieces);
    if (rule.filled) most = max(most, min((long long)(rule.filled / rule.KT), (units + kSMs - 1) / kSMs));
    const int len = (int)min(most, 0x3fffffffll);
    // cu_q can hold anything: counts are clamped to what cannot be, so that sums stay in range
    // (valid batches have at most 2^22 + n_seqs row tiles, see paged_check_batch)
    constexpr long long MOST = 1 << 23;
    const int room = 2 * rule.n_pieces;  // partials in the workspace
    long long items_before = 0;
    int parts_before = 0;
    for (int b0 = 0; b0 < w.n_seqs; b0 += NT) {
        const int b = b0 + tid;
        SeqInfo s = s0;
        int tiles = tiles0, nkt = nkt0;
        if (b0 > 0) {
            tiles = 0;
            if (b < w.n_seqs) {
                s = seq_info(w, b);
                seq_shape(w, rule, s, tiles, nkt);
            }
        }
        const int parts = (nkt + len - 1) / len;
        const long long n_tiles = b < w.n_seqs ? (long long)tiles * w.Hkv : 0;
        const int n_items = (int)min(BY_TILE ? n_tiles : n_tiles * parts, MOST);
        const int n_parts = parts > 1 ? (int)min(n_tiles * parts, (long long)room + 1) : 0;
        int a = n_items, p = n_parts;  // inclusive scans
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int xa = __shfl_up_sync(0xffffffffu, a, o), xp = __shfl_up_sync(0xffffffffu, p, o);
            if (lane >= o) a += xa, p += xp;
        }
        if (lane == 31) sh_scan[warp][0] = a, sh_scan[warp][1] = p;
        __syncthreads();
        int ta = 0, tp = 0;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) {
            if (i == warp) a += ta, p += tp;
            ta += sh_scan[i][0], tp += sh_scan[i][1];
        }
        const long long at = item - items_before - (a - n_items);
        if (at >= 0 && at < n_items) {
            const int local = (int)at;
            Item it;
            it.b = b;
            it.s = s;
            it.n_parts = parts;
            const int t = BY_TILE ? local : local / parts;
            it.part = BY_TILE ? 0 : local - t * parts;
            it.tile = t / w.Hkv;
            it.hk = t - it.tile * w.Hkv;
            it.part_base = parts_before + (p - n_parts) + t * parts;
            // ranges of equal length, to one key tile
            it.kt0 = (int)((long long)nkt * it.part / parts);
            it.kt1 = (int)((long long)nkt * (it.part + 1) / parts);
            sh_item = it;
            sh_found = parts == 1 || it.part_base + parts <= room ? 1 : 2;
        }
        __syncthreads();
        if (sh_found) break;
        items_before += ta;
        parts_before += tp;
    }
    __syncthreads();
    out = sh_item;
    if (sh_found == 2) paged_fault(PAGED_BAD_LEN);  // more partials than a valid batch has
    return sh_found == 1;
}

// ---- arguments and arithmetic of the kernels ----------------------------------------------
struct RowsArgs {
    PagedView w;
    CutRule rule;
    const float* q;
    float* out;
    int64_t q_stride, out_stride;
    const void *k, *v;  // the layer
    float* part_acc;    // [partial][R][HD] of parts, [partial][HD / 4][R][4] of pieces
    float2* part_ml;    // [partial][R]
    float scale_log2;   // scale * log2(e)
    const uint32_t* mask;  // trees: [token][words], see ib_kv_tree
    int words;
    bool sectors;  // rows of out begin on boundaries of 32 bytes
    // The kernel before is the call's narrow one, which writes other rows and workspace: this one
    // starts beside its last CTAs and waits for it at its own end only, so that what follows
    // finds both complete.  (The narrow kernel lets it start after its own wait for what came
    // before the call.)
    bool beside;
};

// ---- what a node of a tree sees ------------------------------------------------------------
// Row of the masks of the segment's row gr (of row 0 where the segment has none).
__device__ __forceinline__ const uint32_t* mask_row(const RowsArgs& A, int q0, int gr, bool there) {
    return A.mask + (int64_t)(q0 + (there ? (int)A.w.group.div((uint32_t)gr) : 0)) * A.words;
}

// Bits first .. first + 31 of a mask row, where negative ones are the context: all there.
__device__ __forceinline__ uint32_t tree_bits(const uint32_t* row, int words, int first) {
    if (first <= -32) return 0xffffffffu;
    const int at = first >> 5;
    auto word = [&](int i) { return i < 0 ? 0xffffffffu : i < words ? __ldg(row + i) : 0u; };
    return __funnelshift_r(word(at), word(at + 1), first & 31);
}

// The last position that every row of a tile sees if it has a page, from its first row: a causal row
// sees all before its own, a node of a tree all of the context.  Behind it tiles are masked.
template <bool TREE>
__device__ __forceinline__ int all_see(int start, int first_row, int G) {
    return TREE ? start - 1 : start + first_row / G;
}

// Row `gr` of the segment's sequence and kv head.
__device__ __forceinline__ float* out_row(const RowsArgs& A, const Segment& it, int G, int gr) {
    const int tok = (int)A.w.group.div((uint32_t)gr);
    return A.out + (int64_t)(it.s.q0 + tok) * A.out_stride +
           (int64_t)(it.hk * G + gr - tok * G) * A.w.HD;
}
__device__ __forceinline__ const float* q_row(const RowsArgs& A, const Segment& it, int G, int gr) {
    const int tok = (int)A.w.group.div((uint32_t)gr);
    return A.q + (int64_t)(it.s.q0 + tok) * A.q_stride + (int64_t)(it.hk * G + gr - tok * G) * A.w.HD;
}

// Element d of row r of a piece's partial result.  Rows run along memory: they are a thread each
// on tcgen05, and a warp's 16 bytes of each of 32 rows would be 32 lines (a chunk of 2048 tokens
// takes 412 us against 417 that way, prompts on FP32 pages 111 against 114).
__device__ __forceinline__ float* part_at(const RowsArgs& A, int part, int r, int d) {
    return A.part_acc + (((int64_t)part * (A.w.HD / 4) + (d >> 2)) * A.rule.R + r) * 4 + (d & 3);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(valid ? 16 : 0)
                 : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two FP16 values with those that are not finite as zero; odd is set when there were any.
__device__ __forceinline__ uint32_t finite16x2(uint32_t x, bool& odd) {
    if ((x & 0x7c00u) == 0x7c00u) odd = true, x &= 0xffff0000u;
    if ((x & 0x7c000000u) == 0x7c000000u) odd = true, x &= 0x0000ffffu;
    return x;
}

// 2^(8 - e) for a largest element of exponent e, and its inverse (1 and 1 for zero, infinity
// and NaN).
__device__ __forceinline__ float pow2_scale(float top, float& inverse) {
    const int e = max(-100, (int)((__float_as_uint(top) >> 23) & 255u) - 127);
    const bool plain = top == 0.f || e > 127;
    inverse = plain ? 1.f : __uint_as_float((uint32_t)(e - 8 + 127) << 23);
    return plain ? 1.f : __uint_as_float((uint32_t)(8 - e + 127) << 23);
}

// Tiles of many rows on tcgen05, for head_dim up to 128 (paged_tensor.cu).
template <typename KV, bool TREE>
CutRule tensor_rule(int head_dim, int min_rows, int max_rows, bool split);
template <typename KV, bool TREE>
int attn_tensor_launch(const RowsArgs& a, int64_t tiles, int64_t max_pos, cudaStream_t st);
int paged_tensor_fault_take(int* code);

}  // namespace ib
