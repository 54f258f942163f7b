// Attention of few query rows over spans of a paged bfloat16 cache, span by span, with the softmax put together afterwards.
//
//   out[row] = sum_j e^(s_j) v_j / sum_j e^(s_j),   s_j = q[row] . k_j
//
// The sums over any set of spans of j follow from each span's own maximum m, sum l = sum e^(s_j - m) and o = sum e^(s_j - m) v_j:
//   m = max m_i,   l = sum e^(m_i - m) l_i,   o = sum e^(m_i - m) o_i,   out = o / l.
//
// Two operators rest on that.  (1) Sequences that share their first pages: the shared pages are read once for all members of
// a group, whose rows (members x query heads of a key/value head) stand side by side as the columns of one product; what a
// sequence has of its own is spans of its own.  (2) Attention that keeps the weight every cached position is given: the
// scores are written down beside the spans' results, and the pass that puts the spans together turns them into weights.
//
// Shared pages with many rows run on the 5th-generation tensor cores (the second half of this file); all else as follows.
// A block takes one span for up to 8 NT rows.  It streams the span's pages through shared memory with cp.async; inside a page
// each of its four warps owns 16 of the 64 keys: scores are an mma.sync chain with the keys as the 16-row operand and the rows as
// columns, maximum, sum and rescaling are 32-bit, the weights turn into the other operand of the second product by a transposing
// move between lanes, and the weighted values are a second chain into 32-bit accumulators.  The warps' four softmaxes meet at the
// end of the span.  Weights are rounded to bfloat16 for the second product (its operand's type); the sums take them unrounded.
// Memory bounds it where there are pages enough: two sequences of 32,700 positions, 32 heads of 128 on 8, with weights, 57 us of which
// the spans take 47 at 5.6 TB/s.  Pages go through shared memory, not straight to registers, because four query heads would each
// need them there: streamed, the same took 199 us.
#include "common.cuh"
#include "decode_common.cuh"
#include "tma.cuh"
#include "tcgen05.cuh"
#include "span_weights.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

#ifndef GL_HEAD_DIM
#error "compile with -DGL_HEAD_DIM=<head size>: this file is built once per head size a model uses, and knows none itself"
#endif
static_assert(GL_HEAD_DIM % 16 == 0 && GL_HEAD_DIM >= 16 && GL_HEAD_DIM <= 256, "head size: 16..256 in steps of 16");

#define SP_HD GL_HEAD_DIM
#define SP_THREADS 128
#define SP_KS (SP_HD / 16)                          // 16-wide steps along the head size
#define SP_CHUNKS (SP_HD / 8)                       // 16-byte pieces of a row
#define SP_ROW (SP_HD * 2 + 16)                     // padded row in bytes: conflict-free ldmatrix
#define SP_TILE (GL_PAGE * SP_ROW)                  // one page of keys (or values) of one head
#define SP_MAX_NT (SP_HD <= 128 ? 4 : 2)            // columns of 8 rows: the accumulators of more do not fit the registers
#define SP_LOG2E 1.4426950408889634f

struct SpanArgs {
    const __nv_bfloat16* q;       // [rows, nH*hd], scaled
    __nv_bfloat16* out;           // [rows, nH*hd]
    const __nv_bfloat16* k_cache; // [pages, nKV, GL_PAGE, hd]
    const __nv_bfloat16* v_cache;
    const int* seq_row;           // [B] row of q and out, or null (row b is sequence b)
    const int* seq_qlen;          // [B] or null: a sequence of no tokens has no row
    const int* seq_ctx;           // [B] positions cached before this step: a row sees positions 0..seq_ctx[b]
    const int* pages;             // [B, max_pages]
    const int* order;             // sequences group by group (shared pages), or null
    const int* items;             // [n_items, 6]: first member in order, first row, rows, first page, page behind the last, slot
    const int* seq_shared;        // [B, 2]: pages shared with the group, slots they take; or null (nothing is shared)
    float* part_o;                // [B, nH, slots, hd]
    float* part_ml;               // [B, nH, slots, 2]
    float* scores;                // [B, nH, reach] or null
    float* weights;               // [pages, nKV, GL_PAGE] or null
    float* given;                 // [B, nKV, reach]: where sequences may hold a page together, what each gives its positions; or null
    int B, nH, nKV, max_pages, n_pages, n_items, splits, slots, chunks, reach;
    int short_spans;              // a block has a page or two to walk
    int early, held;              // set by the launchers: see the kernel
};

__device__ __forceinline__ void sp_cp16(unsigned dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes));
}
__device__ __forceinline__ void sp_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void sp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// rows [0, n_valid) of a page (64 rows of hd bf16) to padded rows; the rest is zero, so that what an earlier sequence left there
// cannot reach a product
__device__ __forceinline__ void sp_load_page(unsigned dst, const __nv_bfloat16* src, int n_valid) {
#pragma unroll
    for (int j = 0; j < SP_KS; ++j) {
        const int i = threadIdx.x + j * SP_THREADS;
        const int r = i / SP_CHUNKS, c = i - r * SP_CHUNKS;
        const bool ok = r < n_valid;
        sp_cp16(dst + r * SP_ROW + c * 16, ok ? (const void*)((const unsigned char*)src + (size_t)i * 16) : (const void*)src, ok ? 16 : 0);
    }
}
__device__ __forceinline__ void sp_ldm2(unsigned addr, unsigned& a, unsigned& b) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr));
}
// lane (r, t) holds elements (r, 2t) and (r, 2t + 1) of an 8 x 8 matrix of 16-bit numbers; it gets (2t, r) and (2t + 1, r)
__device__ __forceinline__ unsigned sp_transpose(unsigned v) {
    unsigned o;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(o) : "r"(v));
    return o;
}
__device__ __forceinline__ float sp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Maxima are kept as powers of two, m log2(e): every factor is then one difference and one power.  The factor that a partial
// result with maximum m_i takes in one with maximum m >= m_i (nothing seen yet: both -inf):
__device__ __forceinline__ float sp_factor(float m_i, float m) { return m_i == m ? 1.0f : sp_exp2(m_i - m); }

// loads that stay behind the wait before them (what another kernel wrote meanwhile)
__device__ __forceinline__ float2 sp_read(const float2* p) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float4 sp_read(const float4* p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}


// The end of a block whose split is one of a cluster: fin_o [rows][hd] and fin_ml [rows][2] are its result, in its shared memory.
// The blocks put their results and what the shared pages gave together: every block the factors of all parts, a row a warp, then its
// share of the outputs, four at a time.  held [rows][a.held]: its scores, which ``scale`` makes powers of two, or nothing; behind them room
// for the factors; stat: room for [rows][2].
struct SpanEnd { int seq, g, head, rows, p_begin, p_end, total; };
__device__ __forceinline__ void span_join(const SpanArgs& a, const SpanEnd& e, const float* fin_o, const float* fin_ml, float* held, float* stat,
                                          const int* pg, float scale) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rows = e.rows, b = e.seq;
    cg::cluster_group cluster = cg::this_cluster();
    const int S = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int n_pre = a.seq_shared ? a.seq_shared[2 * b + 1] : 0, parts = S + n_pre;
    float* fac = held + (a.weights ? rows * a.held : 0);           // [rows][parts]: factor / sum
    if (a.early) gl_grid_wait();
    if (S > 1) cluster.sync();
    else __syncthreads();
    for (int r = warp; r < rows; r += blockDim.x / 32) {
        const float2* pre = (const float2*)a.part_ml + ((size_t)b * a.nH + e.head + r) * a.slots - S;
        auto part = [&](int k) { return k < S ? ((const float2*)(S > 1 ? cluster.map_shared_rank((float*)fin_ml, k) : fin_ml))[r] : sp_read(pre + k); };
        float m = -INFINITY, l = 0.f;
        for (int k = lane; k < parts; k += 32) m = fmaxf(m, part(k).x);
        m = gl_warp_max(m);
        for (int k = lane; k < parts; k += 32) {
            const float2 ml = part(k);
            const float f = sp_factor(ml.x, m);
            fac[r * parts + k] = f;
            l = fmaf(f, ml.y, l);
        }
        l = gl_warp_sum(l);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        for (int k = lane; k < parts; k += 32) fac[r * parts + k] *= inv;
        if (lane == 0) { stat[2 * r] = m; stat[2 * r + 1] = inv; }
    }
    __syncthreads();
    for (int i = tid * S + rank; i < rows * (SP_HD / 4); i += blockDim.x * S) {
        const int r = i / (SP_HD / 4), c = i - r * (SP_HD / 4);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float f, const float4 v) {
            sum.x = fmaf(f, v.x, sum.x); sum.y = fmaf(f, v.y, sum.y); sum.z = fmaf(f, v.z, sum.z); sum.w = fmaf(f, v.w, sum.w);
        };
        for (int k = 0; k < S; ++k) add(fac[r * parts + k], ((const float4*)(S > 1 ? cluster.map_shared_rank((float*)fin_o, k) : fin_o))[i]);
        const float4* pre = (const float4*)a.part_o + (((size_t)b * a.nH + e.head + r) * a.slots) * (SP_HD / 4) + c;
#pragma unroll 8
        for (int k = 0; k < n_pre; ++k) add(fac[r * parts + S + k], sp_read(pre + (size_t)k * (SP_HD / 4)));
        const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
        *(uint2*)(a.out + ((size_t)(a.seq_row ? a.seq_row[b] : b) * a.nH + e.head + r) * SP_HD + 4 * c) = make_uint2(*(const unsigned*)&lo, *(const unsigned*)&hi);
    }
    if (a.weights) {                                       // this block's scores become weights
        const int n = min(min((e.p_end - e.p_begin) * GL_PAGE, e.total - e.p_begin * GL_PAGE), a.held);
        for (int i = tid; i < n; i += blockDim.x) {
            float given = 0.f;
            for (int r = 0; r < rows; ++r) given = fmaf(sp_exp2(fmaf(held[r * a.held + i], scale, -stat[2 * r])), stat[2 * r + 1], given);
            const int j = e.p_begin * GL_PAGE + i;
            if (a.given) {
                if (j < a.reach) a.given[((size_t)b * a.nKV + e.g) * a.reach + j] = given;
                continue;
            }
            float* w = a.weights + ((size_t)gl_checked(pg[j / GL_PAGE], a.n_pages, GL_BAD_PAGE) * a.nKV + e.g) * GL_PAGE + j % GL_PAGE;
            // (an addition that nobody waits for; one a position, as no two sequences share it: their order is no matter)
            if (j < e.total - 1) atomicAdd(w, given);
            else *w = given;
        }
    }
    if (S > 1) cluster.sync();                             // a block's memory stays until its peers have read it
}

template <int NT>
__host__ __device__ constexpr int sp_fixed_bytes() {       // queries, then per row: sequence, head, last position seen
    return 8 * NT * SP_ROW + 8 * NT * 12;
}
template <int NT, int STAGES>
__host__ __device__ constexpr size_t sp_smem() {
    const size_t pages = 2 * STAGES * (size_t)SP_TILE;
    const size_t merge = sizeof(float) * (4 * 8 * NT * 2 + 5 * (size_t)SP_HD * 8 * NT + 8 * NT * 2);       // over the pages, when they are done
    return (pages > merge ? pages : merge) + sp_fixed_bytes<NT>();
}

// What a block does: a stretch of shared pages for the rows of an item of the plan (blockIdx.x: the item), or a split of a
// sequence's own pages for the query heads of a key/value head (blockIdx = split, head and its share of the query heads, sequence),
// whose result is written down for the joining kernel, or joined here: the splits are then the blocks of a cluster, meet in
// distributed shared memory, take in what the shared pages gave and write the output.
enum { SP_ITEM = 0, SP_SPLIT = 1, SP_JOIN = 2 };

template <int NT, int MODE, int STAGES>
__global__ void __launch_bounds__(SP_THREADS)
attn_span_kernel(SpanArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr bool SHARED = MODE == SP_ITEM;
    constexpr size_t AREA = sp_smem<NT, STAGES>() - sp_fixed_bytes<NT>();
    const unsigned sbase = ad_smem(smem);
    unsigned char* qs = smem + AREA;                               // [8 NT] rows of queries
    int* row_seq = (int*)(qs + 8 * NT * SP_ROW);                   // [8 NT]
    int* row_head = row_seq + 8 * NT;
    int* row_last = row_head + 8 * NT;
    float* held = (float*)(smem + sp_smem<NT, STAGES>());                  // [rows][a.held] scores of the split's keys, where they are kept
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int grp = lane >> 2, t = lane & 3;
    const int G = a.nH / a.nKV;
    // A kernel over shared pages lets the next one start once everything before both is complete; that one (early) then walks the
    // sequences' own pages beside it and waits for it only where it takes in its results.
    if (!a.early) gl_grid_wait();
    gl_grid_launch_dependents();

    int g, rows, p_begin, p_end, slot, table;
    if (SHARED) {
        const int* it = a.items + 6 * blockIdx.x;
        g = blockIdx.y;
        rows = it[2]; p_begin = it[3]; p_end = it[4]; slot = it[5];
        table = a.order[it[0]];
        if (tid < 8 * NT) {
            const int r = it[1] + tid, b = tid < rows ? a.order[it[0] + r / G] : -1;
            row_seq[tid] = b;
            row_head[tid] = g * G + r % G;
            row_last[tid] = b >= 0 ? a.seq_ctx[b] : -1;
        }
    } else {
        const int b = blockIdx.z;
        g = blockIdx.y / a.chunks;
        if (a.seq_qlen && a.seq_qlen[b] <= 0) return;
        const int per_chunk = (G + a.chunks - 1) / a.chunks, h0 = (blockIdx.y - g * a.chunks) * per_chunk;
        rows = min(per_chunk, G - h0);
        const int pos = a.seq_ctx[b];
        const int first = a.seq_shared ? a.seq_shared[2 * b] : 0;
        const int n = max(0, pos / GL_PAGE + 1 - first);
        const int per = (n + a.splits - 1) / a.splits;
        p_begin = first + (int)blockIdx.x * per;
        p_end = min(first + n, p_begin + per);
        slot = (a.seq_shared ? a.seq_shared[2 * b + 1] : 0) + blockIdx.x;
        table = b;
        if (tid < 8 * NT) {
            row_seq[tid] = tid < rows ? b : -1;
            row_head[tid] = g * G + h0 + tid;
            row_last[tid] = tid < rows ? pos : -1;
        }
    }
    const int* pg = a.pages + (size_t)table * a.max_pages;
    const size_t head_off = (size_t)g * GL_PAGE * SP_HD, page_stride = (size_t)a.nKV * GL_PAGE * SP_HD;
    // (rows of the last page behind a sequence's own last position were never written)
    const int total = a.seq_ctx[table] + 1;
    auto load = [&](int st, int p) {
        const size_t at = (size_t)gl_checked(pg[p], a.n_pages, GL_BAD_PAGE) * page_stride + head_off;
        const int nv = SHARED ? GL_PAGE : min(GL_PAGE, total - p * GL_PAGE);
        sp_load_page(sbase + 2 * st * SP_TILE, a.k_cache + at, nv);
        sp_load_page(sbase + (2 * st + 1) * SP_TILE, a.v_cache + at, nv);
    };
    if (p_begin < p_end) load(0, p_begin);
    __syncthreads();
    for (int i = tid; i < 8 * NT * SP_CHUNKS; i += SP_THREADS) {
        const int r = i / SP_CHUNKS, c = i - r * SP_CHUNKS, b = row_seq[r];
        uint4 v = make_uint4(0, 0, 0, 0);
        if (b >= 0) v = *(const uint4*)(a.q + ((size_t)(a.seq_row ? a.seq_row[b] : b) * a.nH + row_head[r]) * SP_HD + c * 8);
        *(uint4*)(qs + r * SP_ROW + c * 16) = v;
    }
    int least = 0x7fffffff;                                // the earliest last position among the block's rows
    for (int r = 0; r < rows; ++r) least = min(least, row_last[r]);
    const unsigned qaddr = ad_smem(qs) + (lane & 7) * SP_ROW + ((lane >> 3) & 1) * 16;

    float o[NT][SP_KS][4];                                 // [column tile][d tile][d grp | grp + 8, row 2t | 2t + 1]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < SP_KS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
    float m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) { m_run[n][0] = m_run[n][1] = -INFINITY; l_run[n][0] = l_run[n][1] = 0.f; }

    for (int p = p_begin; p < p_end; ++p) {
        const int st = STAGES == 2 ? (p - p_begin) & 1 : 0;
        if (STAGES == 1 && p > p_begin) {
            __syncthreads();                               // the page read last time is free
            load(0, p);
        }
        sp_commit();
        sp_wait<0>();
        __syncthreads();                                   // page p has landed; the stage read last time is free
        if (STAGES == 2 && p + 1 < p_end) load(st ^ 1, p + 1);
        const int j0 = p * GL_PAGE + warp * 16;            // this warp's first key
        if (!SHARED && j0 >= total) continue;
        const unsigned Ks = sbase + 2 * st * SP_TILE, Vs = Ks + SP_TILE;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < SP_KS; ++kk) {
            unsigned af[4];
            ad_ldm4(Ks + (warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * SP_ROW + (kk * 2 + (lane >> 4)) * 16, af);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                unsigned b0, b1;
                sp_ldm2(qaddr + n * 8 * SP_ROW + kk * 32, b0, b1);
                ad_mma(s[n], af, b0, b1);
            }
        }
        if (MODE == SP_JOIN && a.weights) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = n * 8 + 2 * t + (e & 1);
                    const int i = (p - p_begin) * GL_PAGE + warp * 16 + grp + (e >> 1) * 8;
                    if (r < rows && i < a.held) held[r * a.held + i] = s[n][e];
                }
        }
        if (MODE == SP_SPLIT && a.scores) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = n * 8 + 2 * t + (e & 1), j = j0 + grp + (e >> 1) * 8;
                    if (r < rows && j < total && j < a.reach) a.scores[((size_t)table * a.nH + row_head[r]) * a.reach + j] = s[n][e];
                }
        }
        if (j0 + 15 > least) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j0 + grp + (e >> 1) * 8 > row_last[n * 8 + 2 * t + (e & 1)]) s[n][e] = -INFINITY;
        }
        float corr[NT][2];
        bool moved = false;
        unsigned pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float mu[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float mx = fmaxf(s[n][i], s[n][i + 2]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float m_new = fmaxf(m_run[n][i], mx * SP_LOG2E);
                mu[i] = m_new == -INFINITY ? 0.f : m_new;
                corr[n][i] = sp_factor(m_run[n][i], m_new);
                moved = moved || m_new != m_run[n][i];
                m_run[n][i] = m_new;
            }
            const float p0 = sp_exp2(fmaf(s[n][0], SP_LOG2E, -mu[0])), p1 = sp_exp2(fmaf(s[n][1], SP_LOG2E, -mu[1]));
            const float p2 = sp_exp2(fmaf(s[n][2], SP_LOG2E, -mu[0])), p3 = sp_exp2(fmaf(s[n][3], SP_LOG2E, -mu[1]));
            l_run[n][0] = fmaf(l_run[n][0], corr[n][0], p0 + p2);          // summed over the 8 key lanes at the end
            l_run[n][1] = fmaf(l_run[n][1], corr[n][1], p1 + p3);
            const __nv_bfloat162 lo = __floats2bfloat162_rn(p0, p1), hi = __floats2bfloat162_rn(p2, p3);
            pb[n][0] = sp_transpose(*(const unsigned*)&lo);
            pb[n][1] = sp_transpose(*(const unsigned*)&hi);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int dt = 0; dt < SP_KS; ++dt) {
                    o[n][dt][0] *= corr[n][0]; o[n][dt][1] *= corr[n][1];
                    o[n][dt][2] *= corr[n][0]; o[n][dt][3] *= corr[n][1];
                }
        }
#pragma unroll
        for (int dt = 0; dt < SP_KS; ++dt) {
            unsigned vf[4];
            ad_ldm4t(Vs + (warp * 16 + (lane >> 4) * 8 + (lane & 7)) * SP_ROW + (dt * 2 + ((lane >> 3) & 1)) * 16, vf);
#pragma unroll
            for (int n = 0; n < NT; ++n) ad_mma(o[n][dt], vf, pb[n][0], pb[n][1]);
        }
    }
    sp_wait<0>();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l_run[n][i] += __shfl_xor_sync(0xffffffffu, l_run[n][i], 4);
            l_run[n][i] += __shfl_xor_sync(0xffffffffu, l_run[n][i], 8);
            l_run[n][i] += __shfl_xor_sync(0xffffffffu, l_run[n][i], 16);
        }
    // the four warps' softmaxes meet over the pages' memory
    float* ml_w = (float*)smem;                            // [4][8 NT][2]
    float* o_w = ml_w + 4 * 8 * NT * 2;                    // [4][hd][8 NT]
    float* fin_o = o_w + 4 * SP_HD * 8 * NT;               // [rows][hd] this split's result, for the cluster
    float* fin_ml = fin_o + 8 * NT * SP_HD;                // [rows][2]
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (grp == 0)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ml_w[(warp * 8 * NT + n * 8 + 2 * t + i) * 2] = m_run[n][i];
                ml_w[(warp * 8 * NT + n * 8 + 2 * t + i) * 2 + 1] = l_run[n][i];
            }
#pragma unroll
        for (int dt = 0; dt < SP_KS; ++dt) {
            float* ow = o_w + ((size_t)warp * SP_HD + dt * 16 + grp) * (8 * NT) + n * 8 + 2 * t;
            *(float2*)ow = make_float2(o[n][dt][0], o[n][dt][1]);
            *(float2*)(ow + 8 * 8 * NT) = make_float2(o[n][dt][2], o[n][dt][3]);
        }
    }
    __syncthreads();
    for (int i = tid; i < rows * SP_HD; i += SP_THREADS) {
        const int r = i / SP_HD, d = i - r * SP_HD;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, ml_w[(w * 8 * NT + r) * 2]);
        float ov = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = sp_factor(ml_w[(w * 8 * NT + r) * 2], m);
            ov = fmaf(f, o_w[((size_t)w * SP_HD + d) * (8 * NT) + r], ov);
            l = fmaf(f, ml_w[(w * 8 * NT + r) * 2 + 1], l);
        }
        if (MODE == SP_JOIN) {
            fin_o[i] = ov;
            if (d == 0) { fin_ml[2 * r] = m; fin_ml[2 * r + 1] = l; }
            continue;
        }
        const size_t at = ((size_t)row_seq[r] * a.nH + row_head[r]) * a.slots + slot;
        a.part_o[at * SP_HD + d] = ov;
        if (d == 0) { a.part_ml[at * 2] = m; a.part_ml[at * 2 + 1] = l; }
    }
    if (MODE != SP_JOIN) return;
    const SpanEnd e = {table, g, row_head[0], rows, p_begin, p_end, total};
    span_join(a, e, fin_o, fin_ml, held, ml_w, pg, SP_LOG2E);
}

// The spans of a sequence put together: blockIdx = (x, key/value head, sequence).  The first ``shares`` blocks of a head turn the scores
// of a thousand positions each into weights, added up over the query heads, four positions a thread so that their scores and
// page numbers are under way together; a position new in this step starts from nothing, whatever its place held.  The G blocks
// behind them put a query head's output together, the spans dealt out to as many threads a number as there are.
// Latency bounds it: two reads that depend on one another, and a write.
#define SP_JOIN_THREADS 256
#define SP_JOIN_KEYS 4
template <bool GIVEN>
__global__ void __launch_bounds__(SP_JOIN_THREADS)
attn_span_join_kernel(SpanArgs a, int shares) {
    extern __shared__ float ml_all[];                      // [G][2]: maximum, 1 / sum
    constexpr int PER = SP_JOIN_THREADS / SP_HD > 0 ? SP_JOIN_THREADS / SP_HD : 1;          // threads that share a number of the output
    __shared__ float sums[PER][SP_HD];
    const int b = blockIdx.z, g = blockIdx.y, G = a.nH / a.nKV, tid = threadIdx.x, lane = tid & 31;
    gl_grid_wait();
    gl_grid_launch_dependents();
    if (a.seq_qlen && a.seq_qlen[b] <= 0) return;
    const int n = (a.seq_shared ? a.seq_shared[2 * b + 1] : 0) + a.splits, own = (int)blockIdx.x - shares;
    const int pos = a.seq_ctx[b], most = min(pos + 1, a.reach), j0 = (int)blockIdx.x * SP_JOIN_THREADS * SP_JOIN_KEYS + tid;
    if (own < 0 && j0 - tid >= most) return;
    for (int i = own < 0 ? tid >> 5 : own + (tid >> 5) * G; i < G; i += SP_JOIN_THREADS / 32) {      // (all heads, or the block's)
        const float* ml = a.part_ml + ((size_t)b * a.nH + g * G + i) * a.slots * 2;
        float m = -INFINITY, l = 0.f;
        for (int s = lane; s < n; s += 32) m = fmaxf(m, ml[2 * s]);
        m = gl_warp_max(m);
        for (int s = lane; s < n; s += 32) l = fmaf(sp_factor(ml[2 * s], m), ml[2 * s + 1], l);
        l = gl_warp_sum(l);
        if (lane == 0) { ml_all[2 * i] = m; ml_all[2 * i + 1] = 1.0f / l; }
    }
    __syncthreads();
    if (own >= 0) {
        const size_t row = (size_t)b * a.nH + g * G + own, at = row * a.slots;
        const float m = ml_all[2 * own], inv = ml_all[2 * own + 1];
        if (tid < PER * SP_HD) {
            const int d = tid % SP_HD, first = tid / SP_HD;
            float o = 0.f;
#pragma unroll 8
            for (int s = first; s < n; s += PER) o = fmaf(sp_factor(a.part_ml[(at + s) * 2], m), a.part_o[(at + s) * SP_HD + d], o);
            sums[first][d] = o;
        }
        __syncthreads();
        if (tid < SP_HD) {
            float o = 0.f;
#pragma unroll
            for (int k = 0; k < PER; ++k) o += sums[k][tid];
            a.out[((size_t)(a.seq_row ? a.seq_row[b] : b) * a.nH + g * G + own) * SP_HD + tid] = __float2bfloat16_rn(inv == INFINITY ? 0.f : o * inv);
        }
        return;
    }
    float given[SP_JOIN_KEYS];
    int page[SP_JOIN_KEYS];
#pragma unroll
    for (int u = 0; u < SP_JOIN_KEYS; ++u) {
        const int j = j0 + u * SP_JOIN_THREADS;
        given[u] = 0.f;
        page[u] = !GIVEN && j < most ? a.pages[(size_t)b * a.max_pages + j / GL_PAGE] : 0;
    }
    const float* sc = a.scores + ((size_t)b * a.nH + g * G) * a.reach + j0;
#pragma unroll 4
    for (int i = 0; i < G; ++i) {
        const float m = ml_all[2 * i], inv = ml_all[2 * i + 1];
#pragma unroll
        for (int u = 0; u < SP_JOIN_KEYS; ++u) {
            const float x = j0 + u * SP_JOIN_THREADS < most ? sc[(size_t)i * a.reach + u * SP_JOIN_THREADS] : 0.f;
            given[u] = fmaf(sp_exp2(fmaf(x, SP_LOG2E, -m)), inv, given[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < SP_JOIN_KEYS; ++u) {
        const int j = j0 + u * SP_JOIN_THREADS;
        if (j >= most) return;
        float* w = GIVEN ? a.given + ((size_t)b * a.nKV + g) * a.reach + j
                         : a.weights + ((size_t)gl_checked(page[u], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + j % GL_PAGE;
        if (!GIVEN && j < pos) atomicAdd(w, given[u]);     // (one addition a position: no two sequences share it)
        else *w = given[u];
    }
}


// ---------------------------------------------------------------------------
// One or two query heads on a key/value head, larger than 64: a sequence's own pages go from the cache straight to registers, as in
// attention_spans_f32.cu.  Eight lanes take a key, a warp four keys at a time with 2 UN of their rows under way; no barrier stands between
// two keys, and the weights stay in 32 bits.  Eight columns of a tensor-core product would be empty but for one or two.  Bound by the
// latency of its loads, four blocks an SM being what the registers hold: eight sequences of 300 to 2,047 positions, 32 heads of 80,
// with weights: 30 us, 3.3 TB/s.
// ---------------------------------------------------------------------------
#define SW_CP ((SP_CHUNKS + 7) / 8)       // 16-byte pieces of a row that a lane takes
#define SW_WARPS 4
// eight bfloat16 numbers times eight others, added to x
__device__ __forceinline__ float sw_dot(const uint4& k, const float (&q)[8], float x) {
    const unsigned w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x = fmaf(__uint_as_float(w[i] << 16), q[2 * i], fmaf(__uint_as_float(w[i] & 0xffff0000u), q[2 * i + 1], x));
    return x;
}
__device__ __forceinline__ void sw_add(const uint4& v, float w, float (&o)[8]) {
    const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[2 * i] = fmaf(w, __uint_as_float(u[i] << 16), o[2 * i]);
        o[2 * i + 1] = fmaf(w, __uint_as_float(u[i] & 0xffff0000u), o[2 * i + 1]);
    }
}
template <int R>
__host__ __device__ constexpr size_t sw_smem() { return sizeof(float) * (SW_WARPS + 1) * R * (SP_HD + 2); }

template <int R, int MODE>
__global__ void __launch_bounds__(32 * SW_WARPS)
stream_span_kernel(SpanArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int UN = SW_CP * R <= 2 ? 4 : 2, RUN = 4 * UN;       // keys of a group of lanes, and of a warp, under way
    float* o_w = (float*)smem;                                     // [4][R][hd] what the warps found, [4][R][2]; the block's result [R][hd], [R][2]
    float* ml_w = o_w + SW_WARPS * R * SP_HD;
    float* fin_o = ml_w + SW_WARPS * R * 2;
    float* fin_ml = fin_o + R * SP_HD;
    float* held = fin_ml + 2 * R;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane & 7, grp = lane >> 3;
    if (!a.early) gl_grid_wait();
    gl_grid_launch_dependents();
    const int b = blockIdx.z, g = blockIdx.y;
    if (a.seq_qlen && a.seq_qlen[b] <= 0) return;
    const int pos = a.seq_ctx[b], total = pos + 1, first = a.seq_shared ? a.seq_shared[2 * b] : 0;
    const int n = max(0, pos / GL_PAGE + 1 - first), per = (n + a.splits - 1) / a.splits;
    const int p_begin = first + (int)blockIdx.x * per, p_end = min(first + n, p_begin + per);
    const int n_pre = a.seq_shared ? a.seq_shared[2 * b + 1] : 0, slot = n_pre + blockIdx.x;
    const int* pg = a.pages + (size_t)b * a.max_pages;
    const size_t q_row = (size_t)(a.seq_row ? a.seq_row[b] : b) * a.nH + g * R;
    float q[R][SW_CP][8], o[R][SW_CP][8];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < SW_CP; ++c) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (c * 8 + sub < SP_CHUNKS) v = *(const uint4*)(a.q + (q_row + r) * SP_HD + 8 * (c * 8 + sub));
            const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                q[r][c][2 * i] = __uint_as_float(w[i] << 16) * SP_LOG2E;      // (scores as powers of two)
                q[r][c][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * SP_LOG2E;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) o[r][c][i] = 0.f;
        }
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) { m[r] = -INFINITY; l[r] = 0.f; }
    const int k_end = min(p_end * GL_PAGE, total);
    for (int j0 = p_begin * GL_PAGE + warp * RUN; j0 < k_end; j0 += SW_WARPS * RUN) {
        const size_t at = (((size_t)gl_checked(pg[j0 / GL_PAGE], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + j0 % GL_PAGE + grp) * SP_HD + 8 * sub;
        uint4 k[UN][SW_CP], v[UN][SW_CP];
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int c = 0; c < SW_CP; ++c) {
                const bool ok = j0 + 4 * u + grp < k_end && c * 8 + sub < SP_CHUNKS;
                k[u][c] = ok ? *(const uint4*)(a.k_cache + at + 4 * u * SP_HD + 64 * c) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int c = 0; c < SW_CP; ++c) {
                const bool ok = j0 + 4 * u + grp < k_end && c * 8 + sub < SP_CHUNKS;
                v[u][c] = ok ? *(const uint4*)(a.v_cache + at + 4 * u * SP_HD + 64 * c) : make_uint4(0, 0, 0, 0);
            }
        float s[R][UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int j = j0 + 4 * u + grp;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float x = 0.f;
#pragma unroll
                for (int c = 0; c < SW_CP; ++c) x = sw_dot(k[u][c], q[r][c], x);
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                if (a.weights && sub == r && j < k_end) {
                    if (MODE == SP_JOIN) { if (j - p_begin * GL_PAGE < a.held) held[r * a.held + j - p_begin * GL_PAGE] = x; }
                    else if (j < a.reach) a.scores[((size_t)b * a.nH + g * R + r) * a.reach + j] = x / SP_LOG2E;
                }
                s[r][u] = j < k_end ? x : -INFINITY;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float m_new = m[r];
#pragma unroll
            for (int u = 0; u < UN; ++u) m_new = fmaxf(m_new, s[r][u]);
            const float mu = m_new == -INFINITY ? 0.f : m_new, corr = sp_factor(m[r], m_new);
            if (__any_sync(0xffffffffu, m[r] != m_new)) {
                l[r] *= corr;
#pragma unroll
                for (int c = 0; c < SW_CP; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[r][c][i] *= corr;
            }
            m[r] = m_new;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const float w = sp_exp2(s[r][u] - mu);
                l[r] += w;
#pragma unroll
                for (int c = 0; c < SW_CP; ++c) sw_add(v[u][c], w, o[r][c]);
            }
        }
    }
    // the warp's four groups of lanes, then the warps
#pragma unroll
    for (int x = 8; x < 32; x <<= 1)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float om = __shfl_xor_sync(0xffffffffu, m[r], x), ol = __shfl_xor_sync(0xffffffffu, l[r], x), m_new = fmaxf(m[r], om);
            const float f = sp_factor(m[r], m_new), of = sp_factor(om, m_new);
            l[r] = l[r] * f + ol * of;
            m[r] = m_new;
#pragma unroll
            for (int c = 0; c < SW_CP; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) o[r][c][i] = o[r][c][i] * f + __shfl_xor_sync(0xffffffffu, o[r][c][i], x) * of;
        }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (lane == 0) *(float2*)(ml_w + (warp * R + r) * 2) = make_float2(m[r], l[r]);
        if (grp == 0)
#pragma unroll
            for (int c = 0; c < SW_CP; ++c)
                if (c * 8 + sub < SP_CHUNKS) {
                    float4* dst = (float4*)(o_w + (warp * R + r) * SP_HD + 8 * (c * 8 + sub));
                    dst[0] = make_float4(o[r][c][0], o[r][c][1], o[r][c][2], o[r][c][3]);
                    dst[1] = make_float4(o[r][c][4], o[r][c][5], o[r][c][6], o[r][c][7]);
                }
    }
    __syncthreads();
    for (int i = tid; i < R * (SP_HD / 4); i += 32 * SW_WARPS) {
        const int r = i / (SP_HD / 4), c = i - r * (SP_HD / 4);
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < SW_WARPS; ++w) mm = fmaxf(mm, ml_w[(w * R + r) * 2]);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < SW_WARPS; ++w) {
            const float f = sp_factor(ml_w[(w * R + r) * 2], mm);
            const float4 x = *(const float4*)(o_w + (w * R + r) * SP_HD + 4 * c);
            sum.x = fmaf(f, x.x, sum.x); sum.y = fmaf(f, x.y, sum.y); sum.z = fmaf(f, x.z, sum.z); sum.w = fmaf(f, x.w, sum.w);
            ll = fmaf(f, ml_w[(w * R + r) * 2 + 1], ll);
        }
        const size_t at = ((size_t)b * a.nH + g * R + r) * a.slots + slot;
        *(float4*)(MODE == SP_JOIN ? fin_o + 4 * i : a.part_o + at * SP_HD + 4 * c) = sum;
        if (c == 0) *(float2*)(MODE == SP_JOIN ? fin_ml + 2 * r : a.part_ml + at * 2) = make_float2(mm, ll);
    }
    if (MODE != SP_JOIN) return;
    const SpanEnd e = {b, g, g * R, R, p_begin, p_end, total};
    span_join(a, e, fin_o, fin_ml, held, ml_w, pg, 1.0f);
}

#define SP_HELD_BYTES (56 * 1024)                  // scores a block keeps in shared memory at most
#define SP_FACTOR_BYTES (24 * 1024)                // factors of the parts of its rows

template <int NT, int MODE, int STAGES = 2>
static int launch_span(const SpanArgs& a, dim3 grid, int cluster, cudaStream_t stream) {
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    const size_t most = sp_smem<NT, STAGES>() + (MODE == SP_JOIN ? SP_HELD_BYTES + SP_FACTOR_BYTES : 0);
    if (!allowed[dev]) {
        if (cudaFuncSetAttribute(attn_span_kernel<NT, MODE, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess) {
            cudaGetLastError();
            return GL_ERR_SMEM;
        }
        allowed[dev] = true;
    }
    const size_t smem = sp_smem<NT, STAGES>() + (MODE == SP_JOIN ? sizeof(float) * ((a.weights ? (size_t)a.held * (a.nH / a.nKV) : 0) + 8 * NT * (size_t)(a.slots + a.splits)) : 0);
    if (smem > most) return GL_ERR_SMEM;
    return gl_launch(attn_span_kernel<NT, MODE, STAGES>, grid, dim3(SP_THREADS), smem, stream, cluster, a);
}

template <int R, int MODE>
static int launch_stream(const SpanArgs& a, dim3 grid, int cluster, cudaStream_t stream) {
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    if (!allowed[dev]) {
        if (cudaFuncSetAttribute(stream_span_kernel<R, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sw_smem<R>() + SP_HELD_BYTES + SP_FACTOR_BYTES)) != cudaSuccess) {
            cudaGetLastError();
            return GL_ERR_SMEM;
        }
        allowed[dev] = true;
    }
    const size_t smem = sw_smem<R>() + (MODE == SP_JOIN ? sizeof(float) * ((a.weights ? (size_t)a.held * R : 0) + R * (size_t)(a.slots + a.splits)) : 0);
    return gl_launch(stream_span_kernel<R, MODE>, grid, dim3(32 * SW_WARPS), smem, stream, cluster, a);
}

template <int MODE>
static int launch_spans(const SpanArgs& a, int rows, dim3 grid, int cluster, cudaStream_t stream) {
    // One or two rows a block: the products on CUDA cores, where a row of the cache is long enough that the tensor cores' eight columns,
    // most of them empty, cost more than the sums over eight lanes.  us, streamed against tensor cores, 8 sequences of 300 to 2,047
    // positions, 16 query heads, with weights: one row, heads of 32: 13.0 / 12.3, of 64: 19.0 / 16.6, of 128: 21.1 / 28.5, of
    // 256: 39.5 / 60.9; two rows, of 64: 11.3 / 11.0, of 128: 17.2 / 21.5, of 256: 33.8 / 52.7.
    if constexpr (MODE != SP_ITEM && SP_HD > 64) {
        if (a.nH == a.nKV) return launch_stream<1, MODE>(a, grid, cluster, stream);
        if (a.nH == 2 * a.nKV) return launch_stream<2, MODE>(a, grid, cluster, stream);
    }
    // Pages in flight: two; one, and more blocks an SM, where a block has one page or two to walk (behind shared pages: 1,024 blocks
    // of a page each, heads of 128: 5 us less).
    if constexpr (MODE == SP_JOIN)
        if (rows <= 8 && a.short_spans) return launch_span<1, MODE, 1>(a, grid, cluster, stream);
    if (rows <= 8) return launch_span<1, MODE>(a, grid, cluster, stream);
    if (rows <= 16) return launch_span<2, MODE>(a, grid, cluster, stream);
    return launch_span<SP_MAX_NT, MODE>(a, grid, cluster, stream);
}

static int span_checked(const SpanArgs& a) {
    if (a.nH <= 0 || a.nKV <= 0 || a.nH % a.nKV || a.B > 65535 || a.splits < 1 || a.slots < 0 || a.max_pages <= 0) return GL_ERR_SHAPE;
    const int G = a.nH / a.nKV;
    if (a.chunks < 1 || a.chunks > G || (long long)a.nKV * a.chunks > 65535 || (G + a.chunks - 1) / a.chunks > 8 * SP_MAX_NT) return GL_ERR_SHAPE;
    if ((a.chunks - 1) * ((G + a.chunks - 1) / a.chunks) >= G) return GL_ERR_SHAPE;        // every share of the heads has one
    if (((uintptr_t)a.q | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15 || (uintptr_t)a.out & 7) return GL_ERR_ALIGN;      // (results leave in pieces of 8 bytes)
    return a.slots > 0 && (!a.part_o || !a.part_ml) ? GL_ERR_SHAPE : GL_OK;
}

static int launch_join(const SpanArgs& a, cudaStream_t stream) {
    const int G = a.nH / a.nKV;
    const int shares = a.weights ? (a.reach + SP_JOIN_KEYS * SP_JOIN_THREADS - 1) / (SP_JOIN_KEYS * SP_JOIN_THREADS) : 0;
    const dim3 grid(shares + G, a.nKV, a.B);
    if (a.given) return gl_launch(attn_span_join_kernel<true>, grid, dim3(SP_JOIN_THREADS), 2 * G * sizeof(float), stream, 1, a, shares);
    return gl_launch(attn_span_join_kernel<false>, grid, dim3(SP_JOIN_THREADS), 2 * G * sizeof(float), stream, 1, a, shares);
}

static int shared_tc(const SpanArgs& a, int rows, cudaStream_t stream);

// rows: the most that one of the plan's items has; joined: a sequence's splits are a cluster that joins its results and the shared
// pages' itself (part_o and part_ml have slots for the shared pages alone), else a second kernel does (and they have the splits' too)
GL_API int gl_attention_prefix(const SpanArgs* args, int rows, int joined, cudaStream_t stream) {
    SpanArgs a = *args;
    if (a.B <= 0) return GL_OK;
    int rc = span_checked(a);
    if (rc != GL_OK) return rc;
    if (a.n_items < 0 || a.scores || a.weights || !a.seq_shared || (a.n_items > 0 && (!a.items || !a.order || rows < 1 || a.slots < 1))) return GL_ERR_SHAPE;
    if (joined ? a.splits > 8 || 8 * SP_MAX_NT * (long long)(a.slots + a.splits) * (int)sizeof(float) > SP_FACTOR_BYTES : a.slots < a.splits) return GL_ERR_SHAPE;
    const int G = a.nH / a.nKV;
    a.early = a.held = 0;
    if (a.n_items > 0) {
        rc = rows > 8 * SP_MAX_NT ? shared_tc(a, rows, stream) : launch_spans<SP_ITEM>(a, rows, dim3(a.n_items, a.nKV), 1, stream);
        if (rc != GL_OK) return rc;
        a.early = joined && gl_pdl;
    }
    const dim3 grid(a.splits, a.nKV * a.chunks, a.B);
    if (joined) return launch_spans<SP_JOIN>(a, (G + a.chunks - 1) / a.chunks, grid, a.splits, stream);
    if ((rc = launch_spans<SP_SPLIT>(a, (G + a.chunks - 1) / a.chunks, grid, 1, stream)) != GL_OK) return rc;
    return launch_join(a, stream);
}

// Without ``scores`` the splits are a cluster that joins its results and keeps its scores in shared memory, else a second kernel
// joins the splits' partial results and reads the scores back.
GL_API int gl_attention_weighed(const SpanArgs* args, cudaStream_t stream) {
    SpanArgs a = *args;
    if (a.B <= 0) return GL_OK;
    int rc = span_checked(a);
    if (rc != GL_OK) return rc;
    if (!a.weights || a.seq_shared || a.reach <= 0) return GL_ERR_SHAPE;
    const int G = a.nH / a.nKV;
    const dim3 grid(a.splits, a.nKV * a.chunks, a.B);
    a.early = a.held = 0;
    if (!a.scores) {
        // (a pitch of 4 more than whole pages: the eight keys of four rows that a warp stores lie in different banks)
        a.held = ((a.reach + GL_PAGE - 1) / GL_PAGE + a.splits - 1) / a.splits * GL_PAGE + 4;
        if (a.chunks > 1 || a.splits > 8 || a.slots > 0 || (long long)a.held * G * (int)sizeof(float) > SP_HELD_BYTES) return GL_ERR_SHAPE;
        rc = launch_spans<SP_JOIN>(a, G, grid, a.splits, stream);
    } else {
        if (a.slots < a.splits) return GL_ERR_SHAPE;
        if ((rc = launch_spans<SP_SPLIT>(a, (G + a.chunks - 1) / a.chunks, grid, 1, stream)) != GL_OK) return rc;
        rc = launch_join(a, stream);
    }
    return rc != GL_OK || !a.given ? rc : launch_given_join(a, a.given, 1, 1, stream);
}

// ---------------------------------------------------------------------------
// Shared pages with many rows, on the 5th-generation tensor cores: the same partial results as attn_span_kernel<SP_ITEM>.
//
// A block takes 128 or 256 rows of an item (members x query heads, whatever their places in q) as one or two tiles and walks
// the item's pages.  One warp feeds key and value pages by TMA through a ring; each tile has a thread of its own that issues
// tcgen05.mma: scores S = Q K^T (M 128, N 64) into one of two buffers in tensor memory, two pages ahead of the rows, and O += P V
// (M 128, N = head size, the weights read from tensor memory where their scores were, the values MN-major as the cache holds
// them).  Four warps a tile own a row a thread: no shuffles for the sum, and a maximum only where a page needs one.  All
// pages are seen whole, so there is no mask but for a caller whose sequences end inside.
// Bound by the issue of the products (12 a page of 64 keys at a head size of 128) beside the powers, and by memory where one tile holds
// all rows.  32 heads of 128 on 8: 128 sequences on one document of 16,384 tokens, 46 us, 0.75 PFLOP/s, a page of two tiles some 1,850 clocks, of
// which the powers need 1,024; 64 sequences on four texts of 8,192, 24 us.  Scores of two pages at once (N 128) leave no room in tensor
// memory for a second buffer and took 6 us more in all.  Waits are bounded; a block whose wait runs out records it, frees its tensor memory and returns.
// ---------------------------------------------------------------------------
#if SP_HD <= 128
#define ST_BM 128
#define ST_THREADS(NT) ((NT) * 160 + 32)
#define ST_TMEM_COLS(NT) (256 * (NT))
// pieces of the head size for queries and keys: widths 64, 64, 32, 16 as far as they fit
struct StSeg { int off, width; };
__host__ __device__ constexpr int st_nseg() { return (SP_HD / 64) + ((SP_HD % 64) >= 32 ? 1 : 0) + ((SP_HD % 32) >= 16 ? 1 : 0); }
__host__ __device__ constexpr StSeg st_seg(int i) {
    int off = 0, idx = 0;
    for (int k = 0; k < SP_HD / 64; ++k) { if (idx == i) return StSeg{off, 64}; off += 64; ++idx; }
    if ((SP_HD % 64) >= 32) { if (idx == i) return StSeg{off, 32}; off += 32; ++idx; }
    if ((SP_HD % 32) >= 16) { if (idx == i) return StSeg{off, 16}; off += 16; ++idx; }
    return StSeg{0, 0};
}
__host__ __device__ constexpr int st_seg_base(int i, int rows) {
    int b = 0;
    for (int k = 0; k < i; ++k) b += ((rows * st_seg(k).width * 2 + 1023) / 1024) * 1024;
    return b;
}
#define ST_NSEG st_nseg()
#define ST_Q_BYTES st_seg_base(ST_NSEG, ST_BM)
#define ST_K_BYTES st_seg_base(ST_NSEG, GL_PAGE)
#define ST_VATOMS ((SP_HD + 63) / 64)
#define ST_VATOM_BYTES (GL_PAGE * 128)
#define ST_V_BYTES (ST_VATOMS * ST_VATOM_BYTES)
// pages in flight: with one tile no more than leaves room on the SM for a block that walks own pages beside it
__host__ __device__ constexpr int st_stages(int nt) {
    const int n = ((nt == 2 ? 224 * 1024 : 144 * 1024) - nt * ST_Q_BYTES) / (ST_K_BYTES + ST_V_BYTES);
    return n > 8 ? 8 : n;
}
static_assert(st_stages(2) >= 3 && st_stages(1) >= 3, "shared memory holds too few pages");
struct StMaps { CUtensorMap k[4], v; };

// the one lane of a whole warp that issues: the same one every time
__device__ __forceinline__ bool elect_one() {
    unsigned p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}

template <int NT>
__global__ void __launch_bounds__(ST_THREADS(NT), 1)
shared_tc_kernel(SpanArgs a, const __grid_constant__ StMaps maps) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ unsigned tmem_slot;
    __shared__ volatile int failed;
    unsigned char* smem = smem_raw + ((1024u - (gl_smem_u32(smem_raw) & 1023u)) & 1023u);
    constexpr int STAGES = st_stages(NT), PRODUCER = 4 * NT;
    const unsigned base = gl_smem_u32(smem);
    const unsigned sQ = base, sK = sQ + NT * ST_Q_BYTES, sV = sK + STAGES * ST_K_BYTES, bars = sV + STAGES * ST_V_BYTES;
    const unsigned bar_f = bars, bar_e = bar_f + 8 * STAGES;       // a page's keys and values are there; are done with
    const unsigned bar_t = bar_e + 8 * STAGES;             // per tile: scores full [2], weights full [2], last product but one done, output full, queries there
#define ST_SF(t, i) (bar_t + 64 * (t) + 8 * (i))
#define ST_PF(t, i) (bar_t + 64 * (t) + 16 + 8 * (i))
#define ST_PD(t) (bar_t + 64 * (t) + 32)
#define ST_OF(t) (bar_t + 64 * (t) + 40)
#define ST_QF(t) (bar_t + 64 * (t) + 48)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(bar_f + 8 * s, 1); mbar_init(bar_e + 8 * s, NT); }
        for (int t = 0; t < NT; ++t) {
            for (int i = 0; i < 2; ++i) { mbar_init(ST_SF(t, i), 1); mbar_init(ST_PF(t, i), 4); }
            mbar_init(ST_PD(t), 1); mbar_init(ST_OF(t), 1); mbar_init(ST_QF(t), 4);
        }
        mbar_fence_init();
    }
    if (warp == PRODUCER) tmem_alloc(gl_smem_u32(&tmem_slot), ST_TMEM_COLS(NT));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_slot;
    gl_grid_wait();                                        // (then the next kernel may start: all before both is complete)
    gl_grid_launch_dependents();

    const int* it = a.items + 6 * blockIdx.x;
    const int g = blockIdx.y, first = it[1], rows_all = it[2], p_begin = it[3], n = it[4] - it[3], slot = it[5];
    const int* members = a.order + it[0];
    const int G = a.nH / a.nKV;
    // tile t: score buffers at columns 256 t and 256 t + 64 (a page's weights overwrite the first 32 columns of its scores, two a
    // column), output at 256 t + 128.  A second tile without rows takes no part.
    const int tiles = rows_all > ST_BM ? 2 : 1;
    int issued = 0;

    if (warp == PRODUCER) {
        if (lane == 0) {
            const int* pg = a.pages + (size_t)members[0] * a.max_pages + p_begin;
            for (int j = 0; j < n && !failed; ++j) {
                const int st = j % STAGES;
                const unsigned par = ((j / STAGES) - 1) & 1;
                const int row = (gl_checked(pg[j], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE;
                if (j >= STAGES && !mbar_wait(bar_e + 8 * st, par)) { failed = 1; break; }
                mbar_expect_tx(bar_f + 8 * st, GL_PAGE * SP_HD * 2 + ST_V_BYTES);       // zero fill counts
#pragma unroll
                for (int s = 0; s < ST_NSEG; ++s)
                    tma_load_2d(sK + st * ST_K_BYTES + st_seg_base(s, GL_PAGE), &maps.k[s], st_seg(s).off, row, bar_f + 8 * st);
#pragma unroll
                for (int c = 0; c < ST_VATOMS; ++c)
                    tma_load_2d(sV + st * ST_V_BYTES + c * ST_VATOM_BYTES, &maps.v, 64 * c, row, bar_f + 8 * st);
                issued = j + 1;
            }
        }
    } else if (warp > PRODUCER) {
        // (the whole warp goes through the waits and addresses, which are the same for all its lanes, and one lane issues: where one lane
        // went through all of it alone, 128 sequences on a document of 16,384 tokens took 55 us against 52)
        constexpr uint32_t idesc_s = umma_idesc_bf16(GL_PAGE, 0);
        constexpr uint32_t idesc_o = umma_idesc_bf16(SP_HD, 1);
        const int t = warp - PRODUCER - 1, nt = t < tiles ? n : 0;
        auto wait = [](unsigned bar, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };
        auto issue_scores = [&](int j) {
            const int st = j % STAGES;
            bool begin = true;
            if (elect_one()) {
#pragma unroll
                for (int s = 0; s < ST_NSEG; ++s) {
                    const int rb = st_seg(s).width * 2;
                    const uint64_t dq = umma_tile_desc(sQ + t * ST_Q_BYTES + st_seg_base(s, ST_BM), rb);
                    const uint64_t dk = umma_tile_desc(sK + st * ST_K_BYTES + st_seg_base(s, GL_PAGE), rb);
#pragma unroll
                    for (int k = 0; k < st_seg(s).width / 16; ++k) {
                        umma_bf16(tmem + 256 * t + 64 * (j & 1), dq + 2 * k, dk + 2 * k, idesc_s, begin ? 0u : 1u);
                        begin = false;
                    }
                }
                umma_commit(ST_SF(t, j & 1));
            }
            __syncwarp();
        };
        // What this thread does a page is what the kernel waits for, and a wait costs it some 250 clocks even where there is nothing to wait
        // for, a commit 40: so a page's keys and values arrive together (that page's wait was made before its scores), go back
        // together behind the second product, and the products done are announced by the scores behind them (a commit
        // speaks for all that its thread issued before) but for the last product that has none.
        bool ok = nt == 0 || wait(ST_QF(t), 0);
        for (int j = 0; ok && j < 2 && j < nt; ++j) {
            ok = wait(bar_f + 8 * (j % STAGES), (j / STAGES) & 1);
            if (ok) { tc_fence_after(); issue_scores(j); }
        }
        for (int j = 0; ok && j < nt; ++j) {
            const int st = j % STAGES;
            if (NT > 1 && j + 2 < nt) ok = wait(bar_f + 8 * ((j + 2) % STAGES), ((j + 2) / STAGES) & 1);
            ok = ok && wait(ST_PF(t, j & 1), (j >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dv = umma_smem_desc(sV + st * ST_V_BYTES, ST_VATOM_BYTES, 1024, 2);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < GL_PAGE / 16; ++k)
                    umma_bf16_tmem_a(tmem + 256 * t + 128, tmem + 256 * t + 64 * (j & 1) + 8 * k, dv + (uint64_t)((16 * 128) >> 4) * k, idesc_o, (j | k) ? 1u : 0u);
                umma_commit(bar_e + 8 * st);
                if (j == nt - 2) umma_commit(ST_PD(t));
                if (j == nt - 1) umma_commit(ST_OF(t));
            }
            __syncwarp();
            if (j + 2 < nt) {                          // over S_j and P_j, which the rows and the product above are done with
                if (NT == 1) ok = wait(bar_f + 8 * ((j + 2) % STAGES), ((j + 2) / STAGES) & 1);
                if (!ok) break;
                tc_fence_after();
                issue_scores(j + 2);
            }
        }
        // a tile without rows still hands every page back, once it has been loaded
        for (int j = nt; ok && j < n && !__any_sync(0xffffffffu, failed); ++j) {
            const int st = j % STAGES;
            ok = wait(bar_f + 8 * st, (j / STAGES) & 1);
            if (ok && lane == 0) mbar_arrive(bar_e + 8 * st);
        }
        if (!ok) failed = 1;
    } else if ((warp >> 2) < tiles) {
        const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, row = t * ST_BM + r;
        const bool real = row < rows_all;
        const int b = real ? members[(first + row) / G] : -1, h = g * G + (first + row) % G;
        const int last = real ? a.seq_ctx[b] : 0x7fffffff;
        {   // this row's query into the tile, in the order that the products read it (16-byte pieces turned by the row)
            const uint4* src = (const uint4*)(a.q + ((size_t)(real ? b : 0) * a.nH + (real ? h : 0)) * SP_HD);
#pragma unroll
            for (int s = 0; s < ST_NSEG; ++s) {
                const int rb = st_seg(s).width * 2, pieces = rb / 16;
                unsigned char* dst = smem + t * ST_Q_BYTES + st_seg_base(s, ST_BM) + r * rb;
                const int turn = ((r * rb) >> 7) & (pieces - 1);
#pragma unroll
                for (int c = 0; c < pieces; ++c)
                    *(uint4*)(dst + ((c ^ turn) << 4)) = real ? src[st_seg(s).off / 8 + c] : make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(ST_QF(t));
        }
        const unsigned lane_off = (unsigned)(quarter * 32) << 16;
        const unsigned tS = tmem + 256 * t + lane_off, tO = tS + 128;
        float m_run = -INFINITY, l_run = 0.f;              // (the maximum as a power of two, as of the last rescaling)
        bool alive = true;
        for (int j = 0; j < n; ++j) {
            bool ok = mbar_wait(ST_SF(t, j & 1), (j >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) { failed = 1; alive = false; break; }
            tc_fence_after();
            float sc[GL_PAGE];
            {
                unsigned (&su)[GL_PAGE] = reinterpret_cast<unsigned (&)[GL_PAGE]>(sc);
                tmem_ld32_issue(tS + 64 * (j & 1), *reinterpret_cast<unsigned (*)[32]>(&su[0]));
                tmem_ld32_issue(tS + 64 * (j & 1) + 32, *reinterpret_cast<unsigned (*)[32]>(&su[32]));
                tmem_ld_wait();
            }
            const int j0 = (p_begin + j) * GL_PAGE;
            if (j0 + GL_PAGE - 1 > last) {
#pragma unroll
                for (int i = 0; i < GL_PAGE; ++i)
                    if (j0 + i > last) sc[i] = -INFINITY;
            }
            // The powers' reference is a maximum of an earlier page, whichever: what lies above it by less than 2^60 loses nothing, in the
            // weights (bfloat16 has the range of 32 bits) or in the sums (of values below 2^50: 16,384 pages of them stay in range), and takes no
            // search for the maximum.  The first page,
            // and one whose sum says that a score lay higher, is done with its own maximum, the output rescaled.
            float mu = m_run == -INFINITY ? 0.f : m_run, sum;
            unsigned pk[32];
            auto weigh = [&]() {
                float ps4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < GL_PAGE; i += 4) {
                    const float e0 = sp_exp2(fmaf(sc[i], SP_LOG2E, -mu)), e1 = sp_exp2(fmaf(sc[i + 1], SP_LOG2E, -mu));
                    const float e2 = sp_exp2(fmaf(sc[i + 2], SP_LOG2E, -mu)), e3 = sp_exp2(fmaf(sc[i + 3], SP_LOG2E, -mu));
                    ps4[0] += e0; ps4[1] += e1; ps4[2] += e2; ps4[3] += e3;
                    __nv_bfloat162 p0 = __floats2bfloat162_rn(e0, e1), p1 = __floats2bfloat162_rn(e2, e3);
                    pk[i / 2] = *(unsigned*)&p0; pk[i / 2 + 1] = *(unsigned*)&p1;
                }
                sum = (ps4[0] + ps4[1]) + (ps4[2] + ps4[3]);
            };
            weigh();
            if (__any_sync(0xffffffffu, m_run == -INFINITY || !(sum <= 1.152921504606847e18f))) {
                float mx = sc[0];
#pragma unroll
                for (int i = 1; i < GL_PAGE; ++i) mx = fmaxf(mx, sc[i]);
                const float m_new = fmaxf(m_run, mx * SP_LOG2E), corr = sp_factor(m_run, m_new);
                m_run = m_new;
                mu = m_run == -INFINITY ? 0.f : m_run;
                if (j >= 1) {
                    // the products so far are complete: the scores behind them are there, or the last but one is announced
                    ok = j + 1 < n ? mbar_wait(ST_SF(t, (j + 1) & 1), ((j + 1) >> 1) & 1) : mbar_wait(ST_PD(t), 0);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) { failed = 1; alive = false; break; }
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < SP_HD; c += 16) {
                        unsigned t16[16];
                        tmem_ld16(tO + c, t16);
#pragma unroll
                        for (int i = 0; i < 16; ++i) t16[i] = __float_as_uint(__uint_as_float(t16[i]) * corr);
                        tmem_st16(tO + c, t16);
                    }
                }
                l_run *= corr;
                weigh();
            }
            tmem_st32(tS + 64 * (j & 1), pk);
            l_run += sum;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ST_PF(t, j & 1));
        }
        if (alive) {
            bool ok = mbar_wait(ST_OF(t), 0);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                tc_fence_after();
                const size_t at = ((size_t)(real ? b : 0) * a.nH + h) * a.slots + slot;
#pragma unroll
                for (int c = 0; c < SP_HD; c += 16) {
                    unsigned t16[16];
                    tmem_ld16(tO + c, t16);
                    if (real)                              // (a row a thread: whole 32-byte sectors)
#pragma unroll
                        for (int i = 0; i < 16; i += 8)
                            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(a.part_o + at * SP_HD + c + i), "r"(t16[i]), "r"(t16[i + 1]),
                                         "r"(t16[i + 2]), "r"(t16[i + 3]), "r"(t16[i + 4]), "r"(t16[i + 5]), "r"(t16[i + 6]), "r"(t16[i + 7]) : "memory");
                }
                if (real) { a.part_ml[at * 2] = m_run; a.part_ml[at * 2 + 1] = l_run; }
            } else {
                failed = 1;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == PRODUCER) {
        tc_fence_after();
        tmem_dealloc(tmem, ST_TMEM_COLS(NT));
        if (failed && lane == 0)                           // a wait ran out: nothing is left on its way into this block's memory
            for (int j = max(0, issued - STAGES); j < issued; ++j) (void)mbar_wait(bar_f + 8 * (j % STAGES), (j / STAGES) & 1);
    }
    if (threadIdx.x == 0 && failed) atomicExch(&gl_wait_failed, 1);
}

template <int NT>
static int launch_shared_tc(const SpanArgs& a, const StMaps& maps, cudaStream_t stream) {
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    const size_t smem = NT * (size_t)ST_Q_BYTES + st_stages(NT) * ((size_t)ST_K_BYTES + ST_V_BYTES) + 32 * st_stages(NT) + 64 * NT + 1024;
    if (!allowed[dev]) {
        if (cudaFuncSetAttribute(shared_tc_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
            cudaGetLastError();
            return GL_ERR_SMEM;
        }
        allowed[dev] = true;
    }
    return gl_launch(shared_tc_kernel<NT>, dim3(a.n_items, a.nKV), dim3(ST_THREADS(NT)), smem, stream, 1, a, maps);
}
static int shared_tc(const SpanArgs& a, int rows, cudaStream_t stream) {
    if (rows > 2 * ST_BM) return GL_ERR_SHAPE;
    if ((uintptr_t)a.part_o & 31) return GL_ERR_ALIGN;
    StMaps maps;
    const uint64_t kv_rows = (uint64_t)a.n_pages * a.nKV * GL_PAGE;
    if (kv_rows > 0x7fffffffULL) return GL_ERR_SHAPE;      // (a row's number is a coordinate)
    for (int s = 0; s < ST_NSEG; ++s) {
        const int rc = gl_cached_map(&maps.k[s], a.k_cache, kv_rows, SP_HD, GL_PAGE, st_seg(s).width, 2);
        if (rc != GL_OK) return rc;
    }
    const int rc = gl_cached_map(&maps.v, a.v_cache, kv_rows, SP_HD, GL_PAGE, 64, 2);       // what a box has beyond the head size reads as zero
    if (rc != GL_OK) return rc;
    return rows > ST_BM ? launch_shared_tc<2>(a, maps, stream) : launch_shared_tc<1>(a, maps, stream);
}
#else
static int shared_tc(const SpanArgs&, int, cudaStream_t) { return GL_ERR_SHAPE; }
#endif

// ---------------------------------------------------------------------------
// Runs of several tokens: the weights their positions are given.  The attention itself is the prefill kernels'; what it does
// not leave behind, each row's maximum and sum, is computed here from the scores alone, and a second kernel walks the cache page
// by page: w[j] += sum over the rows that see j of e^(s - m) / l.  Rows are (query, query head of a key/value head), queries
// first.  Both are a chain of mma.sync and one power a score, which bounds them.  No sum depends on the order of the blocks.  These two
// serve heads above 128, whose tiles of 128 rows and keys do not fit beside one another; smaller ones run as the next kernel does.
// ---------------------------------------------------------------------------
struct RunArgs {
    const __nv_bfloat16* q;       // [rows, nH*hd], scaled
    const __nv_bfloat16* k_cache; // [pages, nKV, GL_PAGE, hd]
    const int* seq_row;           // [B] first row of q
    const int* seq_qlen;          // [B]
    const int* seq_ctx;           // [B]
    const int* pages;             // [B, max_pages]
    float* ml;                    // [nH, rows, 2]: maximum, sum
    float* weights;               // [pages, nKV, GL_PAGE]
    float* sums;                  // [parts, B, nKV, reach], where parts > 1 or sequences may hold a page together (shared)
    int B, nH, nKV, max_pages, n_pages, reach, last, parts, rows, shared;
};
#define RW_ROWS 64                                  // rows of q of a tile

// rows [r0, r0 + 64) of a run (queries x heads) to padded rows of shared memory; what lies behind ``end`` is zero
__device__ __forceinline__ void rw_load_rows(unsigned dst, const RunArgs& a, int row0, int g, int G, int r0, int end) {
#pragma unroll
    for (int j = 0; j < SP_KS; ++j) {
        const int i = threadIdx.x + j * SP_THREADS;
        const int r = i / SP_CHUNKS, c = i - r * SP_CHUNKS, row = r0 + r;
        const bool ok = row < end;
        const int tok = ok ? row / G : 0;
        sp_cp16(dst + r * SP_ROW + c * 16, a.q + ((size_t)(row0 + tok) * a.nH + g * G + (ok ? row - tok * G : 0)) * SP_HD + c * 8, ok ? 16 : 0);
    }
}
__device__ __forceinline__ void rw_load_keys(unsigned dst, const RunArgs& a, const int* pg, int p, int g, int total) {
    const size_t at = ((size_t)gl_checked(pg[p], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE * SP_HD;
    sp_load_page(dst, a.k_cache + at, min(GL_PAGE, total - p * GL_PAGE));
}

// blockIdx = (tile of 64 rows from the far end, key/value head, sequence)
__global__ void __launch_bounds__(SP_THREADS)
run_stats_kernel(RunArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    const unsigned sbase = ad_smem(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = lane >> 2, t = lane & 3;
    const int b = blockIdx.z, g = blockIdx.y, G = a.nH / a.nKV;
    gl_grid_launch_dependents();
    gl_grid_wait();
    const int qlen = a.seq_qlen[b], ctx = a.seq_ctx[b], row0 = a.seq_row[b], end = qlen * G;
    const int start = a.last > 0 ? max(0, qlen - a.last) * G : 0;
    const int r0 = start + (int)(gridDim.x - 1 - blockIdx.x) * RW_ROWS;
    if (r0 >= end) return;
    const int* pg = a.pages + (size_t)b * a.max_pages;
    const int n = (ctx + (min(r0 + RW_ROWS, end) - 1) / G) / GL_PAGE + 1;
    rw_load_rows(sbase, a, row0, g, G, r0, end);
    rw_load_keys(sbase + SP_TILE, a, pg, 0, g, ctx + qlen);
    sp_commit();
    unsigned qf[SP_KS][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};        // rows grp and grp + 8 of the warp's 16, this thread's keys only
    const int row_lo = r0 + warp * 16 + grp;
    const int last_lo = ctx + row_lo / G, last_hi = ctx + (row_lo + 8) / G, least = ctx + (r0 + warp * 16) / G;
    for (int p = 0; p < n; ++p) {
        sp_wait<0>();
        __syncthreads();
        if (p + 1 < n) rw_load_keys(sbase + (1 + ((p + 1) & 1)) * SP_TILE, a, pg, p + 1, g, ctx + qlen);
        sp_commit();
        if (p == 0)
#pragma unroll
            for (int kk = 0; kk < SP_KS; ++kk)
                ad_ldm4(sbase + (warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * SP_ROW + (kk * 2 + (lane >> 4)) * 16, qf[kk]);
        const unsigned Ks = sbase + (1 + (p & 1)) * SP_TILE;
        float s[8][4];
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[k][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < SP_KS; ++kk)
#pragma unroll
            for (int k = 0; k < 8; k += 2) {                       // 16 keys: (keys, dims), (keys, dims + 8), (keys + 8, dims), (keys + 8, dims + 8)
                unsigned kf[4];
                ad_ldm4(Ks + (k * 8 + (lane & 7) + (lane >> 4) * 8) * SP_ROW + (kk * 2 + ((lane >> 3) & 1)) * 16, kf);
                ad_mma(s[k], qf[kk], kf[0], kf[1]);
                ad_mma(s[k + 1], qf[kk], kf[2], kf[3]);
            }
        const int j0 = p * GL_PAGE;
        if (j0 + GL_PAGE - 1 > least)
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j0 + k * 8 + 2 * t + (e & 1) > (e < 2 ? last_lo : last_hi)) s[k][e] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float mx = s[0][2 * i];
#pragma unroll
            for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fmaxf(s[k][2 * i], s[k][2 * i + 1]));
            const float m_new = fmaxf(m[i], mx * SP_LOG2E), mu = m_new == -INFINITY ? 0.f : m_new;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += sp_exp2(fmaf(s[k][2 * i], SP_LOG2E, -mu)) + sp_exp2(fmaf(s[k][2 * i + 1], SP_LOG2E, -mu));
            l[i] = fmaf(l[i], sp_factor(m[i], m_new), sum);
            m[i] = m_new;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m[i], x), ol = __shfl_xor_sync(0xffffffffu, l[i], x), m_new = fmaxf(m[i], om);
            l[i] = l[i] * sp_factor(m[i], m_new) + ol * sp_factor(om, m_new);
            m[i] = m_new;
        }
        const int row = row_lo + 8 * i;
        if (t == 0 && row < end) {
            float* ml = a.ml + ((size_t)(g * G + row % G) * a.rows + row0 + row / G) * 2;
            ml[0] = m[i];
            ml[1] = l[i];
        }
    }
}

// blockIdx = (page, key/value head, sequence): the first pages, which most rows see, start first
__global__ void __launch_bounds__(SP_THREADS)
run_weigh_kernel(RunArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    const unsigned sbase = ad_smem(smem);
    float* stat = (float*)(smem + 3 * SP_TILE);                     // [2][64][2] maximum, 1 / sum
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = lane >> 2, t = lane & 3;
    const int b = blockIdx.z, g = blockIdx.y, p = blockIdx.x, G = a.nH / a.nKV;
    gl_grid_launch_dependents();
    gl_grid_wait();
    const int qlen = a.seq_qlen[b], ctx = a.seq_ctx[b], row0 = a.seq_row[b], end = qlen * G, total = ctx + qlen;
    if (qlen <= 0 || p * GL_PAGE >= total) return;
    const int* pg = a.pages + (size_t)b * a.max_pages;
    const int start = max(max(0, p * GL_PAGE - ctx), a.last > 0 ? qlen - a.last : 0) * G;
    const int n = (end - start + RW_ROWS - 1) / RW_ROWS;
    auto load = [&](int i) {
        const int r0 = start + i * RW_ROWS;
        rw_load_rows(sbase + (1 + (i & 1)) * SP_TILE, a, row0, g, G, r0, end);
        if (tid < RW_ROWS) {
            const int row = r0 + tid;
            float2 ml = make_float2(0.f, 1.f);
            if (row < end) ml = *(const float2*)(a.ml + ((size_t)(g * G + row % G) * a.rows + row0 + row / G) * 2);
            stat[(i & 1) * 2 * RW_ROWS + 2 * tid] = ml.x;
            stat[(i & 1) * 2 * RW_ROWS + 2 * tid + 1] = 1.0f / ml.y;
        }
    };
    rw_load_keys(sbase, a, pg, p, g, total);
    if (n > 0) load(0);
    sp_commit();
    unsigned kf[SP_KS][4];
    float given[2] = {0.f, 0.f};
    const int j_lo = p * GL_PAGE + warp * 16 + grp;                 // this thread's keys: j_lo and j_lo + 8
    for (int i = 0; i < n; ++i) {
        sp_wait<0>();
        __syncthreads();
        if (i + 1 < n) load(i + 1);
        sp_commit();
        if (i == 0)
#pragma unroll
            for (int kk = 0; kk < SP_KS; ++kk)
                ad_ldm4(sbase + (warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * SP_ROW + (kk * 2 + (lane >> 4)) * 16, kf[kk]);
        const unsigned Qs = sbase + (1 + (i & 1)) * SP_TILE;
        const float* st = stat + (i & 1) * 2 * RW_ROWS;
        float s[8][4];
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[k][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < SP_KS; ++kk)
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                unsigned qf[4];
                ad_ldm4(Qs + (k * 8 + (lane & 7) + (lane >> 4) * 8) * SP_ROW + (kk * 2 + ((lane >> 3) & 1)) * 16, qf);
                ad_mma(s[k], kf[kk], qf[0], qf[1]);
                ad_mma(s[k + 1], kf[kk], qf[2], qf[3]);
            }
        const int r0 = start + i * RW_ROWS;
        const bool cut = p * GL_PAGE + GL_PAGE - 1 > ctx + r0 / G || r0 + RW_ROWS > end;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float4 c = *(const float4*)(st + 2 * (k * 8 + 2 * t));          // two rows: maximum, 1 / sum
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float w = sp_exp2(fmaf(s[k][e], SP_LOG2E, -(e & 1 ? c.z : c.x))) * (e & 1 ? c.w : c.y);
                if (cut) {
                    const int row = r0 + k * 8 + 2 * t + (e & 1);
                    if (row >= end || j_lo + (e >> 1) * 8 > ctx + row / G) w = 0.f;
                }
                given[e >> 1] += w;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        given[i] += __shfl_xor_sync(0xffffffffu, given[i], 1);
        given[i] += __shfl_xor_sync(0xffffffffu, given[i], 2);
        const int j = j_lo + 8 * i;
        if (t == 0 && j < total) {
            float* w = a.weights + ((size_t)gl_checked(pg[p], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + (j % GL_PAGE);
            if (!a.sums) *w = j < ctx ? *w + given[i] : given[i];
            else if (j < a.reach) a.sums[((size_t)b * a.nKV + g) * a.reach + j] = given[i];
        }
    }
    sp_wait<0>();
}

// The same on the 5th-generation tensor cores, for heads of up to 128: a block has 128 keys (two pages) and walks the run's queries
// 128 at a time, head by head of the key/value head; S = Q K^T (M 128, N 128) goes to one of two buffers in tensor memory.  A thread
// owns a row, whose statistics it holds in registers, and a quarter of the keys, whose sums over its rows it holds in 32 more: per score
// one FMA, one power, one FMA, and no shared memory (with a key a thread the queries' statistics come from shared memory, which
// takes as long as the powers).  At the end the 128 rows' sums are added up in a fixed order.  2,048 tokens, 32 heads of 80: 36 us, of
// which the powers (16 a clock and SM) need 17; the rest is what a warp does between two tiles.  Where there are few keys and heads the queries are shared
// out among ``parts`` blocks, whose sums a last kernel adds up in order.  Waits are bounded, as above.
#if SP_HD <= 128
#define RT_WARPS 16                       // four times four warps of rows, each four with a quarter of the keys
#define RT_COLS 32
#define RT_THREADS (32 * RT_WARPS + 64)   // and one that feeds shared memory, one that issues
#define RT_TILE_BYTES ST_Q_BYTES          // 128 rows of keys, or of queries
__host__ __device__ constexpr int rt_stages() { return 200 * 1024 / RT_TILE_BYTES - 2 > 6 ? 6 : 200 * 1024 / RT_TILE_BYTES - 2; }
static_assert(rt_stages() >= 3, "shared memory holds too few queries");
struct RtMaps { CUtensorMap q[4], k[4]; };

// The sum over a warp's lanes of v[i]: lane l ends with that of column l.
__device__ __forceinline__ float rt_sum_lanes(float (&v)[RT_COLS], int lane) {
#pragma unroll
    for (int n = 16; n >= 1; n >>= 1) {                    // a lane keeps half of its columns and takes its partner's share of them
        const bool up = lane & n;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < n) {
                const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, give, n);
            }
    }
    return v[0];
}

// An item is a block of 128 keys of a key/value head and a share of the queries that see them.
struct RtItem { int g, b, k0, part, qlen, ctx, row0, start, n_q, t0, n; };
__device__ __forceinline__ RtItem rt_item(const RunArgs& a, int i) {
    RtItem x;
    const int G = a.nH / a.nKV;
    x.g = i % a.nKV; i /= a.nKV;
    x.b = i % a.B; i /= a.B;
    x.part = i % a.parts;
    x.k0 = i / a.parts * ST_BM;
    x.qlen = a.seq_qlen[x.b]; x.ctx = a.seq_ctx[x.b]; x.row0 = a.seq_row[x.b];
    x.start = max(max(0, x.k0 - x.ctx), a.last > 0 ? x.qlen - a.last : 0);
    x.n_q = (x.qlen - x.start + ST_BM - 1) / ST_BM;
    const int all = x.n_q > 0 && x.k0 < x.ctx + x.qlen ? x.n_q * G : 0;
    // its tiles: head by head, queries rising
    x.t0 = (int)((long long)all * x.part / a.parts);
    x.n = (int)((long long)all * (x.part + 1) / a.parts) - x.t0;
    return x;
}

// A block an SM takes items in turn.  The items are numbered with the keys' positions as the slowest index, so those that most
// queries see come first, and dealt out forwards and backwards in turn, which evens their sums out; while the rows add up
// one item's sums, the next one's keys and scores are under way.
__global__ void __launch_bounds__(RT_THREADS, 1)
run_weigh_tc_kernel(RunArgs a, int n_items, const __grid_constant__ RtMaps maps) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ unsigned tmem_slot;
    __shared__ volatile int failed;
    __shared__ __align__(8) float sums[2][RT_WARPS][RT_COLS];
    unsigned char* smem = smem_raw + ((1024u - (gl_smem_u32(smem_raw) & 1023u)) & 1023u);
    constexpr int STAGES = rt_stages(), PRODUCER = RT_WARPS;
    const unsigned sK = gl_smem_u32(smem), sQ = sK + 2 * RT_TILE_BYTES, bars = sQ + STAGES * RT_TILE_BYTES;
    const unsigned bar_kf = bars, bar_ke = bars + 16, bar_sf = bars + 32, bar_se = bars + 48, bar_qf = bars + 64, bar_qe = bar_qf + 8 * STAGES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(bar_qf + 8 * s, 1); mbar_init(bar_qe + 8 * s, 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(bar_kf + 8 * s, 1); mbar_init(bar_ke + 8 * s, 1); mbar_init(bar_sf + 8 * s, 1); mbar_init(bar_se + 8 * s, RT_WARPS); }
        mbar_fence_init();
    }
    if (warp == PRODUCER) tmem_alloc(gl_smem_u32(&tmem_slot), 256);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_slot;
    gl_grid_wait();
    gl_grid_launch_dependents();
    const int G = a.nH / a.nKV;
    auto item_of = [&](int round) { return round * (int)gridDim.x + (round & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x); };
    const int rounds = (n_items + gridDim.x - 1) / gridDim.x;
    int j = 0, k = 0;                                      // tiles and items so far

    if (warp == PRODUCER) {
        if (lane == 0) {
            bool ok = true;
            for (int round = 0; round < rounds && ok && !failed; ++round) {
                if (item_of(round) >= n_items) continue;
                const RtItem x = rt_item(a, item_of(round));
                if (x.n == 0) continue;
                const int* pg = a.pages + (size_t)x.b * a.max_pages;
                const int total = x.ctx + x.qlen, kb = k & 1;
                if (k >= 2 && !(ok = mbar_wait(bar_ke + 8 * kb, ((k >> 1) - 1) & 1))) break;
                mbar_expect_tx(bar_kf + 8 * kb, ST_BM * SP_HD * 2);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int p = x.k0 / GL_PAGE + half, page = gl_checked(pg[p * GL_PAGE < total ? p : x.k0 / GL_PAGE], a.n_pages, GL_BAD_PAGE);
#pragma unroll
                    for (int s = 0; s < ST_NSEG; ++s)
                        tma_load_2d(sK + kb * RT_TILE_BYTES + st_seg_base(s, ST_BM) + half * GL_PAGE * st_seg(s).width * 2, &maps.k[s], st_seg(s).off,
                                    (page * a.nKV + x.g) * GL_PAGE, bar_kf + 8 * kb);
                }
                ++k;
                int h = x.g * G + x.t0 / x.n_q, i0 = x.start + x.t0 % x.n_q * ST_BM;
                for (int i = 0; i < x.n; ++i, ++j) {
                    const int st = j % STAGES;
                    if (j >= STAGES && !(ok = mbar_wait(bar_qe + 8 * st, ((j / STAGES) - 1) & 1))) break;
                    mbar_expect_tx(bar_qf + 8 * st, ST_BM * SP_HD * 2);
#pragma unroll
                    for (int s = 0; s < ST_NSEG; ++s)
                        tma_load_2d(sQ + st * RT_TILE_BYTES + st_seg_base(s, ST_BM), &maps.q[s], h * SP_HD + st_seg(s).off, x.row0 + i0, bar_qf + 8 * st);
                    i0 += ST_BM;
                    if (i0 >= x.qlen) { i0 = x.start; ++h; }
                }
            }
            if (!ok) failed = 1;
        }
    } else if (warp == PRODUCER + 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = umma_idesc_bf16(ST_BM, 0);
            bool ok = true;
            for (int round = 0; round < rounds && ok && !failed; ++round) {
                if (item_of(round) >= n_items) continue;
                const int n = rt_item(a, item_of(round)).n, kb = k & 1;
                if (n == 0) continue;
                ok = mbar_wait(bar_kf + 8 * kb, (k >> 1) & 1);
                for (int i = 0; ok && i < n; ++i, ++j) {
                    const int st = j % STAGES;
                    ok = mbar_wait(bar_qf + 8 * st, (j / STAGES) & 1) && (j < 2 || mbar_wait(bar_se + 8 * (j & 1), ((j >> 1) - 1) & 1));
                    if (!ok) break;
                    tc_fence_after();
                    bool begin = true;
#pragma unroll
                    for (int s = 0; s < ST_NSEG; ++s) {
                        const int rb = st_seg(s).width * 2;
                        const uint64_t dk = umma_tile_desc(sK + kb * RT_TILE_BYTES + st_seg_base(s, ST_BM), rb);
                        const uint64_t dq = umma_tile_desc(sQ + st * RT_TILE_BYTES + st_seg_base(s, ST_BM), rb);
#pragma unroll
                        for (int c = 0; c < st_seg(s).width / 16; ++c) {
                            umma_bf16(tmem + ST_BM * (j & 1), dq + 2 * c, dk + 2 * c, idesc, begin ? 0u : 1u);
                            begin = false;
                        }
                    }
                    umma_commit(bar_sf + 8 * (j & 1));
                    umma_commit(bar_qe + 8 * st);
                }
                if (ok) umma_commit(bar_ke + 8 * kb);
                ++k;
            }
            if (!ok) failed = 1;
            if (failed && j > 0) (void)mbar_wait(bar_sf + 8 * ((j - 1) & 1), ((j - 1) >> 1) & 1);      // (its last product writes to tensor memory)
        }
    } else {
        const int r = (warp & 3) * 32 + lane, col = (warp >> 2) * RT_COLS;      // the row of each tile, the first of its keys
        const unsigned tS = tmem + ((unsigned)((warp & 3) * 32) << 16) + col;
        // What an item needs of global memory is asked for while the one before is under way, and its sums leave by additions that nobody
        // waits for: every stall here would be the tensor core's too.  (One addition a position: their order is no matter.)
        auto skipped = [&](const RtItem& x) { return x.n == 0 && (!a.sums || x.k0 >= x.ctx + x.qlen || x.qlen <= 0); };
        auto item_from = [&](int& round) {                 // the next item with something to do, from ``round`` on
            RtItem x = {};
            for (; round < rounds; ++round) {
                if (item_of(round) >= n_items) continue;
                x = rt_item(a, item_of(round));
                if (!skipped(x)) break;
            }
            return x;
        };
        int round = 0, done = 0;
        bool ok = true;
        RtItem x = item_from(round);
        // the rows' statistics, a tile ahead of the scores: where the next tile's lie, and how many tiles its head has left
        const float2* at = nullptr;
        int f0 = 0, left = 0;
        auto begin = [&](const RtItem& y) {
            const int q = y.n > 0 ? y.t0 % y.n_q : 0, h = y.g * G + (y.n > 0 ? y.t0 / y.n_q : 0);
            f0 = y.start + q * ST_BM + r;
            at = (const float2*)a.ml + (size_t)h * a.rows + y.row0 + f0;
            left = y.n_q - q;
        };
        auto fetch = [&](const RtItem& y) {
            const float2 v = f0 < y.qlen ? *at : make_float2(0.f, 1.f);
            at += ST_BM;
            f0 += ST_BM;
            if (--left == 0) {                             // on to the next head's first tile
                at += a.rows - y.n_q * ST_BM;
                f0 -= y.n_q * ST_BM;
                left = y.n_q;
            }
            return v;
        };
        auto page_of = [&](const RtItem& y) {              // of the key whose sum this thread writes
            const int key = y.k0 + threadIdx.x;
            return threadIdx.x < ST_BM && key < y.ctx + y.qlen ? gl_checked(a.pages[(size_t)y.b * a.max_pages + key / GL_PAGE], a.n_pages, GL_BAD_PAGE) : 0;
        };
        float2 next = make_float2(0.f, 1.f);
        int page = 0;
        if (round < rounds) {
            begin(x);
            if (x.n > 0) next = fetch(x);
            page = page_of(x);
        }
        while (round < rounds) {
            int after = round + 1;
            const RtItem y = item_from(after);             // (the one behind)
            const int total = x.ctx + x.qlen;
            // of this thread's keys the row of the tile at i0 sees the first i0 + r + ahead; none if there is no such query
            const int ahead = x.ctx - x.k0 - col + 1, sure = RT_COLS - ahead - (warp & 3) * 32, end = x.qlen - (warp & 3) * 32 - 31;
            int i0 = x.start + (x.n > 0 ? x.t0 % x.n_q * ST_BM : 0);
            float acc[RT_COLS];
#pragma unroll
            for (int i = 0; i < RT_COLS; ++i) acc[i] = 0.f;
            for (int i = 0; i < x.n; ++i, ++j) {
                // (an approximate quotient, off by 2 steps of 2^-23 at most: less than the power beside it)
                const float m = next.x, inv = __fdividef(1.0f, next.y);
                if (i + 1 < x.n) next = fetch(x);
                // (a warp whose wait ran out goes on through the motions: the others meet it at the barrier)
                ok = ok && mbar_wait(bar_sf + 8 * (j & 1), (j >> 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) continue;
                tc_fence_after();
                unsigned su[RT_COLS];
                tmem_ld32(tS + ST_BM * (j & 1), su);
                tc_fence_before();                         // (all read: the buffer may be written again)
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_se + 8 * (j & 1));
                if (i0 >= sure && i0 < end) {              // the warp's rows are there and see all of its keys
#pragma unroll
                    for (int q = 0; q < RT_COLS; ++q) acc[q] = fmaf(sp_exp2(fmaf(__uint_as_float(su[q]), SP_LOG2E, -m)), inv, acc[q]);
                } else {
                    const int seen = i0 + r < x.qlen ? i0 + r + ahead : 0;
#pragma unroll
                    for (int q = 0; q < RT_COLS; ++q) {
                        const float e = sp_exp2(fmaf(__uint_as_float(su[q]), SP_LOG2E, -m)) * inv;
                        acc[q] += q < seen ? e : 0.f;
                    }
                }
                i0 += ST_BM;
                if (i0 >= x.qlen) i0 = x.start;
            }
            if (!ok) failed = 1;
            const int mine = page;
            if (after < rounds) {
                begin(y);
                if (y.n > 0) next = fetch(y);
                page = page_of(y);
            }
            sums[done & 1][warp][lane] = rt_sum_lanes(acc, lane);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * RT_WARPS) : "memory");
            const int key = x.k0 + threadIdx.x;
            if (threadIdx.x < ST_BM && key < total && !failed) {
                const float (*f)[RT_COLS] = &sums[done & 1][threadIdx.x / RT_COLS * 4];
                const int c = threadIdx.x % RT_COLS;
                const float given = (f[0][c] + f[1][c]) + (f[2][c] + f[3][c]);
                if (a.sums) {
                    if (key < a.reach) a.sums[(((size_t)x.part * a.B + x.b) * a.nKV + x.g) * a.reach + key] = given;
                } else {
                    float* w = a.weights + ((size_t)mine * a.nKV + x.g) * GL_PAGE + key % GL_PAGE;
                    if (key < x.ctx) atomicAdd(w, given);
                    else *w = given;
                }
            }
            x = y;
            round = after;
            ++done;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == PRODUCER) {
        tc_fence_after();
        tmem_dealloc(tmem, 256);
        if (failed && lane == 0) {                         // a wait ran out: nothing is left on its way into this block's memory
            for (int i = max(0, j - STAGES); i < j; ++i) (void)mbar_wait(bar_qf + 8 * (i % STAGES), (i / STAGES) & 1);
            for (int i = max(0, k - 2); i < k; ++i) (void)mbar_wait(bar_kf + 8 * (i & 1), (i >> 1) & 1);
        }
    }
    if (threadIdx.x == 0 && failed) atomicExch(&gl_wait_failed, 1);
}

static int launch_run_tc(const RunArgs& a, int n_tokens, int sms, cudaStream_t stream) {
    RtMaps maps;
    const uint64_t kv_rows = (uint64_t)a.n_pages * a.nKV * GL_PAGE;
    if (kv_rows > 0x7fffffffULL || a.parts < 1 || a.parts > 65535 || (a.parts > 1 && !a.sums)) return GL_ERR_SHAPE;
    for (int s = 0; s < ST_NSEG; ++s) {
        int rc = gl_cached_map(&maps.k[s], a.k_cache, kv_rows, SP_HD, GL_PAGE, st_seg(s).width, 2);
        if (rc == GL_OK) rc = gl_cached_map(&maps.q[s], a.q, (uint64_t)n_tokens, (uint64_t)a.nH * SP_HD, ST_BM, st_seg(s).width, 2);
        if (rc != GL_OK) return rc;
    }
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    const size_t smem = (size_t)RT_TILE_BYTES * (2 + rt_stages()) + 16 * rt_stages() + 64 + 1024;
    if (!allowed[dev]) {
        if (cudaFuncSetAttribute(run_weigh_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
            cudaGetLastError();
            return GL_ERR_SMEM;
        }
        allowed[dev] = true;
    }
    const long long items = (long long)((a.reach + ST_BM - 1) / ST_BM) * a.nKV * a.B * a.parts;
    if (items > 0x3fffffffLL || sms < 1) return GL_ERR_SHAPE;
    const int rc = gl_launch(run_weigh_tc_kernel, dim3((unsigned)(items < sms ? items : sms)), dim3(RT_THREADS), smem, stream, 1, a, (int)items, maps);
    return rc != GL_OK || !a.sums ? rc : launch_given_join(a, a.sums, a.parts, a.shared, stream);
}
#else
static int launch_run_tc(const RunArgs&, int, int, cudaStream_t) { return GL_ERR_SHAPE; }
#endif

#define RW_SMEM (3 * SP_TILE + 2 * RW_ROWS * 2 * 4)
// The weights of runs of up to max_qlen tokens whose attention has been computed.  known: ml holds the rows' statistics already (the
// tcgen05 attention left them), else they are computed into it.  tensor > 0: on tcgen05, on that many SMs (heads of up to 128; known).
GL_API int gl_attention_weigh_runs(const RunArgs* args, int max_qlen, int n_tokens, int known, int tensor, cudaStream_t stream) {
    const RunArgs& a = *args;
    if (a.B <= 0 || max_qlen <= 0) return GL_OK;
    if (a.nH <= 0 || a.nKV <= 0 || a.nH % a.nKV || a.B > 65535 || a.nKV > 65535 || a.reach <= 0 || a.last < 0 || !a.ml || !a.weights) return GL_ERR_SHAPE;
    if ((a.parts > 1 || a.shared) && !a.sums) return GL_ERR_SHAPE;
    if (((uintptr_t)a.q | (uintptr_t)a.k_cache) & 15 || (uintptr_t)a.ml & 7) return GL_ERR_ALIGN;
    if (tensor) return known ? launch_run_tc(a, n_tokens, tensor, stream) : GL_ERR_SHAPE;
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    if (!allowed[dev]) {
        if (cudaFuncSetAttribute(run_stats_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RW_SMEM) != cudaSuccess ||
            cudaFuncSetAttribute(run_weigh_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RW_SMEM) != cudaSuccess) {
            cudaGetLastError();
            return GL_ERR_SMEM;
        }
        allowed[dev] = true;
    }
    if (!known) {
        const int counted = a.last > 0 && a.last < max_qlen ? a.last : max_qlen;
        const long long tiles = ((long long)counted * (a.nH / a.nKV) + RW_ROWS - 1) / RW_ROWS;
        if (tiles > 0x7fffffffLL) return GL_ERR_SHAPE;
        const int rc = gl_launch(run_stats_kernel, dim3((unsigned)tiles, a.nKV, a.B), dim3(SP_THREADS), (size_t)RW_SMEM, stream, 1, a);
        if (rc != GL_OK) return rc;
    }
    const int rc = gl_launch(run_weigh_kernel, dim3((a.reach + GL_PAGE - 1) / GL_PAGE, a.nKV, a.B), dim3(SP_THREADS), (size_t)RW_SMEM, stream, 1, a);
    return rc != GL_OK || !a.sums ? rc : launch_given_join(a, a.sums, 1, a.shared, stream);
}
