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
// A block takes one span for up to 8 NT rows.  It streams the span's pages through shared memory with cp.async; inside a page
// each of its four warps owns 16 of the 64 keys: scores are an mma.sync chain with the keys as the 16-row operand and the rows as
// columns, maximum, sum and rescaling are 32-bit, the weights turn into the other operand of the second product by a transposing
// move between lanes, and the weighted values are a second chain into 32-bit accumulators.  The warps' four softmaxes meet at the
// end of the span.  Weights are rounded to bfloat16 for the second product (its operand's type); the sums take them unrounded.
#include "common.cuh"
#include "decode_common.cuh"

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
#define SP_STAGES 2                                 // pages of keys and values in flight
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
    int B, nH, nKV, max_pages, n_pages, n_items, splits, slots, chunks, reach;
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

template <int NT>
__host__ __device__ constexpr int sp_fixed_bytes() {       // queries, then per row: sequence, head, last position seen
    return 8 * NT * SP_ROW + 8 * NT * 12;
}
template <int NT>
__host__ __device__ constexpr size_t sp_smem() {
    const size_t pages = 2 * SP_STAGES * (size_t)SP_TILE;
    const size_t merge = sizeof(float) * (4 * 8 * NT * 2 + 4 * (size_t)SP_HD * 8 * NT);       // over the pages, when they are done
    return (pages > merge ? pages : merge) + sp_fixed_bytes<NT>();
}

// SHARED: blockIdx.x is an item of the plan; else blockIdx = (split, key/value head and its share of the query heads, sequence).
template <int NT, bool SHARED>
__global__ void __launch_bounds__(SP_THREADS)
attn_span_kernel(SpanArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr size_t AREA = sp_smem<NT>() - sp_fixed_bytes<NT>();
    const unsigned sbase = ad_smem(smem);
    unsigned char* qs = smem + AREA;                               // [8 NT] rows of queries
    int* row_seq = (int*)(qs + 8 * NT * SP_ROW);                   // [8 NT]
    int* row_head = row_seq + 8 * NT;
    int* row_last = row_head + 8 * NT;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int grp = lane >> 2, t = lane & 3;
    const int G = a.nH / a.nKV;
    gl_grid_launch_dependents();
    gl_grid_wait();

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
#pragma unroll
    for (int s = 0; s < SP_STAGES - 1; ++s) {
        if (p_begin + s < p_end) load(s, p_begin + s);
        sp_commit();
    }
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
        const int st = (p - p_begin) % SP_STAGES;
        sp_wait<SP_STAGES - 2>();
        __syncthreads();                                   // page p has landed; the stage read last time is free
        {
            const int pn = p + SP_STAGES - 1;
            if (pn < p_end) load((pn - p_begin) % SP_STAGES, pn);
            sp_commit();
        }
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
        if (!SHARED && a.scores) {
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
        const size_t at = ((size_t)row_seq[r] * a.nH + row_head[r]) * a.slots + slot;
        a.part_o[at * SP_HD + d] = ov;
        if (d == 0) { a.part_ml[at * 2] = m; a.part_ml[at * 2 + 1] = l; }
    }
}

// The spans of a row put together: blockIdx = (head, sequence).
__global__ void attn_span_join_kernel(SpanArgs a) {
    gl_grid_launch_dependents();
    gl_grid_wait();
    const int h = blockIdx.x, b = blockIdx.y;
    if (a.seq_qlen && a.seq_qlen[b] <= 0) return;
    const int n = (a.seq_shared ? a.seq_shared[2 * b + 1] : 0) + a.splits;
    const size_t at = ((size_t)b * a.nH + h) * a.slots;
    const float* ml = a.part_ml + at * 2;
    float m = -INFINITY;
    for (int s = 0; s < n; ++s) m = fmaxf(m, ml[2 * s]);
    __nv_bfloat16* out = a.out + ((size_t)(a.seq_row ? a.seq_row[b] : b) * a.nH + h) * SP_HD;
    for (int d = threadIdx.x; d < SP_HD; d += blockDim.x) {
        float o = 0.f, l = 0.f;
        for (int s = 0; s < n; ++s) {
            const float f = sp_factor(ml[2 * s], m);
            o = fmaf(f, a.part_o[(at + s) * SP_HD + d], o);
            l = fmaf(f, ml[2 * s + 1], l);
        }
        out[d] = __float2bfloat16_rn(l == 0.f ? 0.f : o / l);
    }
}

// The weights a row gave its positions, added up over the query heads of a key/value head: blockIdx = (page, key/value head, sequence).
// A position new in this step starts from nothing, whatever its place held.
__global__ void __launch_bounds__(GL_PAGE)
attn_span_weigh_kernel(SpanArgs a) {
    gl_grid_launch_dependents();
    gl_grid_wait();
    const int b = blockIdx.z, g = blockIdx.y, p = blockIdx.x, G = a.nH / a.nKV;
    const int pos = a.seq_ctx[b], j = p * GL_PAGE + threadIdx.x;
    if ((a.seq_qlen && a.seq_qlen[b] <= 0) || p > pos / GL_PAGE) return;
    float given = 0.f;
    for (int h = g * G; h < (g + 1) * G; ++h) {
        const float* ml = a.part_ml + ((size_t)b * a.nH + h) * a.slots * 2;
        float m = -INFINITY, l = 0.f;
        for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[2 * s]);
        for (int s = 0; s < a.splits; ++s) l = fmaf(sp_factor(ml[2 * s], m), ml[2 * s + 1], l);
        if (j <= pos && j < a.reach) given += sp_exp2(fmaf(a.scores[((size_t)b * a.nH + h) * a.reach + j], SP_LOG2E, -m)) / l;
    }
    if (j > pos || j >= a.reach) return;
    float* w = a.weights + ((size_t)gl_checked(a.pages[(size_t)b * a.max_pages + p], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + threadIdx.x;
    *w = j < pos ? *w + given : given;
}

template <int NT, bool SHARED>
static int launch_span(const SpanArgs& a, dim3 grid, cudaStream_t stream) {
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    if (!allowed[dev]) {
        if (cudaFuncSetAttribute(attn_span_kernel<NT, SHARED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sp_smem<NT>()) != cudaSuccess) {
            cudaGetLastError();
            return GL_ERR_SMEM;
        }
        allowed[dev] = true;
    }
    return gl_launch(attn_span_kernel<NT, SHARED>, grid, dim3(SP_THREADS), sp_smem<NT>(), stream, 1, a);
}

template <bool SHARED>
static int launch_spans(const SpanArgs& a, int rows, dim3 grid, cudaStream_t stream) {
    if (rows <= 8) return launch_span<1, SHARED>(a, grid, stream);
    if (rows <= 16) return launch_span<2, SHARED>(a, grid, stream);
    return launch_span<SP_MAX_NT, SHARED>(a, grid, stream);
}

static int span_checked(const SpanArgs& a) {
    if (a.nH <= 0 || a.nKV <= 0 || a.nH % a.nKV || a.B > 65535 || a.splits < 1 || a.slots < a.splits || a.max_pages <= 0) return GL_ERR_SHAPE;
    const int G = a.nH / a.nKV;
    if (a.chunks < 1 || a.chunks > G || (long long)a.nKV * a.chunks > 65535 || (G + a.chunks - 1) / a.chunks > 8 * SP_MAX_NT) return GL_ERR_SHAPE;
    if ((a.chunks - 1) * ((G + a.chunks - 1) / a.chunks) >= G) return GL_ERR_SHAPE;        // every share of the heads has one
    if (((uintptr_t)a.q | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) return GL_ERR_ALIGN;
    if (!a.part_o || !a.part_ml) return GL_ERR_SHAPE;
    return GL_OK;
}

GL_API int gl_attention_span_rows() { return 8 * SP_MAX_NT; }        // rows of q a span takes at most

// rows: the most that one of the plan's items has
GL_API int gl_attention_prefix(const SpanArgs* args, int rows, cudaStream_t stream) {
    const SpanArgs& a = *args;
    if (a.B <= 0) return GL_OK;
    int rc = span_checked(a);
    if (rc != GL_OK) return rc;
    if (a.n_items < 0 || a.scores || a.weights || !a.seq_shared || (a.n_items > 0 && (!a.items || !a.order || rows < 1 || rows > 8 * SP_MAX_NT))) return GL_ERR_SHAPE;
    if (a.n_items > 0 && (rc = launch_spans<true>(a, rows, dim3(a.n_items, a.nKV), stream)) != GL_OK) return rc;
    const int G = a.nH / a.nKV;
    if ((rc = launch_spans<false>(a, (G + a.chunks - 1) / a.chunks, dim3(a.splits, a.nKV * a.chunks, a.B), stream)) != GL_OK) return rc;
    return gl_launch(attn_span_join_kernel, dim3(a.nH, a.B), dim3(SP_HD >= 128 ? 128 : 64), 0, stream, 1, a);
}

GL_API int gl_attention_weighed(const SpanArgs* args, cudaStream_t stream) {
    const SpanArgs& a = *args;
    if (a.B <= 0) return GL_OK;
    int rc = span_checked(a);
    if (rc != GL_OK) return rc;
    if (!a.scores || !a.weights || a.seq_shared || a.reach <= 0) return GL_ERR_SHAPE;
    const int G = a.nH / a.nKV, n_pages = (a.reach + GL_PAGE - 1) / GL_PAGE;
    if ((rc = launch_spans<false>(a, (G + a.chunks - 1) / a.chunks, dim3(a.splits, a.nKV * a.chunks, a.B), stream)) != GL_OK) return rc;
    if ((rc = gl_launch(attn_span_join_kernel, dim3(a.nH, a.B), dim3(SP_HD >= 128 ? 128 : 64), 0, stream, 1, a)) != GL_OK) return rc;
    return gl_launch(attn_span_weigh_kernel, dim3(n_pages, a.nKV, a.B), dim3(GL_PAGE), 0, stream, 1, a);
}

// ---------------------------------------------------------------------------
// Runs of several tokens: the weights their positions are given.  The attention itself is the prefill kernels'; what it does
// not leave behind, each row's maximum and sum, is computed here from the scores alone, and a second kernel walks the cache page
// by page: w[j] += sum over the rows that see j of e^(s - m) / l.  Rows are (query, query head of a key/value head), queries
// first.  Both are a chain of mma.sync and one power a score, which bounds them.  No sum depends on the order of the blocks.
// ---------------------------------------------------------------------------
struct RunArgs {
    const __nv_bfloat16* q;       // [rows, nH*hd], scaled
    const __nv_bfloat16* k_cache; // [pages, nKV, GL_PAGE, hd]
    const int* seq_row;           // [B] first row of q
    const int* seq_qlen;          // [B]
    const int* seq_ctx;           // [B]
    const int* pages;             // [B, max_pages]
    float* ml;                    // [rows, nH, 2]
    float* weights;               // [pages, nKV, GL_PAGE]
    int B, nH, nKV, max_pages, n_pages, reach, last;
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
            float* ml = a.ml + ((size_t)(row0 + row / G) * a.nH + g * G + row % G) * 2;
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
            if (row < end) ml = *(const float2*)(a.ml + ((size_t)(row0 + row / G) * a.nH + g * G + row % G) * 2);
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
            *w = j < ctx ? *w + given[i] : given[i];
        }
    }
    sp_wait<0>();
}

#define RW_SMEM (3 * SP_TILE + 2 * RW_ROWS * 2 * 4)
// The weights of runs of up to max_qlen tokens whose attention has been computed (ml: scratch).
GL_API int gl_attention_weigh_runs(const RunArgs* args, int max_qlen, cudaStream_t stream) {
    const RunArgs& a = *args;
    if (a.B <= 0 || max_qlen <= 0) return GL_OK;
    if (a.nH <= 0 || a.nKV <= 0 || a.nH % a.nKV || a.B > 65535 || a.nKV > 65535 || a.reach <= 0 || a.last < 0 || !a.ml || !a.weights) return GL_ERR_SHAPE;
    if (((uintptr_t)a.q | (uintptr_t)a.k_cache) & 15) return GL_ERR_ALIGN;
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
    const int counted = a.last > 0 && a.last < max_qlen ? a.last : max_qlen;
    const long long tiles = ((long long)counted * (a.nH / a.nKV) + RW_ROWS - 1) / RW_ROWS;
    if (tiles > 0x7fffffffLL) return GL_ERR_SHAPE;
    const int rc = gl_launch(run_stats_kernel, dim3((unsigned)tiles, a.nKV, a.B), dim3(SP_THREADS), (size_t)RW_SMEM, stream, 1, a);
    if (rc != GL_OK) return rc;
    return gl_launch(run_weigh_kernel, dim3((a.reach + GL_PAGE - 1) / GL_PAGE, a.nKV, a.B), dim3(SP_THREADS), (size_t)RW_SMEM, stream, 1, a);
}
