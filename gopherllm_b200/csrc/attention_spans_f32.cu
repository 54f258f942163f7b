// Attention of few query rows over spans of a paged cache in 32 bits: the same two operators as for bfloat16 (shared first
// pages; the weight every position is given), with 32-bit products and sums throughout, any head size up to 256.
//
// A block takes one span for up to R rows (8 at most).  Pages of keys and values come to shared memory by cp.async; a thread
// multiplies one key with half the rows (its key in 16-byte pieces at an odd pitch of them, so that eight lanes touch all
// banks; the rows' pieces are broadcasts), a warp takes the softmax of a row, and a thread adds up one or two dims of the
// values for all rows.  What bounds it is the FMA pipe once a block has eight rows, memory below.
//
// Runs of several tokens take rows of consecutive queries; a second kernel then walks the cache page by page, multiplies its
// keys with all the rows that see them and adds up e^(s - m) / l.  No sum depends on the order in which blocks run.
#include "common.cuh"

#define SF_THREADS 128
#define SF_MAX_HD 256

struct SpanF32Args {
    const float* q;               // [rows, nH*hd], scaled
    float* out;
    const float* k_cache;         // [pages, nKV, GL_PAGE, hd]
    const float* v_cache;
    const int* seq_row;           // [B] first row of q and out, or null (row b is sequence b)
    const int* seq_qlen;          // [B] or null (one token each)
    const int* seq_ctx;           // [B] positions cached before this step
    const int* pages;             // [B, max_pages]
    const int* order;             // as in attention_spans.cu
    const int* items;
    const int* seq_shared;
    float* part_o;                // [B, nH, slots, hd]
    float* part_ml;               // [B, nH, slots, 2], for runs [rows, nH, 2]
    float* scores;                // [B, nH, reach] or null
    float* weights;               // [pages, nKV, GL_PAGE] or null
    int B, nH, nKV, max_pages, n_pages, n_items, splits, slots, chunks, reach, hd, last;
};

enum { SF_OWN = 0, SF_SHARED = 1, SF_RUN = 2 };

__host__ __device__ inline int sf_pitch(int hd) { return 4 * (((hd + 3) / 4) | 1); }      // floats between two keys: an odd number of 16-byte pieces
__host__ __device__ inline int sf_stages(int hd) { return hd <= 128 ? 2 : 1; }
static size_t sf_smem(int hd) {
    return sizeof(float) * (2 * (size_t)sf_stages(hd) * GL_PAGE * sf_pitch(hd) + 8 * (size_t)sf_pitch(hd) + 8 * GL_PAGE + 3 * 8 + 8 * SF_MAX_HD) + sizeof(int) * 3 * 8;
}

// rows [0, n_valid) of a page to the pitch of shared memory, zero behind them and behind the head size
__device__ __forceinline__ void sf_load_page(float* dst, const float* src, int n_valid, int hd, int pitch) {
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
    if ((hd & 3) == 0) {
        const int n = hd >> 2;
        for (int i = threadIdx.x; i < GL_PAGE * n; i += SF_THREADS) {
            const int r = i / n, c = i - r * n;
            const bool ok = r < n_valid;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + (r * pitch + 4 * c) * 4), "l"(ok ? src + (size_t)r * hd + 4 * c : src), "r"(ok ? 16 : 0));
        }
    } else {
        const int n = (hd + 3) & ~3;
        for (int i = threadIdx.x; i < GL_PAGE * n; i += SF_THREADS) {
            const int r = i / n, c = i - r * n;
            const bool ok = r < n_valid && c < hd;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d + (r * pitch + c) * 4), "l"(ok ? src + (size_t)r * hd + c : src), "r"(ok ? 4 : 0));
        }
    }
}
__device__ __forceinline__ float sf_factor(float m_i, float m) { return m_i == m ? 1.0f : expf(m_i - m); }

// scores of one key with N rows of queries (row pitch as for keys)
template <int N>
__device__ __forceinline__ void sf_scores(const float* key, const float* q, int pitch, int n4, float (&s)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
    for (int c = 0; c < n4; ++c) {
        const float4 k = *(const float4*)(key + 4 * c);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float4 x = *(const float4*)(q + i * pitch + 4 * c);
            s[i] = fmaf(k.x, x.x, fmaf(k.y, x.y, fmaf(k.z, x.z, fmaf(k.w, x.w, s[i]))));
        }
    }
}

template <int R, int KIND>
__global__ void __launch_bounds__(SF_THREADS)
span_f32_kernel(SpanF32Args a) {
    extern __shared__ __align__(16) float sf[];
    const int hd = a.hd, pitch = sf_pitch(hd), stages = sf_stages(hd), n4 = (hd + 3) / 4;
    float* pages_at = sf;                                          // [stages][keys, values][64][pitch]
    float* qs = pages_at + 2 * stages * GL_PAGE * pitch;           // [8][pitch]
    float* ps = qs + 8 * pitch;                                    // [8][64] scores, then weights
    float* row_m = ps + 8 * GL_PAGE;                               // [8] maximum, sum, factor
    float* row_l = row_m + 8;
    float* row_c = row_l + 8;
    float* halves = row_c + 8;                                     // [8][hd <= 64] the second half of the keys' sums
    int* row_seq = (int*)(halves + 8 * SF_MAX_HD);                 // [8] sequence (runs: row of q), head, last position seen
    int* row_head = row_seq + 8;
    int* row_last = row_head + 8;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.nH / a.nKV;
    gl_grid_launch_dependents();
    gl_grid_wait();

    int g, rows, p_begin, p_end, slot, table;
    if (KIND == SF_SHARED) {
        const int* it = a.items + 6 * blockIdx.x;
        g = blockIdx.y;
        rows = it[2]; p_begin = it[3]; p_end = it[4]; slot = it[5];
        table = a.order[it[0]];
        if (tid < 8) {
            const int r = it[1] + tid, b = tid < rows ? a.order[it[0] + r / G] : -1;
            row_seq[tid] = b;
            row_head[tid] = g * G + r % G;
            row_last[tid] = b >= 0 ? a.seq_ctx[b] : -1;
        }
    } else if (KIND == SF_RUN) {
        const int b = blockIdx.z, n = a.seq_qlen[b] * G, r0 = blockIdx.x * R;
        if (r0 >= n) return;
        g = blockIdx.y; rows = min(R, n - r0); slot = 0; table = b;
        p_begin = 0;
        p_end = (a.seq_ctx[b] + (r0 + rows - 1) / G) / GL_PAGE + 1;
        if (tid < 8) {
            const int i = (r0 + tid) / G;
            row_seq[tid] = tid < rows ? a.seq_row[b] + i : -1;
            row_head[tid] = g * G + (r0 + tid) % G;
            row_last[tid] = tid < rows ? a.seq_ctx[b] + i : -1;
        }
    } else {
        const int b = blockIdx.z;
        g = blockIdx.y / a.chunks;
        if (a.seq_qlen && a.seq_qlen[b] <= 0) return;
        const int per_chunk = (G + a.chunks - 1) / a.chunks, h0 = (blockIdx.y - g * a.chunks) * per_chunk;
        rows = min(per_chunk, G - h0);
        const int pos = a.seq_ctx[b], first = a.seq_shared ? a.seq_shared[2 * b] : 0;
        const int n = max(0, pos / GL_PAGE + 1 - first), per = (n + a.splits - 1) / a.splits;
        p_begin = first + (int)blockIdx.x * per;
        p_end = min(first + n, p_begin + per);
        slot = (a.seq_shared ? a.seq_shared[2 * b + 1] : 0) + blockIdx.x;
        table = b;
        if (tid < 8) {
            row_seq[tid] = tid < rows ? b : -1;
            row_head[tid] = g * G + h0 + tid;
            row_last[tid] = tid < rows ? pos : -1;
        }
    }
    if (tid < 8) { row_m[tid] = -INFINITY; row_l[tid] = 0.f; }
    const int total = a.seq_ctx[table] + (KIND == SF_RUN ? a.seq_qlen[table] : 1);      // positions of the sequence that were written
    const int* pg = a.pages + (size_t)table * a.max_pages;
    auto load = [&](int st, int p) {
        const size_t at = ((size_t)gl_checked(pg[p], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE * hd;
        const int nv = KIND == SF_SHARED ? GL_PAGE : min(GL_PAGE, total - p * GL_PAGE);
        sf_load_page(pages_at + 2 * st * GL_PAGE * pitch, a.k_cache + at, nv, hd, pitch);
        sf_load_page(pages_at + (2 * st + 1) * GL_PAGE * pitch, a.v_cache + at, nv, hd, pitch);
    };
    if (stages == 2) {
        if (p_begin < p_end) load(0, p_begin);
        asm volatile("cp.async.commit_group;");
    }
    __syncthreads();
    for (int i = tid; i < 8 * 4 * n4; i += SF_THREADS) {
        const int r = i / (4 * n4), c = i - r * 4 * n4, b = row_seq[r];
        const int at = b >= 0 && KIND != SF_RUN && a.seq_row ? a.seq_row[b] : b;
        qs[r * pitch + c] = b >= 0 && c < hd ? a.q[((size_t)at * a.nH + row_head[r]) * hd + c] : 0.f;
    }
    int least = 0x7fffffff;                                       // the earliest last position among the block's rows
    for (int r = 0; r < rows; ++r) least = min(least, row_last[r]);
    constexpr int RH = R > 1 ? R / 2 : 1;                         // rows a thread multiplies its key with
    float o[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) o[r][0] = o[r][1] = 0.f;
    const bool narrow = hd <= 64;                                 // two threads a dim, each with half the keys; else up to two dims a thread
    const int d0 = narrow ? tid & 63 : tid, k0 = narrow ? (tid >> 6) * 32 : 0, k1 = narrow ? k0 + 32 : GL_PAGE;

    for (int p = p_begin; p < p_end; ++p) {
        int st = 0;
        __syncthreads();                                          // the page read last time is free
        if (stages == 2) {
            st = (p - p_begin) & 1;
            if (p + 1 < p_end) load(st ^ 1, p + 1);
            asm volatile("cp.async.commit_group;");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            load(0, p);
            asm volatile("cp.async.commit_group;");
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        const float* ks = pages_at + 2 * st * GL_PAGE * pitch;
        const float* vs = ks + GL_PAGE * pitch;
        const int j0 = p * GL_PAGE;
        {
            const int key = tid & 63, r0 = (tid >> 6) * RH;
            if (r0 < R) {
                float s[RH];
                sf_scores<RH>(ks + key * pitch, qs + r0 * pitch, pitch, n4, s);
#pragma unroll
                for (int i = 0; i < RH; ++i) {
                    if (KIND == SF_OWN && a.scores && r0 + i < rows && j0 + key < min(total, a.reach))
                        a.scores[((size_t)table * a.nH + row_head[r0 + i]) * a.reach + j0 + key] = s[i];
                    ps[(r0 + i) * GL_PAGE + key] = j0 + key <= row_last[r0 + i] ? s[i] : -INFINITY;
                }
            }
        }
        __syncthreads();
        for (int r = warp; r < R; r += SF_THREADS / 32) {
            const float x = ps[r * GL_PAGE + lane], y = ps[r * GL_PAGE + 32 + lane];
            const float old = row_m[r], m = fmaxf(old, gl_warp_max(fmaxf(x, y))), mu = m == -INFINITY ? 0.f : m;
            const float e = expf(x - mu), f = expf(y - mu), sum = gl_warp_sum(e + f), c = sf_factor(old, m);
            ps[r * GL_PAGE + lane] = e;
            ps[r * GL_PAGE + 32 + lane] = f;
            __syncwarp();
            if (lane == 0) { row_m[r] = m; row_c[r] = c; row_l[r] = fmaf(row_l[r], c, sum); }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) { const float c = row_c[r]; o[r][0] *= c; o[r][1] *= c; }
        for (int k = k0; k < k1; k += 4) {
            float v[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i][0] = d0 < hd ? vs[(k + i) * pitch + d0] : 0.f;
                v[i][1] = !narrow && d0 + SF_THREADS < hd ? vs[(k + i) * pitch + d0 + SF_THREADS] : 0.f;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float4 w = *(const float4*)(ps + r * GL_PAGE + k);
                if (j0 + k + 3 > least) {                         // a value that a row does not see must not reach it, were it NaN
                    const int n = row_last[r] - j0 - k;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (n >= 0) o[r][i] = fmaf(w.x, v[0][i], o[r][i]);
                        if (n >= 1) o[r][i] = fmaf(w.y, v[1][i], o[r][i]);
                        if (n >= 2) o[r][i] = fmaf(w.z, v[2][i], o[r][i]);
                        if (n >= 3) o[r][i] = fmaf(w.w, v[3][i], o[r][i]);
                    }
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) o[r][i] = fmaf(w.x, v[0][i], fmaf(w.y, v[1][i], fmaf(w.z, v[2][i], fmaf(w.w, v[3][i], o[r][i]))));
            }
        }
    }
    if (stages == 2) asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (narrow && tid >= 64)
#pragma unroll
        for (int r = 0; r < R; ++r) halves[r * 64 + d0] = o[r][0];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= rows || (narrow && tid >= 64)) continue;
        const float l = row_l[r];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = d0 + i * SF_THREADS;
            if (d >= hd || (narrow && i)) continue;
            const float v = narrow ? o[r][0] + halves[r * 64 + d] : o[r][i];
            if (KIND == SF_RUN) a.out[((size_t)row_seq[r] * a.nH + row_head[r]) * hd + d] = l == 0.f ? 0.f : v / l;
            else a.part_o[(((size_t)row_seq[r] * a.nH + row_head[r]) * a.slots + slot) * hd + d] = v;
        }
        if (tid == 0) {
            float* ml = a.part_ml + ((size_t)row_seq[r] * a.nH + row_head[r]) * 2 * (KIND == SF_RUN ? 1 : a.slots) + 2 * slot;
            ml[0] = row_m[r];
            ml[1] = l;
        }
    }
}

// The spans of a row put together: blockIdx = (head, sequence).
__global__ void span_f32_join_kernel(SpanF32Args a) {
    gl_grid_launch_dependents();
    gl_grid_wait();
    const int h = blockIdx.x, b = blockIdx.y;
    if (a.seq_qlen && a.seq_qlen[b] <= 0) return;
    const int n = (a.seq_shared ? a.seq_shared[2 * b + 1] : 0) + a.splits;
    const size_t at = ((size_t)b * a.nH + h) * a.slots;
    const float* ml = a.part_ml + at * 2;
    float m = -INFINITY;
    for (int s = 0; s < n; ++s) m = fmaxf(m, ml[2 * s]);
    float* out = a.out + ((size_t)(a.seq_row ? a.seq_row[b] : b) * a.nH + h) * a.hd;
    for (int d = threadIdx.x; d < a.hd; d += blockDim.x) {
        float o = 0.f, l = 0.f;
        for (int s = 0; s < n; ++s) {
            const float f = sf_factor(ml[2 * s], m);
            o = fmaf(f, a.part_o[(at + s) * a.hd + d], o);
            l = fmaf(f, ml[2 * s + 1], l);
        }
        out[d] = l == 0.f ? 0.f : o / l;
    }
}

// One token a sequence: the scores written down become weights, added up over the query heads of a key/value head.
__global__ void __launch_bounds__(GL_PAGE)
span_f32_weigh_kernel(SpanF32Args a) {
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
        for (int s = 0; s < a.splits; ++s) l = fmaf(sf_factor(ml[2 * s], m), ml[2 * s + 1], l);
        if (j <= pos && j < a.reach) given += expf(a.scores[((size_t)b * a.nH + h) * a.reach + j] - m) / l;
    }
    if (j > pos || j >= a.reach) return;
    float* w = a.weights + ((size_t)gl_checked(a.pages[(size_t)b * a.max_pages + p], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + threadIdx.x;
    *w = j < pos ? *w + given : given;
}

// Runs: blockIdx = (page, key/value head, sequence); the page's keys against all rows of the run that see them.
__global__ void __launch_bounds__(SF_THREADS)
run_f32_weigh_kernel(SpanF32Args a) {
    extern __shared__ __align__(16) float sf[];
    const int hd = a.hd, pitch = sf_pitch(hd), n4 = (hd + 3) / 4, G = a.nH / a.nKV;
    float* ks = sf;                                                // [64][pitch]
    float* qs = ks + GL_PAGE * pitch;                              // [8][pitch]
    float* row_m = qs + 8 * pitch;                                 // [8]
    float* row_l = row_m + 8;
    float* halves = row_l + 8;                                     // [64]
    int* row_last = (int*)(halves + GL_PAGE);                      // [8]
    const int tid = threadIdx.x, b = blockIdx.z, g = blockIdx.y, p = blockIdx.x;
    gl_grid_launch_dependents();
    gl_grid_wait();
    const int qlen = a.seq_qlen[b], ctx = a.seq_ctx[b], total = ctx + qlen;
    if (qlen <= 0 || p * GL_PAGE >= total) return;
    const size_t page = (size_t)gl_checked(a.pages[(size_t)b * a.max_pages + p], a.n_pages, GL_BAD_PAGE);
    sf_load_page(ks, a.k_cache + (page * a.nKV + g) * GL_PAGE * hd, min(GL_PAGE, total - p * GL_PAGE), hd, pitch);
    asm volatile("cp.async.commit_group;");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    const int key = tid & 63, half = tid >> 6, j = p * GL_PAGE + key;
    const int i0 = max(max(0, p * GL_PAGE - ctx), a.last > 0 ? qlen - a.last : 0);
    float given = 0.f;
    for (int r0 = i0 * G; r0 < qlen * G; r0 += 8) {
        __syncthreads();
        for (int i = tid; i < 8 * 4 * n4; i += SF_THREADS) {
            const int r = i / (4 * n4), c = i - r * 4 * n4, row = r0 + r;
            const bool ok = row < qlen * G && c < hd;
            qs[r * pitch + c] = ok ? a.q[((size_t)(a.seq_row[b] + row / G) * a.nH + g * G + row % G) * hd + c] : 0.f;
        }
        if (tid < 8) {
            const int row = r0 + tid;
            const bool ok = row < qlen * G;
            const float* ml = a.part_ml + ((size_t)(a.seq_row[b] + (ok ? row / G : 0)) * a.nH + g * G + (ok ? row % G : 0)) * 2;
            row_m[tid] = ml[0];
            row_l[tid] = ml[1];
            row_last[tid] = ok ? ctx + row / G : -1;
        }
        __syncthreads();
        float s[4];
        sf_scores<4>(ks + key * pitch, qs + half * 4 * pitch, pitch, n4, s);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j <= row_last[half * 4 + i]) given += expf(s[i] - row_m[half * 4 + i]) / row_l[half * 4 + i];
    }
    if (half) halves[key] = given;
    __syncthreads();
    if (half || j >= total) return;
    float* w = a.weights + (page * a.nKV + g) * GL_PAGE + key;
    given += halves[key];
    *w = j < ctx ? *w + given : given;
}

template <typename F>
static int allow_smem(F* kernel, size_t bytes) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess) return GL_OK;
    cudaGetLastError();
    return GL_ERR_SMEM;
}
template <int R, int KIND>
static int launch_f32(const SpanF32Args& a, dim3 grid, cudaStream_t stream) {
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    if (!allowed[dev]) {
        const size_t a128 = sf_smem(128), a256 = sf_smem(SF_MAX_HD);
        if (allow_smem(span_f32_kernel<R, KIND>, a128 > a256 ? a128 : a256) != GL_OK) return GL_ERR_SMEM;
        allowed[dev] = true;
    }
    return gl_launch(span_f32_kernel<R, KIND>, grid, dim3(SF_THREADS), sf_smem(a.hd), stream, 1, a);
}
template <int KIND>
static int launch_f32_rows(const SpanF32Args& a, int rows, dim3 grid, cudaStream_t stream) {
    if (rows <= 1) return launch_f32<1, KIND>(a, grid, stream);
    if (rows <= 2) return launch_f32<2, KIND>(a, grid, stream);
    if (rows <= 4) return launch_f32<4, KIND>(a, grid, stream);
    return launch_f32<8, KIND>(a, grid, stream);
}

static int f32_checked(const SpanF32Args& a) {
    if (a.nH <= 0 || a.nKV <= 0 || a.nH % a.nKV || a.nKV > 65535 || a.B > 65535 || a.hd <= 0 || a.hd > SF_MAX_HD || a.max_pages <= 0) return GL_ERR_SHAPE;
    if ((((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) && a.hd % 4 == 0) return GL_ERR_ALIGN;
    return a.part_ml ? GL_OK : GL_ERR_SHAPE;
}
static int f32_spans_checked(const SpanF32Args& a) {
    const int G = a.nH / a.nKV;
    if (a.splits < 1 || a.slots < a.splits || !a.part_o) return GL_ERR_SHAPE;
    if (a.chunks < 1 || a.chunks > G || (long long)a.nKV * a.chunks > 65535 || (G + a.chunks - 1) / a.chunks > 8) return GL_ERR_SHAPE;
    return (a.chunks - 1) * ((G + a.chunks - 1) / a.chunks) >= G ? GL_ERR_SHAPE : GL_OK;
}

GL_API int gl_attention_prefix_f32(const SpanF32Args* args, int rows, cudaStream_t stream) {
    const SpanF32Args& a = *args;
    if (a.B <= 0) return GL_OK;
    int rc = f32_checked(a);
    if (rc == GL_OK) rc = f32_spans_checked(a);
    if (rc != GL_OK) return rc;
    if (a.n_items < 0 || a.scores || a.weights || !a.seq_shared || (a.n_items > 0 && (!a.items || !a.order || rows < 1 || rows > 8))) return GL_ERR_SHAPE;
    if (a.n_items > 0 && (rc = launch_f32_rows<SF_SHARED>(a, rows, dim3(a.n_items, a.nKV), stream)) != GL_OK) return rc;
    const int G = a.nH / a.nKV;
    if ((rc = launch_f32_rows<SF_OWN>(a, (G + a.chunks - 1) / a.chunks, dim3(a.splits, a.nKV * a.chunks, a.B), stream)) != GL_OK) return rc;
    return gl_launch(span_f32_join_kernel, dim3(a.nH, a.B), dim3(a.hd >= 128 ? 128 : 64), 0, stream, 1, a);
}

GL_API int gl_attention_weighed_f32(const SpanF32Args* args, cudaStream_t stream) {
    const SpanF32Args& a = *args;
    if (a.B <= 0) return GL_OK;
    int rc = f32_checked(a);
    if (rc == GL_OK) rc = f32_spans_checked(a);
    if (rc != GL_OK) return rc;
    if (!a.scores || !a.weights || a.seq_shared || a.reach <= 0) return GL_ERR_SHAPE;
    const int G = a.nH / a.nKV;
    if ((rc = launch_f32_rows<SF_OWN>(a, (G + a.chunks - 1) / a.chunks, dim3(a.splits, a.nKV * a.chunks, a.B), stream)) != GL_OK) return rc;
    if ((rc = gl_launch(span_f32_join_kernel, dim3(a.nH, a.B), dim3(a.hd >= 128 ? 128 : 64), 0, stream, 1, a)) != GL_OK) return rc;
    return gl_launch(span_f32_weigh_kernel, dim3((a.reach + GL_PAGE - 1) / GL_PAGE, a.nKV, a.B), dim3(GL_PAGE), 0, stream, 1, a);
}

// runs of up to max_qlen tokens
GL_API int gl_attention_weighed_runs_f32(const SpanF32Args* args, int max_qlen, cudaStream_t stream) {
    const SpanF32Args& a = *args;
    if (a.B <= 0 || max_qlen <= 0) return GL_OK;
    int rc = f32_checked(a);
    if (rc != GL_OK) return rc;
    if (!a.weights || !a.seq_row || !a.seq_qlen || a.reach <= 0 || a.last < 0) return GL_ERR_SHAPE;
    const long long tiles = ((long long)max_qlen * (a.nH / a.nKV) + 7) / 8;
    if (tiles > 0x7fffffffLL) return GL_ERR_SHAPE;
    if ((rc = launch_f32<8, SF_RUN>(a, dim3((unsigned)tiles, a.nKV, a.B), stream)) != GL_OK) return rc;
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    auto need = [](int hd) { return sizeof(float) * ((GL_PAGE + 8) * (size_t)sf_pitch(hd) + 16 + GL_PAGE) + sizeof(int) * 8; };
    if (!allowed[dev]) {
        if (allow_smem(run_f32_weigh_kernel, need(SF_MAX_HD)) != GL_OK) return GL_ERR_SMEM;
        allowed[dev] = true;
    }
    return gl_launch(run_f32_weigh_kernel, dim3((a.reach + GL_PAGE - 1) / GL_PAGE, a.nKV, a.B), dim3(SF_THREADS), need(a.hd), stream, 1, a);
}
