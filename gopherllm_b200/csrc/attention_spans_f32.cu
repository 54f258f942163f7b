// Attention of few query rows over spans of a paged cache in 32 bits: the same two operators as for bfloat16 (shared first
// pages; the weight every position is given), with 32-bit products and sums throughout, any head size up to 256.
//
// A block takes one span for up to R rows (8 at most).  Pages of keys and values come to shared memory by cp.async; a thread
// multiplies one key with half the rows (its key in 16-byte pieces at an odd pitch of them, so that eight lanes touch all
// banks; the rows' pieces are broadcasts), a warp takes the softmax of a row, and a thread adds up one or two dims of the
// values for all rows.  So it is for heads that are no whole 16-byte pieces; all others stream (below).
#include "common.cuh"
#include "span_weights.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

#define SF_THREADS 128
#define SF_MAX_HD 256

struct SpanF32Args {
    const float* q;               // [rows, nH*hd], scaled
    float* out;
    const float* k_cache;         // [pages, nKV, GL_PAGE, hd]
    const float* v_cache;
    const int* seq_row;           // [B] row of q and out, or null (row b is sequence b)
    const int* seq_qlen;          // [B] or null (one token each)
    const int* seq_ctx;           // [B] positions cached before this step
    const int* pages;             // [B, max_pages]
    const int* order;             // as in attention_spans.cu
    const int* items;
    const int* seq_shared;
    float* part_o;                // [B, nH, slots, hd]
    float* part_ml;               // [B, nH, slots, 2]
    float* scores;                // [B, nH, reach] or null
    float* weights;               // [pages, nKV, GL_PAGE] or null
    float* given;                 // [B, nKV, reach]: where sequences may hold a page together, what each gives its positions; or null
    int B, nH, nKV, max_pages, n_pages, n_items, splits, slots, chunks, reach, hd;
    int early, held, joined;      // set by the launchers
};

enum { SF_OWN = 0, SF_SHARED = 1 };

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
    int* row_seq = (int*)(halves + 8 * SF_MAX_HD);                 // [8] sequence, head, last position seen
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
    const int total = a.seq_ctx[table] + 1;                       // positions of the sequence that were written
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
        const int at = b >= 0 && a.seq_row ? a.seq_row[b] : b;
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
            a.part_o[(((size_t)row_seq[r] * a.nH + row_head[r]) * a.slots + slot) * hd + d] = v;
        }
        if (tid == 0) {
            float* ml = a.part_ml + ((size_t)row_seq[r] * a.nH + row_head[r]) * 2 * a.slots + 2 * slot;
            ml[0] = row_m[r];
            ml[1] = l;
        }
    }
}

// The spans of a sequence put together, as in attention_spans.cu: blockIdx = (x, key/value head, sequence), first the blocks of a thousand
// positions each, then a block a query head for its output.
#define SF_JOIN_THREADS 256
#define SF_JOIN_KEYS 4
template <bool GIVEN>
__global__ void __launch_bounds__(SF_JOIN_THREADS)
span_f32_join_kernel(SpanF32Args a, int shares) {
    extern __shared__ __align__(16) float sf[];                    // [G][2]: maximum, sum
    __shared__ float sums[SF_JOIN_THREADS];
    const int b = blockIdx.z, g = blockIdx.y, G = a.nH / a.nKV, tid = threadIdx.x, lane = tid & 31;
    gl_grid_wait();
    gl_grid_launch_dependents();
    if (a.seq_qlen && a.seq_qlen[b] <= 0) return;
    const int n = (a.seq_shared ? a.seq_shared[2 * b + 1] : 0) + a.splits, own = (int)blockIdx.x - shares;
    const int pos = a.seq_ctx[b], most = min(pos + 1, a.reach), j0 = (int)blockIdx.x * SF_JOIN_THREADS * SF_JOIN_KEYS + tid;
    if (own < 0 && j0 - tid >= most) return;
    for (int i = own < 0 ? tid >> 5 : own + (tid >> 5) * G; i < G; i += SF_JOIN_THREADS / 32) {      // (all heads, or the block's)
        const float* ml = a.part_ml + ((size_t)b * a.nH + g * G + i) * a.slots * 2;
        float m = -INFINITY, l = 0.f;
        for (int s = lane; s < n; s += 32) m = fmaxf(m, ml[2 * s]);
        m = gl_warp_max(m);
        for (int s = lane; s < n; s += 32) l = fmaf(sf_factor(ml[2 * s], m), ml[2 * s + 1], l);
        l = gl_warp_sum(l);
        if (lane == 0) { sf[2 * i] = m; sf[2 * i + 1] = l; }
    }
    __syncthreads();
    if (own >= 0) {
        const size_t at = ((size_t)b * a.nH + g * G + own) * a.slots;
        const float m = sf[2 * own], l = sf[2 * own + 1];
        const int per = SF_JOIN_THREADS / a.hd, first = tid / a.hd, d = tid - first * a.hd;          // (heads of up to 256)
        float o = 0.f;
        if (first < per) {
#pragma unroll 8
            for (int s = first; s < n; s += per) o = fmaf(sf_factor(a.part_ml[(at + s) * 2], m), a.part_o[(at + s) * a.hd + d], o);
        }
        sums[tid] = o;
        __syncthreads();
        if (tid < a.hd) {
            for (int k = 1; k < per; ++k) o += sums[k * a.hd + tid];
            a.out[((size_t)(a.seq_row ? a.seq_row[b] : b) * a.nH + g * G + own) * a.hd + tid] = l == 0.f ? 0.f : o / l;
        }
        return;
    }
    float given[SF_JOIN_KEYS];
    int page[SF_JOIN_KEYS];
#pragma unroll
    for (int u = 0; u < SF_JOIN_KEYS; ++u) {
        const int j = j0 + u * SF_JOIN_THREADS;
        given[u] = 0.f;
        page[u] = !GIVEN && j < most ? a.pages[(size_t)b * a.max_pages + j / GL_PAGE] : 0;
    }
    const float* sc = a.scores + ((size_t)b * a.nH + g * G) * a.reach + j0;
#pragma unroll 4
    for (int i = 0; i < G; ++i) {
        const float m = sf[2 * i], l = sf[2 * i + 1];
#pragma unroll
        for (int u = 0; u < SF_JOIN_KEYS; ++u)
            if (j0 + u * SF_JOIN_THREADS < most) given[u] += expf(sc[(size_t)i * a.reach + u * SF_JOIN_THREADS] - m) / l;
    }
#pragma unroll
    for (int u = 0; u < SF_JOIN_KEYS; ++u) {
        const int j = j0 + u * SF_JOIN_THREADS;
        if (j >= most) return;
        float* w = GIVEN ? a.given + ((size_t)b * a.nKV + g) * a.reach + j
                         : a.weights + ((size_t)gl_checked(page[u], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + j % GL_PAGE;
        if (!GIVEN && j < pos) atomicAdd(w, given[u]);             // (one addition a position: no two sequences share it)
        else *w = given[u];
    }
}

// ---------------------------------------------------------------------------
// Heads of whole 16-byte pieces: keys and values go from the cache straight to registers.  Eight lanes take a key (a lane CP pieces of it),
// so a warp takes four at a time and has 2 UN of their pieces' rows under way; no barrier stands between two keys.  With R rows
// the eight lanes' shares of R products are added up and dealt out in one exchange, so that a lane ends with the whole score of
// row ``lane mod R`` and takes its power alone.  Each of a warp's four groups of lanes has a softmax of its own; they meet at the end of
// the span, then the warps, then the blocks of a cluster (as in attention_spans.cu).  Bound by latency at the sizes that 32 bits serve:
// twelve sequences on two texts of 1,024 tokens, 32 heads of 64, 19 us; four of 50 to 700 positions with weights, 11 us.
// ---------------------------------------------------------------------------
#define ST_WARPS 4
// loads that stay behind the wait before them (what another kernel wrote meanwhile)
__device__ __forceinline__ float2 st_read(const float2* p) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float4 st_read(const float4* p) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}
// the sum over the group's eight lanes of v[r], r = lane mod R, in every lane
template <int R>
__device__ __forceinline__ float st_deal(float (&v)[R], int lane) {
    int n = R;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        if (n > 1) {                                               // hand over half the rows, take the partner's share of the other half
            n >>= 1;
            const bool up = lane & n;
#pragma unroll
            for (int i = 0; i < R / 2; ++i)
                if (i < n) {
                    const float give = up ? v[i] : v[i + n];
                    v[i] = (up ? v[i + n] : v[i]) + __shfl_xor_sync(0xffffffffu, give, n);
                }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], o == 4 ? 4 : (R == 2 ? 2 * o : R == 4 ? 4 : o));
        }
    }
    return v[0];
}

template <int CP, int R, int MODE>
__global__ void __launch_bounds__(32 * ST_WARPS)
stream_f32_kernel(SpanF32Args a) {
    extern __shared__ __align__(16) float sf[];
    constexpr int UN = CP * R <= 4 ? 4 : 2;                        // keys of a group under way
    const int hd = a.hd, G = a.nH / a.nKV, pieces = hd >> 2;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane & 7, grp = lane >> 3;
    // shared memory: what the warps found [4][R][hd], [4][R][2]; the block's result [R][hd], [R][2]; scores kept; factors of the parts
    float* o_w = sf;
    float* ml_w = o_w + ST_WARPS * R * hd;
    float* fin_o = ml_w + ST_WARPS * R * 2;
    float* fin_ml = fin_o + R * hd;
    float* held = fin_ml + 2 * R;
    if (!a.early) gl_grid_wait();
    gl_grid_launch_dependents();

    int g, rows, p_begin, p_end, slot, table;
    int seq[R], head[R], least = 0x7fffffff;
    if (MODE == SF_SHARED) {
        const int* it = a.items + 6 * blockIdx.x;
        g = blockIdx.y;
        rows = it[2]; p_begin = it[3]; p_end = it[4]; slot = it[5];
        table = a.order[it[0]];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = it[1] + min(r, rows - 1);
            seq[r] = a.order[it[0] + i / G];
            head[r] = g * G + i % G;
            least = min(least, a.seq_ctx[seq[r]]);
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
        least = pos;
#pragma unroll
        for (int r = 0; r < R; ++r) { seq[r] = b; head[r] = g * G + h0 + min(r, rows - 1); }
    }
    const int total = a.seq_ctx[table] + 1, mine = sub % R;        // mine: the row whose softmax this lane keeps
    int last = least;
    if (MODE == SF_SHARED) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r == mine) last = a.seq_ctx[seq[r]];
    }
    float q[R][CP * 4], o[R][CP * 4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float* src = a.q + ((size_t)(MODE != SF_SHARED && a.seq_row ? a.seq_row[seq[r]] : seq[r]) * a.nH + head[r]) * hd;
#pragma unroll
        for (int c = 0; c < CP; ++c) {
            const float4 v = c * 8 + sub < pieces ? *(const float4*)(src + 4 * (c * 8 + sub)) : make_float4(0.f, 0.f, 0.f, 0.f);
            q[r][4 * c] = v.x; q[r][4 * c + 1] = v.y; q[r][4 * c + 2] = v.z; q[r][4 * c + 3] = v.w;
            o[r][4 * c] = o[r][4 * c + 1] = o[r][4 * c + 2] = o[r][4 * c + 3] = 0.f;
        }
    }
    float m = -INFINITY, l = 0.f;                                  // of row ``mine`` over this group's keys
    const int* pg = a.pages + (size_t)table * a.max_pages;
    // warps take runs of 4 UN keys in turn, group by group of lanes
    constexpr int RUN = 4 * UN;
    const int k_end = min(p_end * GL_PAGE, MODE == SF_SHARED ? p_end * GL_PAGE : total);
    for (int j0 = p_begin * GL_PAGE + warp * RUN; j0 < k_end; j0 += ST_WARPS * RUN) {
        const size_t at = (((size_t)gl_checked(pg[j0 / GL_PAGE], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + j0 % GL_PAGE) * hd;
        float4 k[UN][CP], v[UN][CP];
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int c = 0; c < CP; ++c) {
                const bool ok = j0 + 4 * u + grp < k_end && c * 8 + sub < pieces;
                const size_t off = at + (size_t)(4 * u + grp) * hd + 4 * (c * 8 + sub);
                k[u][c] = ok ? *(const float4*)(a.k_cache + off) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int c = 0; c < CP; ++c) {
                const bool ok = j0 + 4 * u + grp < k_end && c * 8 + sub < pieces;
                const size_t off = at + (size_t)(4 * u + grp) * hd + 4 * (c * 8 + sub);
                v[u][c] = ok ? *(const float4*)(a.v_cache + off) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        float s[UN], m_new = m;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            float part[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float x = 0.f;
#pragma unroll
                for (int c = 0; c < CP; ++c)
                    x = fmaf(k[u][c].x, q[r][4 * c], fmaf(k[u][c].y, q[r][4 * c + 1], fmaf(k[u][c].z, q[r][4 * c + 2], fmaf(k[u][c].w, q[r][4 * c + 3], x))));
                part[r] = x;
            }
            s[u] = st_deal<R>(part, lane);
            const int j = j0 + 4 * u + grp;
            if (MODE == SF_OWN && a.weights && sub < rows && j < k_end) {
                if (!a.scores) { if (j - p_begin * GL_PAGE < a.held) held[sub * a.held + j - p_begin * GL_PAGE] = s[u]; }
                else if (j < a.reach) {
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        if (r == sub) a.scores[((size_t)table * a.nH + head[r]) * a.reach + j] = s[u];
                }
            }
            if (j >= k_end || j > last) s[u] = -INFINITY;
            m_new = fmaxf(m_new, s[u]);
        }
        const float mu = m_new == -INFINITY ? 0.f : m_new, corr = sf_factor(m, m_new);
        l *= corr;
#pragma unroll
        for (int u = 0; u < UN; ++u) { s[u] = expf(s[u] - mu); l += s[u]; }
        if (__any_sync(0xffffffffu, m != m_new)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float c = __shfl_sync(0xffffffffu, corr, (lane & 24) + r);
#pragma unroll
                for (int i = 0; i < CP * 4; ++i) o[r][i] *= c;
            }
        }
        m = m_new;
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float w = __shfl_sync(0xffffffffu, s[u], (lane & 24) + r);
#pragma unroll
                for (int c = 0; c < CP; ++c) {
                    o[r][4 * c] = fmaf(w, v[u][c].x, o[r][4 * c]); o[r][4 * c + 1] = fmaf(w, v[u][c].y, o[r][4 * c + 1]);
                    o[r][4 * c + 2] = fmaf(w, v[u][c].z, o[r][4 * c + 2]); o[r][4 * c + 3] = fmaf(w, v[u][c].w, o[r][4 * c + 3]);
                }
            }
    }
    // the warp's four groups
#pragma unroll
    for (int x = 8; x < 32; x <<= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, x), ol = __shfl_xor_sync(0xffffffffu, l, x), m_new = fmaxf(m, om);
        const float f = sf_factor(m, m_new), of = sf_factor(om, m_new);
        l = l * f + ol * of;
        m = m_new;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float fr = __shfl_sync(0xffffffffu, f, (lane & 24) + r), ofr = __shfl_sync(0xffffffffu, of, (lane & 24) + r);
#pragma unroll
            for (int i = 0; i < CP * 4; ++i) o[r][i] = o[r][i] * fr + __shfl_xor_sync(0xffffffffu, o[r][i], x) * ofr;
        }
    }
    if (lane < R) { ml_w[(warp * R + lane) * 2] = m; ml_w[(warp * R + lane) * 2 + 1] = l; }
    if (grp == 0)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < CP; ++c)
                if (c * 8 + sub < pieces)
                    *(float4*)(o_w + (warp * R + r) * hd + 4 * (c * 8 + sub)) = make_float4(o[r][4 * c], o[r][4 * c + 1], o[r][4 * c + 2], o[r][4 * c + 3]);
    __syncthreads();
    const bool join = MODE == SF_OWN && a.joined;
    for (int i = tid; i < rows * pieces; i += 32 * ST_WARPS) {
        const int r = i / pieces, c = i - r * pieces;
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < ST_WARPS; ++w) mm = fmaxf(mm, ml_w[(w * R + r) * 2]);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < ST_WARPS; ++w) {
            const float f = sf_factor(ml_w[(w * R + r) * 2], mm);
            const float4 x = *(const float4*)(o_w + (w * R + r) * hd + 4 * c);
            sum.x = fmaf(f, x.x, sum.x); sum.y = fmaf(f, x.y, sum.y); sum.z = fmaf(f, x.z, sum.z); sum.w = fmaf(f, x.w, sum.w);
            ll = fmaf(f, ml_w[(w * R + r) * 2 + 1], ll);
        }
        int b = seq[0], h = head[0];
#pragma unroll
        for (int k = 1; k < R; ++k)
            if (k == r) { b = seq[k]; h = head[k]; }
        const size_t at = ((size_t)b * a.nH + h) * a.slots + slot;
        *(float4*)(join ? fin_o + r * hd + 4 * c : a.part_o + at * hd + 4 * c) = sum;
        if (c == 0) *(float2*)(join ? fin_ml + 2 * r : a.part_ml + at * 2) = make_float2(mm, ll);
    }
    if (!join) return;
    // the blocks of the cluster, and what the shared pages gave
    cg::cluster_group cluster = cg::this_cluster();
    const int S = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int b = table, n_pre = a.seq_shared ? a.seq_shared[2 * b + 1] : 0, parts = S + n_pre, h_first = head[0];
    float* fac = held + (a.weights ? rows * a.held : 0);          // [rows][parts]: factor / sum
    float* stat = ml_w;                                            // [rows][2]: maximum, 1 / sum
    if (a.early) gl_grid_wait();
    if (S > 1) cluster.sync();
    else __syncthreads();
    for (int r = warp; r < rows; r += ST_WARPS) {
        const float2* pre = (const float2*)a.part_ml + ((size_t)b * a.nH + h_first + r) * a.slots - S;
        auto part = [&](int k) { return k < S ? ((const float2*)(S > 1 ? cluster.map_shared_rank(fin_ml, k) : fin_ml))[r] : st_read(pre + k); };
        float mm = -INFINITY, ll = 0.f;
        for (int k = lane; k < parts; k += 32) mm = fmaxf(mm, part(k).x);
        mm = gl_warp_max(mm);
        for (int k = lane; k < parts; k += 32) {
            const float2 ml = part(k);
            const float f = sf_factor(ml.x, mm);
            fac[r * parts + k] = f;
            ll = fmaf(f, ml.y, ll);
        }
        ll = gl_warp_sum(ll);
        if (lane == 0) { stat[2 * r] = mm; stat[2 * r + 1] = ll; }
    }
    __syncthreads();
    for (int i = tid * S + rank; i < rows * pieces; i += 32 * ST_WARPS * S) {
        const int r = i / pieces, c = i - r * pieces;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float f, const float4 x) {
            sum.x = fmaf(f, x.x, sum.x); sum.y = fmaf(f, x.y, sum.y); sum.z = fmaf(f, x.z, sum.z); sum.w = fmaf(f, x.w, sum.w);
        };
        for (int k = 0; k < S; ++k) add(fac[r * parts + k], ((const float4*)(S > 1 ? cluster.map_shared_rank(fin_o, k) : fin_o))[i]);
        const float4* pre = (const float4*)a.part_o + ((size_t)b * a.nH + h_first + r) * a.slots * pieces + c;
#pragma unroll 8
        for (int k = 0; k < n_pre; ++k) add(fac[r * parts + S + k], st_read(pre + (size_t)k * pieces));
        const float ll = stat[2 * r + 1];
        const float4 y = ll == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(sum.x / ll, sum.y / ll, sum.z / ll, sum.w / ll);
        *(float4*)(a.out + ((size_t)(a.seq_row ? a.seq_row[b] : b) * a.nH + h_first + r) * hd + 4 * c) = y;
    }
    if (a.weights) {
        const int n = min(min(p_end * GL_PAGE, total) - p_begin * GL_PAGE, a.held);
        for (int i = tid; i < n; i += 32 * ST_WARPS) {
            float given = 0.f;
            for (int r = 0; r < rows; ++r) given += expf(held[r * a.held + i] - stat[2 * r]) / stat[2 * r + 1];
            const int j = p_begin * GL_PAGE + i;
            if (a.given) {
                if (j < a.reach) a.given[((size_t)b * a.nKV + g) * a.reach + j] = given;
                continue;
            }
            float* w = a.weights + ((size_t)gl_checked(pg[j / GL_PAGE], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + j % GL_PAGE;
            if (j < total - 1) atomicAdd(w, given);               // (nobody waits for it; one a position, as no two sequences share it: their order is no matter)
            else *w = given;
        }
    }
    if (S > 1) cluster.sync();
}

// ---------------------------------------------------------------------------
// Runs of several tokens: the weights their positions are given (the attention itself is attention_generic.cu's).  Rows are (query, query
// head of a key/value head), queries first.  A first kernel finds each row's maximum and sum, a second walks the cache page by page:
// w[j] += sum over the rows that see j of e^(s - m) / l.  Both multiply 64 rows with a page of keys at a time: a thread has 8 x 4 of the
// scores in registers and reads 12 pieces of 16 bytes for 128 products, so the FMA pipe bounds them.  Where there are few pages and heads
// the rows are shared out among ``parts`` blocks, whose sums a last kernel adds up in order.
// ---------------------------------------------------------------------------
struct RunF32Args {
    const float* q;               // [rows, nH*hd], scaled
    const float* k_cache;         // [pages, nKV, GL_PAGE, hd]
    const int* seq_row;           // [B] first row of q
    const int* seq_qlen;          // [B]
    const int* seq_ctx;           // [B]
    const int* pages;             // [B, max_pages]
    float* ml;                    // [nH, rows, 2]: maximum, sum
    float* weights;               // [pages, nKV, GL_PAGE]
    float* sums;                  // [parts, B, nKV, reach], where parts > 1 or sequences may hold a page together (shared)
    int B, nH, nKV, max_pages, n_pages, reach, last, parts, rows, shared, hd;
};
#define RF_ROWS 64
// rows [r0, r0 + 64) of a run to the pitch of shared memory; what lies behind ``end`` or the head size is zero
__device__ __forceinline__ void rf_load_rows(float* dst, const RunF32Args& a, int row0, int g, int G, int r0, int end, int pitch) {
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
    const int vec = (a.hd & 3) == 0 ? 4 : 1, n = (a.hd + 3) / 4 * (4 / vec);
    for (int i = threadIdx.x; i < RF_ROWS * n; i += SF_THREADS) {
        const int r = i / n, c = (i - r * n) * vec, row = r0 + r, tok = row / G;
        const bool ok = row < end && c < a.hd;
        const float* src = ok ? a.q + ((size_t)(row0 + tok) * a.nH + g * G + row - tok * G) * a.hd + c : a.q;
        if (vec == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + (r * pitch + c) * 4), "l"(src), "r"(ok ? 16 : 0));
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d + (r * pitch + c) * 4), "l"(src), "r"(ok ? 4 : 0));
    }
}
// scores of rows ty + 8 i with keys tx + 16 j
__device__ __forceinline__ void rf_scores(const float* q, const float* k, int pitch, int n4, int ty, int tx, float (&s)[8][4]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    for (int c = 0; c < n4; ++c) {
        float4 x[8], y[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = *(const float4*)(q + (ty + 8 * i) * pitch + 4 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = *(const float4*)(k + (tx + 16 * j) * pitch + 4 * c);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                s[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, s[i][j]))));
    }
}
__device__ __forceinline__ void rf_load_keys(float* dst, const RunF32Args& a, int b, int g, int p, int total, int pitch) {
    const size_t page = (size_t)gl_checked(a.pages[(size_t)b * a.max_pages + p], a.n_pages, GL_BAD_PAGE);
    sf_load_page(dst, a.k_cache + (page * a.nKV + g) * GL_PAGE * a.hd, min(GL_PAGE, total - p * GL_PAGE), a.hd, pitch);
}

// blockIdx = (tile of 64 rows from the far end, key/value head, sequence)
__global__ void __launch_bounds__(SF_THREADS)
run_f32_stats_kernel(RunF32Args a) {
    extern __shared__ __align__(16) float sf[];
    const int pitch = sf_pitch(a.hd), n4 = (a.hd + 3) / 4, tile = RF_ROWS * pitch, G = a.nH / a.nKV;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, b = blockIdx.z, g = blockIdx.y;
    gl_grid_wait();
    gl_grid_launch_dependents();
    const int qlen = a.seq_qlen[b], ctx = a.seq_ctx[b], row0 = a.seq_row[b], end = qlen * G;
    const int start = a.last > 0 ? max(0, qlen - a.last) * G : 0;
    const int r0 = start + (int)(gridDim.x - 1 - blockIdx.x) * RF_ROWS;
    if (r0 >= end) return;
    const int n = (ctx + (min(r0 + RF_ROWS, end) - 1) / G) / GL_PAGE + 1, least = ctx + r0 / G;
    rf_load_rows(sf, a, row0, g, G, r0, end, pitch);
    rf_load_keys(sf + tile, a, b, g, 0, ctx + qlen, pitch);
    float m[8], l[8];
    int last[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { m[i] = -INFINITY; l[i] = 0.f; last[i] = ctx + (r0 + ty + 8 * i) / G; }
    for (int p = 0; p < n; ++p) {
        asm volatile("cp.async.commit_group;");
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        if (p + 1 < n) rf_load_keys(sf + (1 + ((p + 1) & 1)) * tile, a, b, g, p + 1, ctx + qlen, pitch);
        float s[8][4];
        rf_scores(sf, sf + (1 + (p & 1)) * tile, pitch, n4, ty, tx, s);
        const bool cut = p * GL_PAGE + GL_PAGE - 1 > least;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (cut && p * GL_PAGE + tx + 16 * j > last[i]) s[i][j] = -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
            const float mu = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum += expf(s[i][j] - mu);
            l[i] = m[i] == mx ? l[i] + sum : fmaf(l[i], expf(m[i] - mx), sum);
            m[i] = mx;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m[i], x), ol = __shfl_xor_sync(0xffffffffu, l[i], x), mx = fmaxf(m[i], om);
            l[i] = l[i] * sf_factor(m[i], mx) + ol * sf_factor(om, mx);
            m[i] = mx;
        }
        const int row = r0 + ty + 8 * i;
        if (tx == 0 && row < end) *(float2*)(a.ml + ((size_t)(g * G + row % G) * a.rows + row0 + row / G) * 2) = make_float2(m[i], l[i]);
    }
}

// blockIdx = (page and part, key/value head, sequence): the first pages, which most rows see, start first
__global__ void __launch_bounds__(SF_THREADS)
run_f32_weigh_kernel(RunF32Args a) {
    extern __shared__ __align__(16) float sf[];
    const int pitch = sf_pitch(a.hd), n4 = (a.hd + 3) / 4, tile = RF_ROWS * pitch, G = a.nH / a.nKV;
    float2* stat = (float2*)(sf + 3 * tile);                       // [2][64]: maximum, 1 / sum
    float* sums = (float*)(stat + 2 * RF_ROWS);                    // [8][64]
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, b = blockIdx.z, g = blockIdx.y, p = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    gl_grid_wait();
    gl_grid_launch_dependents();
    const int qlen = a.seq_qlen[b], ctx = a.seq_ctx[b], row0 = a.seq_row[b], end = qlen * G, total = ctx + qlen;
    if (qlen <= 0 || p * GL_PAGE >= total) return;
    const int start = max(max(0, p * GL_PAGE - ctx), a.last > 0 ? qlen - a.last : 0) * G;
    const int all = (end - start + RF_ROWS - 1) / RF_ROWS, t0 = (int)((long long)all * part / a.parts), n = (int)((long long)all * (part + 1) / a.parts) - t0;
    auto load = [&](int i) {
        const int r0 = start + (t0 + i) * RF_ROWS;
        rf_load_rows(sf + (1 + (i & 1)) * tile, a, row0, g, G, r0, end, pitch);
        if (tid < RF_ROWS) {
            const int row = r0 + tid;
            float2 v = make_float2(0.f, 1.f);
            if (row < end) v = *(const float2*)(a.ml + ((size_t)(g * G + row % G) * a.rows + row0 + row / G) * 2);
            stat[(i & 1) * RF_ROWS + tid] = make_float2(v.x, 1.0f / v.y);
        }
    };
    rf_load_keys(sf, a, b, g, p, total, pitch);
    if (n > 0) load(0);
    float given[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < n; ++i) {
        asm volatile("cp.async.commit_group;");
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        if (i + 1 < n) load(i + 1);
        float s[8][4];
        rf_scores(sf + (1 + (i & 1)) * tile, sf, pitch, n4, ty, tx, s);
        const int r0 = start + (t0 + i) * RF_ROWS;
        const bool cut = p * GL_PAGE + GL_PAGE - 1 > ctx + r0 / G || r0 + RF_ROWS > end;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 x = stat[(i & 1) * RF_ROWS + ty + 8 * k];
            const int row = r0 + ty + 8 * k, last = row < end ? ctx + row / G : -1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w = expf(s[k][j] - x.x) * x.y;
                given[j] += !cut || p * GL_PAGE + tx + 16 * j <= last ? w : 0.f;
            }
        }
    }
    asm volatile("cp.async.commit_group;");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[ty * GL_PAGE + tx + 16 * j] = given[j];
    __syncthreads();
    const int key = p * GL_PAGE + tid;
    if (tid >= GL_PAGE || key >= total) return;
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) x += sums[k * GL_PAGE + tid];
    if (a.sums) {
        if (key < a.reach) a.sums[(((size_t)part * a.B + b) * a.nKV + g) * a.reach + key] = x;
    } else {
        float* w = a.weights + ((size_t)gl_checked(a.pages[(size_t)b * a.max_pages + p], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + tid;
        if (key < ctx) atomicAdd(w, x);                            // (one addition a position: no two sequences share it)
        else *w = x;
    }
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
// rows a block takes of heads of a given size, streaming: what the registers hold
static int stream_rows(int hd) { return hd % 4 ? 8 : hd <= 64 ? 8 : hd <= 128 ? 4 : 2; }

#define ST_HELD_BYTES (56 * 1024)
#define ST_FACTOR_BYTES (24 * 1024)
template <int CP, int R, int KIND>
static int launch_stream(const SpanF32Args& a, dim3 grid, int cluster, cudaStream_t stream) {
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    const size_t fixed = sizeof(float) * (ST_WARPS + 1) * R * (a.hd + 2);
    if (!allowed[dev]) {
        if (allow_smem(stream_f32_kernel<CP, R, KIND>, sizeof(float) * (ST_WARPS + 1) * R * (32 * CP + 2) + ST_HELD_BYTES + ST_FACTOR_BYTES) != GL_OK) return GL_ERR_SMEM;
        allowed[dev] = true;
    }
    const size_t smem = fixed + (a.joined && KIND == SF_OWN ? sizeof(float) * ((a.weights ? (size_t)a.held * (a.nH / a.nKV) : 0) + R * (size_t)(a.slots + a.splits)) : 0);
    return gl_launch(stream_f32_kernel<CP, R, KIND>, grid, dim3(32 * ST_WARPS), smem, stream, cluster, a);
}
template <int CP, int MOST, int KIND>
static int launch_stream_rows(const SpanF32Args& a, int rows, dim3 grid, int cluster, cudaStream_t stream) {
    if (rows <= 1) return launch_stream<CP, 1, KIND>(a, grid, cluster, stream);
    if (rows <= 2) return launch_stream<CP, 2, KIND>(a, grid, cluster, stream);
    if constexpr (MOST >= 4)
        if (rows <= 4) return launch_stream<CP, 4, KIND>(a, grid, cluster, stream);
    if constexpr (MOST >= 8)
        if (rows <= 8) return launch_stream<CP, 8, KIND>(a, grid, cluster, stream);
    return GL_ERR_SHAPE;
}
template <int KIND>
static int launch_f32_rows(const SpanF32Args& a, int rows, dim3 grid, int cluster, cudaStream_t stream) {
    if (a.hd % 4 == 0) {
        if (a.hd <= 32) return launch_stream_rows<1, 8, KIND>(a, rows, grid, cluster, stream);
        if (a.hd <= 64) return launch_stream_rows<2, 8, KIND>(a, rows, grid, cluster, stream);
        if (a.hd <= 96) return launch_stream_rows<3, 4, KIND>(a, rows, grid, cluster, stream);
        if (a.hd <= 128) return launch_stream_rows<4, 4, KIND>(a, rows, grid, cluster, stream);
        if (a.hd <= 192) return launch_stream_rows<6, 2, KIND>(a, rows, grid, cluster, stream);
        return launch_stream_rows<8, 2, KIND>(a, rows, grid, cluster, stream);
    }
    if (rows <= 2) return launch_f32<2, KIND>(a, grid, stream);
    return launch_f32<8, KIND>(a, grid, stream);
}

static int f32_checked(const SpanF32Args& a) {
    if (a.nH <= 0 || a.nKV <= 0 || a.nH % a.nKV || a.nKV > 65535 || a.B > 65535 || a.hd <= 0 || a.hd > SF_MAX_HD || a.max_pages <= 0) return GL_ERR_SHAPE;
    if ((((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) && a.hd % 4 == 0) return GL_ERR_ALIGN;
    return GL_OK;
}
static int f32_spans_checked(const SpanF32Args& a) {
    const int G = a.nH / a.nKV;
    if (a.splits < 1 || a.slots < 0 || (a.slots > 0 && (!a.part_o || !a.part_ml))) return GL_ERR_SHAPE;
    if (a.chunks < 1 || a.chunks > G || (long long)a.nKV * a.chunks > 65535 || (G + a.chunks - 1) / a.chunks > stream_rows(a.hd)) return GL_ERR_SHAPE;
    return (a.chunks - 1) * ((G + a.chunks - 1) / a.chunks) >= G ? GL_ERR_SHAPE : GL_OK;
}
static int launch_join(const SpanF32Args& a, cudaStream_t stream) {
    const int G = a.nH / a.nKV, shares = a.weights ? (a.reach + SF_JOIN_KEYS * SF_JOIN_THREADS - 1) / (SF_JOIN_KEYS * SF_JOIN_THREADS) : 0;
    const dim3 grid(shares + G, a.nKV, a.B);
    if (a.given) return gl_launch(span_f32_join_kernel<true>, grid, dim3(SF_JOIN_THREADS), 2 * G * sizeof(float), stream, 1, a, shares);
    return gl_launch(span_f32_join_kernel<false>, grid, dim3(SF_JOIN_THREADS), 2 * G * sizeof(float), stream, 1, a, shares);
}

// rows, joined: as for gl_attention_prefix (joined: heads of whole 16-byte pieces only)
GL_API int gl_attention_prefix_f32(const SpanF32Args* args, int rows, int joined, cudaStream_t stream) {
    SpanF32Args a = *args;
    if (a.B <= 0) return GL_OK;
    int rc = f32_checked(a);
    if (rc == GL_OK) rc = f32_spans_checked(a);
    if (rc != GL_OK) return rc;
    if (a.n_items < 0 || a.scores || a.weights || !a.seq_shared || (a.n_items > 0 && (!a.items || !a.order || rows < 1 || rows > stream_rows(a.hd) || a.slots < 1))) return GL_ERR_SHAPE;
    if (joined ? a.hd % 4 || a.splits > 8 || 8 * (long long)(a.slots + a.splits) * (int)sizeof(float) > ST_FACTOR_BYTES : a.slots < a.splits) return GL_ERR_SHAPE;
    a.early = a.held = a.joined = 0;
    if (a.n_items > 0 && (rc = launch_f32_rows<SF_SHARED>(a, rows, dim3(a.n_items, a.nKV), 1, stream)) != GL_OK) return rc;
    const int G = a.nH / a.nKV, mine = (G + a.chunks - 1) / a.chunks;
    a.joined = joined;
    a.early = joined && a.n_items > 0 && gl_pdl;
    rc = launch_f32_rows<SF_OWN>(a, mine, dim3(a.splits, a.nKV * a.chunks, a.B), joined ? a.splits : 1, stream);
    return rc != GL_OK || joined ? rc : launch_join(a, stream);
}

GL_API int gl_attention_weighed_f32(const SpanF32Args* args, cudaStream_t stream) {
    SpanF32Args a = *args;
    if (a.B <= 0) return GL_OK;
    int rc = f32_checked(a);
    if (rc == GL_OK) rc = f32_spans_checked(a);
    if (rc != GL_OK) return rc;
    if (!a.weights || a.seq_shared || a.reach <= 0) return GL_ERR_SHAPE;
    const int G = a.nH / a.nKV;
    a.early = a.held = 0;
    a.joined = !a.scores;
    if (a.joined) {
        a.held = ((a.reach + GL_PAGE - 1) / GL_PAGE + a.splits - 1) / a.splits * GL_PAGE + 4;
        if (a.hd % 4 || a.chunks > 1 || a.splits > 8 || a.slots > 0 || (long long)a.held * G * (int)sizeof(float) > ST_HELD_BYTES) return GL_ERR_SHAPE;
    } else if (a.slots < a.splits) {
        return GL_ERR_SHAPE;
    }
    rc = launch_f32_rows<SF_OWN>(a, (G + a.chunks - 1) / a.chunks, dim3(a.splits, a.nKV * a.chunks, a.B), a.joined ? a.splits : 1, stream);
    if (rc == GL_OK && !a.joined) rc = launch_join(a, stream);
    return rc != GL_OK || !a.given ? rc : launch_given_join(a, a.given, 1, 1, stream);
}

// The weights of runs of up to max_qlen tokens.
GL_API int gl_attention_weigh_runs_f32(const RunF32Args* args, int max_qlen, cudaStream_t stream) {
    const RunF32Args& a = *args;
    if (a.B <= 0 || max_qlen <= 0) return GL_OK;
    if (a.nH <= 0 || a.nKV <= 0 || a.nH % a.nKV || a.nKV > 65535 || a.B > 65535 || a.hd <= 0 || a.hd > SF_MAX_HD || a.max_pages <= 0 || a.reach <= 0 || a.last < 0) return GL_ERR_SHAPE;
    if (!a.ml || !a.weights || !a.seq_row || !a.seq_qlen || a.parts < 1 || ((a.parts > 1 || a.shared) && !a.sums)) return GL_ERR_SHAPE;
    if (((((uintptr_t)a.q | (uintptr_t)a.k_cache) & 15) && a.hd % 4 == 0) || ((uintptr_t)a.ml & 7)) return GL_ERR_ALIGN;
    const int G = a.nH / a.nKV, counted = a.last > 0 && a.last < max_qlen ? a.last : max_qlen;
    const long long tiles = ((long long)counted * G + RF_ROWS - 1) / RF_ROWS, pages = (long long)((a.reach + GL_PAGE - 1) / GL_PAGE) * a.parts;
    if (tiles > 0x7fffffffLL || pages > 0x7fffffffLL) return GL_ERR_SHAPE;
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    auto need = [](int hd) { return sizeof(float) * (3 * RF_ROWS * (size_t)sf_pitch(hd) + 4 * RF_ROWS + 8 * GL_PAGE); };
    if (!allowed[dev]) {
        if (allow_smem(run_f32_stats_kernel, need(SF_MAX_HD)) != GL_OK || allow_smem(run_f32_weigh_kernel, need(SF_MAX_HD)) != GL_OK) return GL_ERR_SMEM;
        allowed[dev] = true;
    }
    int rc = gl_launch(run_f32_stats_kernel, dim3((unsigned)tiles, a.nKV, a.B), dim3(SF_THREADS), need(a.hd), stream, 1, a);
    if (rc == GL_OK) rc = gl_launch(run_f32_weigh_kernel, dim3((unsigned)pages, a.nKV, a.B), dim3(SF_THREADS), need(a.hd), stream, 1, a);
    return rc != GL_OK || !a.sums ? rc : launch_given_join(a, a.sums, a.parts, a.shared, stream);
}
