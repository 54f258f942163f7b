// Eviction from a paged cache by the weight its positions have been given: per (layer, sequence, key/value head) the first
// and the most recent positions stay and, of those between, the ones with the largest sums; what stays moves, in order, to the
// head of the sequence's pages (or of other pages).
//
// A (layer, sequence, head) is one block's, or a cluster's.  Of short sequences every block of a cluster selects for itself; the blocks of
// long ones read and count a share of the positions each and add their histograms up in distributed shared memory.
// Selection: the sums become whole numbers of the same order (a NaN below everything, both zeros the same), the m-th largest is found
// digit by digit with histograms (11, 11 and 10 bits), and the positions above it, with as many equal to it as are missing,
// lowest first, are written down in order: every warp counts its stretch, the counts are summed, every warp writes.  Counts
// are whole numbers, so nothing depends on the order of additions.  The sums are read a page a warp, several pages under way.
//
// Moving: a row is its key's and its value's pieces of 16 bytes side by side.  What stays at place i came from place kept[i] >= i,
// and kept grows, so in place a block walks forward: the places it has written lie before everything it has still to read.  The
// blocks of a cluster share out the columns of all rows, so no two touch the same bytes, and begin when all have selected; rows
// that stay where they are are not touched.  Into other pages they share out the rows.  Memory bounds it where heads are many (24 layers
// of four sequences, 32 heads of 64: 295 us, 5.6 TB/s); of two sequences of 32,700 positions and four layers of 8 heads of 128 (72 us, 43 for the
// bytes) the first 25 us go to the three rounds of counting, before which nothing can move.
#include "common.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

struct EvictArgs {
    void* k_cache;                // [layers, pages, nKV, GL_PAGE, row bytes]
    void* v_cache;
    float* weights;               // [layers, pages, nKV, GL_PAGE]
    const int* seq_len;           // [B]
    const int* pages;             // [B, max_pages]
    const int* to;                // [B, to_pages]: where what stays goes (pages itself: in place)
    int* kept;                    // [layers, B, nKV, keep]
    int layers, B, nKV, n_pages, max_pages, to_pages, keep, recent, first, k_bytes, v_bytes;
};

#define EV_BINS 2048
__device__ __forceinline__ unsigned ev_key(float w) {
    if (w != w) return 0u;
    const unsigned u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ int ev_length(const EvictArgs& a, int b) { return min(max(0, a.seq_len[b]), a.max_pages * GL_PAGE); }

#define EV_SMALL 256                      // threads of a block for up to 4,096 positions, and beyond
#define EV_LARGE 512
#define EV_MOST (200 * 1024)              // shared memory for the keys of a sequence's sums and the positions that stay

// The sum of the counts of the warps before this one; lane w holds warp w's.
__device__ __forceinline__ int ev_before(int v, int warp, int lane) {
    int sum = lane < warp ? v : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// The positions of a sequence of n > keep that stay, in order, to ``list``.  keys: room for n, or null: the sums are read again each time.
// With T = EV_LARGE the C blocks of the cluster share the positions out: keys holds those of this block's pages (p_lo on), list is global memory.
template <int T, typename Place>
__device__ __forceinline__ void ev_select(const EvictArgs& a, int n, unsigned* keys, int* list, int (*hists)[EV_BINS], int* warp_sum, int* warp_eq, int* found,
                                          int rank, int C, Place place) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int warps = T / 32, PAGES = T == EV_SMALL ? 4 : 8;    // pages of sums a warp has under way
    constexpr bool SHARED = T == EV_LARGE;
    int lo = a.first, hi = n - a.recent;                            // the positions to choose from
    const int want = a.keep - a.first - a.recent;
    if (!SHARED || rank == 0)
        for (int i = tid; i < a.first; i += T) list[i] = i;
    if (!SHARED || rank == C - 1)
        for (int i = tid; i < a.recent; i += T) list[a.keep - a.recent + i] = hi + i;
    if (want <= 0) return;
    if (SHARED) {
        const int p0 = lo / GL_PAGE, pages = (hi + GL_PAGE - 1) / GL_PAGE - p0;
        const int mine = p0 + (int)((long long)pages * rank / C), behind = p0 + (int)((long long)pages * (rank + 1) / C);
        lo = max(lo, mine * GL_PAGE);
        hi = max(lo, min(hi, behind * GL_PAGE));
    }
    const int key0 = SHARED ? lo / GL_PAGE * GL_PAGE : 0;           // the position whose key is keys[0]
    unsigned prefix = 0, mask = 0;
    int missing = want;                                             // how many of the positions that agree with the prefix stay
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        int* hist = hists[SHARED ? pass & 1 : 0];                   // (the other one may still be read by the cluster)
        for (int i = tid; i < EV_BINS; i += T) hist[i] = 0;
        __syncthreads();
        auto count = [&](int j, unsigned k) {
            if (j >= lo && j < hi && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1);
        };
        if (pass == 0 || !keys) {
            for (int p0 = lo / GL_PAGE + warp * PAGES; p0 * GL_PAGE < hi; p0 += warps * PAGES) {
                float2 w[PAGES];
#pragma unroll
                for (int i = 0; i < PAGES; ++i)
                    if ((p0 + i) * GL_PAGE < hi) w[i] = *(const float2*)place((p0 + i) * GL_PAGE + 2 * lane);
#pragma unroll
                for (int i = 0; i < PAGES; ++i)
                    if ((p0 + i) * GL_PAGE < hi) {
                        const int j = (p0 + i) * GL_PAGE + 2 * lane;
                        const unsigned k0 = ev_key(w[i].x), k1 = ev_key(w[i].y);
                        if (keys) *(uint2*)(keys + j - key0) = make_uint2(k0, k1);
                        count(j, k0);
                        count(j + 1, k1);
                    }
            }
        } else {
            for (int j = lo + tid; j < hi; j += T) count(j, keys[j - key0]);
        }
        // the bin, from the top, in which the count reaches ``missing``: every thread sums a run of bins
        constexpr int per = EV_BINS / T;
        const int top = EV_BINS - 1 - tid * per;                    // its highest bin
        int bins[per], mine = 0;
        if (SHARED) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
#pragma unroll
            for (int i = 0; i < per; ++i) bins[i] = 0;
            for (int c = 0; c < C; ++c) {
                const int4* theirs = (const int4*)cluster.map_shared_rank(hist + top - (per - 1), c);
#pragma unroll
                for (int i = 0; i < per; i += 4) {
                    const int4 v = theirs[(per - 4 - i) / 4];
                    bins[i] += v.w; bins[i + 1] += v.z; bins[i + 2] += v.y; bins[i + 3] += v.x;
                }
            }
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < per; ++i) bins[i] = hist[top - i];
        }
#pragma unroll
        for (int i = 0; i < per; ++i) mine += bins[i];
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        if (lane == 31) warp_sum[warp] = before;
        __syncthreads();
        const int ahead_all = ev_before(lane < warps ? warp_sum[lane] : 0, warp, lane);
        int ahead = before - mine + ahead_all;
        if (ahead < missing && ahead + mine >= missing) {
            bool here = false;
#pragma unroll
            for (int i = 0; i < per; ++i) {
                if (!here && ahead + bins[i] >= missing) { here = true; found[0] = top - i; found[1] = ahead; }
                ahead += bins[i];
            }
        }
        __syncthreads();
        prefix |= (unsigned)found[0] << shift;
        mask |= ((1u << bits) - 1) << shift;
        missing -= found[1];
    }
    // positions above the limit stay, and the first ``missing`` equal to it
    auto key_of = [&](int j) { return keys ? keys[j - key0] : ev_key(*place(j)); };
    const int len = hi - lo, stretch = ((len + warps - 1) / warps + 31) & ~31;
    const int s0 = lo + warp * stretch, s1 = min(hi, s0 + stretch);
    int above = 0, equal = 0;
    for (int j = s0 + lane; j - lane < s1; j += 32) {
        const unsigned k = j < s1 ? key_of(j) : 0u;
        above += __popc(__ballot_sync(0xffffffffu, j < s1 && k > prefix));
        equal += __popc(__ballot_sync(0xffffffffu, j < s1 && k == prefix));
    }
    if (lane == 0) { warp_sum[warp] = above; warp_eq[warp] = equal; }
    __syncthreads();
    // (of the positions equal to the limit the first ``missing`` of all warps')
    int eq = ev_before(lane < warps ? warp_eq[lane] : 0, warp, lane);
    int at = a.first + ev_before(lane < warps ? warp_sum[lane] : 0, warp, lane);
    if (SHARED) {                                                   // the blocks before this one
        if (warp == warps - 1 && lane == 0) { found[2] = at - a.first + above; found[3] = eq + equal; }
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        for (int c = 0; c < rank; ++c) {
            const int* theirs = cluster.map_shared_rank(found, c);
            at += theirs[2];
            eq += theirs[3];
        }
    }
    at += min(eq, missing);
    for (int j = s0 + lane; j - lane < s1; j += 32) {
        const unsigned k = j < s1 ? key_of(j) : 0u;
        const unsigned eqs = __ballot_sync(0xffffffffu, j < s1 && k == prefix), below = (1u << lane) - 1;
        const bool in = j < s1 && (k > prefix || (k == prefix && eq + __popc(eqs & below) < missing));
        const unsigned ins = __ballot_sync(0xffffffffu, in);
        if (in) list[at + __popc(ins & below)] = j;
        at += __popc(ins);
        eq += __popc(eqs);
    }
}

// U: the piece a thread moves (16, 4 or 2 bytes).  blockIdx = (block of the cluster, key/value head, sequence and layer).  Dynamic
// shared memory: the positions that stay (``listed``: else the output itself serves) and, if there is room (``held``), the sums' keys.
template <typename U, int T>
__global__ void __launch_bounds__(T, T == EV_SMALL ? 8 : 2)
evict_kernel(EvictArgs a, int listed, int held) {
    extern __shared__ __align__(16) unsigned ev[];
    constexpr bool SHARED = T == EV_LARGE;
    __shared__ __align__(16) int hists[SHARED ? 2 : 1][EV_BINS];
    __shared__ int warp_sum[32], warp_eq[32], found[4], from;
    const int tid = threadIdx.x;
    const int C = gridDim.x, rank = blockIdx.x, g = blockIdx.y, b = blockIdx.z % a.B, layer = blockIdx.z / a.B;
    gl_grid_wait();
    gl_grid_launch_dependents();
    const int n = ev_length(a, b), stay = min(n, a.keep);
    const bool same = a.to == a.pages;
    const int* pg = a.pages + (size_t)b * a.max_pages;
    const int* to = a.to + (size_t)b * a.to_pages;
    const size_t base = (size_t)layer * a.n_pages;
    auto place = [&](const int* table, int j) {
        return ((base + gl_checked(table[j / GL_PAGE], a.n_pages, GL_BAD_PAGE)) * a.nKV + g) * GL_PAGE + j % GL_PAGE;
    };
    int* kept = a.kept + (((size_t)layer * a.B + b) * a.nKV + g) * a.keep;
    unsigned* keys = held ? ev : nullptr;
    int* list = listed ? (int*)(ev + held) : kept;
    if (n <= a.keep) {
        for (int i = tid; i < a.keep; i += T) {
            if (rank == 0) kept[i] = i < n ? i : -1;
            if (i < n && listed) list[i] = i;
        }
        if (same) return;
        if (SHARED && !listed) cg::this_cluster().sync();          // (the list is the output, which the first block has just written)
    } else {
        ev_select<T>(a, n, keys, SHARED ? kept : list, hists, warp_sum, warp_eq, found, rank, C, [&](int j) { return a.weights + place(pg, j); });
        if (SHARED) {
            cg::this_cluster().sync();                             // the list is whole, and no block reads another's memory any more
            if (listed)
                for (int i = tid; i < a.keep; i += T) list[i] = kept[i];
        }
    }
    __syncthreads();
    if (!SHARED && listed && rank == 0 && n > a.keep)
        for (int i = tid; i < a.keep; i += T) kept[i] = list[i];
    int begin = 0, end = stay;                                     // the rows, and of a row's pieces the columns, that this block moves
    const int ku = a.k_bytes / (int)sizeof(U), vu = a.v_bytes / (int)sizeof(U);
    int u0 = 0, u1 = ku + vu;
    if (same) {
        if (tid == 0) {                                            // the first row that moves: kept[i] - i never falls
            int l = 0, h = stay;
            while (l < h) { const int m = (l + h) / 2; if (list[m] > m) h = m; else l = m + 1; }
            from = l;
        }
        u0 = (int)((long long)(ku + vu) * rank / C);
        u1 = (int)((long long)(ku + vu) * (rank + 1) / C);
        if (!SHARED && C > 1) cg::this_cluster().sync();           // (the sums have been read by all before any moves)
        __syncthreads();
        begin = from;
    } else {
        begin = (int)((long long)stay * rank / C);
        end = (int)((long long)stay * (rank + 1) / C);
    }
    // The list now says where a row lies, its page's number and its place there, not which position it is.
    if (listed) {
        __syncthreads();
        for (int i = tid; i < stay; i += T) {
            const int j = list[i];
            list[i] = gl_checked(pg[j / GL_PAGE], a.n_pages, GL_BAD_PAGE) * GL_PAGE + j % GL_PAGE;
        }
        __syncthreads();
    }
    const size_t first_row = (base * a.nKV + g) * GL_PAGE;
    auto source = [&](int i) {
        const int x = list[i];
        return listed ? first_row + (size_t)(x / GL_PAGE) * a.nKV * GL_PAGE + x % GL_PAGE : place(pg, x);
    };
    // the sums: forward, a block's width at a time
    if (!same || rank == C - 1)
        for (int i0 = begin; i0 < end; i0 += T) {
            const int i = i0 + tid;
            float w = 0.f;
            if (i < end) w = a.weights[source(i)];
            if (same) __syncthreads();
            if (i < end) a.weights[place(to, i)] = w;
        }
    // Pieces a thread has under way.  Small blocks, eight an SM, move and select beside one another (24 layers of 4 x 32 heads of 64, 1,024 of
    // some 1,900 positions stay, 1.66 GB: 295 us; four blocks of eight pieces 358, eight of two 304).
    constexpr int N = T == EV_SMALL ? 4 : 8;
    U* kc = (U*)a.k_cache;
    U* vc = (U*)a.v_cache;
    for (int c0 = u0; c0 < u1; c0 += T) {
        const int width = min(T, u1 - c0), step = T / width, row = tid / width, u = c0 + tid - row * width;
        const bool active = row < step, is_v = u >= ku;
        U* cache = is_v ? vc : kc;
        const int units = is_v ? vu : ku, col = is_v ? u - ku : u;
        for (int i0 = begin; i0 < end; i0 += N * step) {
            U v[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int i = i0 + k * step + row;
                if (active && i < end) v[k] = cache[source(i) * units + col];
            }
            if (same) __syncthreads();
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int i = i0 + k * step + row;
                if (active && i < end) cache[place(to, i) * units + col] = v[k];
            }
        }
    }
}

template <typename U, int T>
static int launch_evict(const EvictArgs& a, int blocks, int listed, int held, cudaStream_t stream) {
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    if (!allowed[dev]) {
        if (cudaFuncSetAttribute(evict_kernel<U, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_MOST) != cudaSuccess) {
            cudaGetLastError();
            return GL_ERR_SMEM;
        }
        allowed[dev] = true;
    }
    return gl_launch(evict_kernel<U, T>, dim3(blocks, a.nKV, a.B * a.layers), dim3(T), ((size_t)held + (listed ? a.keep : 0)) * 4, stream, blocks, a, listed, held);
}

GL_API int gl_cache_evict(const EvictArgs* args, int sms, cudaStream_t stream) {
    const EvictArgs& a = *args;
    if (a.B <= 0 || a.layers <= 0) return GL_OK;
    if (a.nKV <= 0 || a.nKV > 65535 || (long long)a.B * a.layers > 65535 || a.keep <= 0 || a.first < 0 || a.recent < 0 || a.first + a.recent > a.keep) return GL_ERR_SHAPE;
    const long long most = (long long)a.max_pages * GL_PAGE;
    if (a.n_pages <= 0 || a.max_pages <= 0 || most > 0x7fffffff || (long long)a.n_pages * GL_PAGE > 0x7fffffff || (long long)a.to_pages * GL_PAGE < (a.keep < most ? a.keep : most)) return GL_ERR_SHAPE;
    if (a.k_bytes <= 0 || a.v_bytes <= 0 || a.k_bytes > 4096 || a.v_bytes > 4096 || (a.k_bytes | a.v_bytes) % 2) return GL_ERR_SHAPE;
    if ((uintptr_t)a.weights & 7) return GL_ERR_ALIGN;
    const uintptr_t at = (uintptr_t)a.k_cache | (uintptr_t)a.v_cache | (uintptr_t)a.k_bytes | (uintptr_t)a.v_bytes;
    // Blocks of 256 threads, several an SM, for up to 4,096 positions; larger ones beyond.  A cluster shares the rows out where there
    // are fewer heads than the machine takes blocks.
    const int threads = most <= 4096 ? EV_SMALL : EV_LARGE;
    const long long heads = (long long)a.layers * a.B * a.nKV, room = (threads == EV_SMALL ? 4LL : 2LL) * sms;
    int blocks = 1;
    while (blocks < 8 && heads * 2 * blocks <= room && a.keep / (2 * blocks) >= 32) blocks *= 2;
    // What fits in shared memory: the list of what stays, then the keys of the sums that a block reads beside it.
    const int listed = a.keep < most && 4LL * a.keep <= EV_MOST ? 1 : 0;
    if (!listed && threads == EV_SMALL) blocks = 1;                // (the list is then the output itself, which one block writes)
    const long long keys = threads == EV_SMALL ? most : ((a.max_pages + blocks - 1) / blocks + 1LL) * GL_PAGE;
    const int held = 4 * (keys + (listed ? a.keep : 0)) <= EV_MOST ? (int)keys : 0;
    if (threads == EV_SMALL) {
        if (at % 16 == 0) return launch_evict<uint4, EV_SMALL>(a, blocks, listed, held, stream);
        return at % 4 == 0 ? launch_evict<unsigned, EV_SMALL>(a, blocks, listed, held, stream) : launch_evict<unsigned short, EV_SMALL>(a, blocks, listed, held, stream);
    }
    if (at % 16 == 0) return launch_evict<uint4, EV_LARGE>(a, blocks, listed, held, stream);
    return at % 4 == 0 ? launch_evict<unsigned, EV_LARGE>(a, blocks, listed, held, stream) : launch_evict<unsigned short, EV_LARGE>(a, blocks, listed, held, stream);
}
