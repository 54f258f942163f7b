// Eviction from a paged cache by the weight its positions have been given: per (layer, sequence, key/value head) the first
// and the most recent positions stay and, of those between, the ones with the largest sums; what stays moves, in order, to the
// head of the sequence's pages (or of other pages).
//
// Selection: a block a (layer, sequence, head).  The sums become whole numbers of the same order (a NaN below everything, both
// zeros the same), the m-th largest is found digit by digit with histograms (11, 11 and 10 bits), and the positions above it,
// with as many equal to it as are missing, lowest first, are written down in order: every warp counts its stretch, the counts are
// summed, every warp writes.  Counts are whole numbers, so nothing depends on the order of additions.
//
// Moving: rows of 16-byte pieces.  What stays at place i came from place kept[i] >= i, and kept grows, so in place a block walks
// forward: the places it has written lie before everything it has still to read.  A block owns a stretch of columns of all rows of
// a head, so no two blocks touch the same bytes; rows that stay where they are are not touched.  Into other pages rows are
// shared out among blocks as well.  Memory bounds it.
#include "common.cuh"

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

// blockIdx = (key/value head, sequence, layer); dynamic shared memory: the keys of ``held`` positions, or none
__global__ void __launch_bounds__(1024)
evict_select_kernel(EvictArgs a, int held) {
    extern __shared__ unsigned keys[];
    __shared__ int hist[EV_BINS];
    __shared__ int warp_sum[32], warp_eq[32];
    __shared__ int found_bin, found_above;
    const int tid = threadIdx.x, T = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = T >> 5;
    const int g = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
    gl_grid_launch_dependents();
    gl_grid_wait();
    const int n = ev_length(a, b), stay = min(n, a.keep);
    const int* pg = a.pages + (size_t)b * a.max_pages;
    const int* to = a.to + (size_t)b * a.to_pages;
    const size_t base = (size_t)layer * a.n_pages;
    auto place = [&](const int* table, int j) {
        return ((base + gl_checked(table[j / GL_PAGE], a.n_pages, GL_BAD_PAGE)) * a.nKV + g) * GL_PAGE + j % GL_PAGE;
    };
    int* kept = a.kept + (((size_t)layer * a.B + b) * a.nKV + g) * a.keep;
    if (n <= a.keep) {
        for (int i = tid; i < a.keep; i += T) kept[i] = i < n ? i : -1;
    } else {
        const int lo = a.first, hi = n - a.recent;                  // the positions to choose from
        int want = a.keep - a.first - a.recent;
        for (int i = tid; i < a.first; i += T) kept[i] = i;
        for (int i = tid; i < a.recent; i += T) kept[a.keep - a.recent + i] = hi + i;
        if (want > 0) {
            const bool in_smem = hi - lo <= held;
            if (in_smem)
                for (int j = lo + tid; j < hi; j += T) keys[j - lo] = ev_key(a.weights[place(pg, j)]);
            auto key_of = [&](int j) { return in_smem ? keys[j - lo] : ev_key(a.weights[place(pg, j)]); };
            unsigned prefix = 0, mask = 0;
            int missing = want;                                     // how many of the positions that agree with the prefix stay
#pragma unroll 1
            for (int pass = 0; pass < 3; ++pass) {
                const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
                for (int i = tid; i < EV_BINS; i += T) hist[i] = 0;
                __syncthreads();
                for (int j = lo + tid; j < hi; j += T) {
                    const unsigned k = key_of(j);
                    if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1);
                }
                __syncthreads();
                // the bin, from the top, in which the count reaches ``missing``: every thread sums a run of bins
                const int per = EV_BINS / T;                        // (T is a power of two up to 1024)
                const int top = EV_BINS - 1 - tid * per;            // its highest bin
                int mine = 0;
                for (int i = 0; i < per; ++i) mine += hist[top - i];
                int before = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, before, o);
                    if (lane >= o) before += v;
                }
                if (lane == 31) warp_sum[warp] = before;
                __syncthreads();
                int ahead = before - mine;
                for (int w = 0; w < warp; ++w) ahead += warp_sum[w];
                if (ahead < missing && ahead + mine >= missing) {
                    int i = 0;
                    while (ahead + hist[top - i] < missing) { ahead += hist[top - i]; ++i; }
                    found_bin = top - i;
                    found_above = ahead;
                }
                __syncthreads();
                prefix |= (unsigned)found_bin << shift;
                mask |= ((1u << bits) - 1) << shift;
                missing -= found_above;
                __syncthreads();
            }
            // positions above the limit stay, and the first ``missing`` equal to it
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
            int at = a.first, eq = 0;
            for (int w = 0; w < warp; ++w) {
                at += warp_sum[w] + min(warp_eq[w], max(0, missing - eq));
                eq += warp_eq[w];
            }
            for (int j = s0 + lane; j - lane < s1; j += 32) {
                const unsigned k = j < s1 ? key_of(j) : 0u;
                const unsigned eqs = __ballot_sync(0xffffffffu, j < s1 && k == prefix), below = (1u << lane) - 1;
                const bool in = j < s1 && (k > prefix || (k == prefix && eq + __popc(eqs & below) < missing));
                const unsigned ins = __ballot_sync(0xffffffffu, in);
                if (in) kept[at + __popc(ins & below)] = j;
                at += __popc(ins);
                eq += __popc(eqs);
            }
        }
    }
    __syncthreads();
    // the sums move with their positions (forward, a block's width at a time: see above)
    const bool same = a.to == a.pages;
    if (same && n <= a.keep) return;
    for (int i0 = 0; i0 < stay; i0 += T) {
        const int i = i0 + tid;
        float w = 0.f;
        int j = i;
        if (i < stay) {
            j = kept[i];
            w = a.weights[place(pg, j)];
        }
        __syncthreads();
        if (i < stay && !(same && j == i)) a.weights[place(to, i)] = w;
    }
}

// U: the piece a thread moves (16, 4 or 2 bytes).  blockIdx = (keys or values, stretch of columns, share of the rows; head; sequence and layer)
template <typename U>
__global__ void __launch_bounds__(256)
evict_move_kernel(EvictArgs a, int slices, int shares) {
    __shared__ int from;
    const int tid = threadIdx.x;
    int x = blockIdx.x;
    const int which = x & 1;
    x >>= 1;
    const int slice = x % slices, share = x / slices;
    const int g = blockIdx.y, b = blockIdx.z % a.B, layer = blockIdx.z / a.B;
    gl_grid_launch_dependents();
    gl_grid_wait();
    const int n = ev_length(a, b), stay = min(n, a.keep);
    const bool same = a.to == a.pages;
    if (same && n <= a.keep) return;
    const int units = (which ? a.v_bytes : a.k_bytes) / (int)sizeof(U);
    const int per = (units + slices - 1) / slices, u0 = slice * per, width = min(per, units - u0);
    if (width <= 0) return;
    U* cache = (U*)(which ? a.v_cache : a.k_cache) + (size_t)layer * a.n_pages * a.nKV * GL_PAGE * units + u0;
    const int* pg = a.pages + (size_t)b * a.max_pages;
    const int* to = a.to + (size_t)b * a.to_pages;
    const int* kept = a.kept + (((size_t)layer * a.B + b) * a.nKV + g) * a.keep;
    auto row = [&](const int* table, int j) {
        return cache + (((size_t)gl_checked(table[j / GL_PAGE], a.n_pages, GL_BAD_PAGE) * a.nKV + g) * GL_PAGE + j % GL_PAGE) * units;
    };
    int begin = 0, end = stay;
    if (same) {                                                    // the first row that moves: kept[i] - i never falls
        if (tid == 0) {
            int l = 0, h = stay;
            while (l < h) { const int m = (l + h) / 2; if (kept[m] > m) h = m; else l = m + 1; }
            from = l;
        }
        __syncthreads();
        begin = from;
    } else {
        const int rows = (stay + shares - 1) / shares;
        begin = share * rows;
        end = min(stay, begin + rows);
    }
    constexpr int N = 4;                                           // pieces a thread has under way
    const int step = 256 / width, lane_row = tid / width, col = tid - lane_row * width;      // (width <= 256)
    const bool active = lane_row < step;
    for (int i0 = begin; i0 < end; i0 += N * step) {
        U v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = i0 + k * step + lane_row;
            if (active && i < end) v[k] = row(pg, kept[i])[col];
        }
        if (same) __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = i0 + k * step + lane_row;
            if (active && i < end) row(to, i)[col] = v[k];
        }
    }
}

template <typename U>
static int launch_move(const EvictArgs& a, int slices, int shares, cudaStream_t stream) {
    return gl_launch(evict_move_kernel<U>, dim3(2 * slices * shares, a.nKV, a.B * a.layers), dim3(256), 0, stream, 1, a, slices, shares);
}

GL_API int gl_cache_evict(const EvictArgs* args, int sms, cudaStream_t stream) {
    const EvictArgs& a = *args;
    if (a.B <= 0 || a.layers <= 0) return GL_OK;
    if (a.nKV <= 0 || a.nKV > 65535 || (long long)a.B * a.layers > 65535 || a.keep <= 0 || a.first < 0 || a.recent < 0 || a.first + a.recent > a.keep) return GL_ERR_SHAPE;
    if (a.n_pages <= 0 || a.max_pages <= 0 || a.to_pages * GL_PAGE < (a.keep < a.max_pages * GL_PAGE ? a.keep : a.max_pages * GL_PAGE)) return GL_ERR_SHAPE;
    if (a.k_bytes <= 0 || a.v_bytes <= 0 || a.k_bytes > 4096 || a.v_bytes > 4096 || (a.k_bytes | a.v_bytes) % 2) return GL_ERR_SHAPE;
    const uintptr_t at = (uintptr_t)a.k_cache | (uintptr_t)a.v_cache | (uintptr_t)a.k_bytes | (uintptr_t)a.v_bytes;
    // a thousand positions or two a block of 256 threads; longer sequences take larger blocks
    const long long most = (long long)a.max_pages * GL_PAGE;
    const int threads = most <= 4096 ? 256 : 1024;
    const int held = (int)(most < 48 * 1024 ? most : 48 * 1024);
    static bool allowed[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return GL_ERR_DRIVER; }
    if (!allowed[dev]) {
        if (cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 48 * 1024 * 4) != cudaSuccess) {
            cudaGetLastError();
            return GL_ERR_SMEM;
        }
        allowed[dev] = true;
    }
    int rc = gl_launch(evict_select_kernel, dim3(a.nKV, a.B, a.layers), dim3(threads), (size_t)held * 4, stream, 1, a, held);
    if (rc != GL_OK) return rc;
    const bool same = a.to == a.pages;
    const long long heads = 2LL * a.layers * a.B * a.nKV;
    const int size = at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : 2, units = (a.k_bytes > a.v_bytes ? a.k_bytes : a.v_bytes) / size;
    int slices = (units + 255) / 256, shares = 1;
    if (same)
        while (heads * slices < 4LL * sms && units / (2 * slices) * size >= 32) slices *= 2;     // (pieces of 32 bytes still fill a sector)
    else
        while (heads * slices * shares < 8LL * sms && a.keep / (2 * shares) >= 32) shares *= 2;
    if (size == 16) return launch_move<uint4>(a, slices, shares, stream);
    return size == 4 ? launch_move<unsigned>(a, slices, shares, stream) : launch_move<unsigned short>(a, slices, shares, stream);
}
