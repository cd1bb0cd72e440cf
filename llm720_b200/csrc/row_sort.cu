// Positions of table ids in the order of the ids: a stable sort of (id,
// position) pairs by least-significant digits of at most 8 bits.  Equal ids keep
// the order of their positions, so a sum over an id's positions has one fixed
// order.  Ids outside [0, vocab), and the one id given as `skip`, get the key
// `vocab` and end up behind all others.
//
// Up to 65,536 ids (a training batch): one launch.  A cluster of eight blocks holds all pairs in registers and
// shared memory; per digit the blocks tell one another their counts and send every pair to its place in distributed
// shared memory.  16,384 ids below 32,000: 12 us.
//
// More ids: three launches per digit.  (1) every tile of keys counts its digits, (2) every digit scans its
// counts over the tiles, (3) every tile scatters its keys; the rank of a key
// among its tile's equal digits comes from votes over the warp on top of a
// running count per warp and digit.
#include "kernels.h"
#include "row_ops.cuh"
#include "row_shift.cuh"

namespace peer {

namespace {

constexpr int SORT_THREADS = 256;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int MAX_DIGITS = 256;

__device__ __forceinline__ uint32_t source_key(const RowSortArgs& a, int64_t i) {
    const int64_t id = a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
    return (id < 0 || id >= a.vocab || id == a.skip) ? static_cast<uint32_t>(a.vocab) : static_cast<uint32_t>(id);
}

// Lanes of the warp whose digit equals this lane's: one vote per bit.  (match.any does the same in one instruction,
// but takes about a microsecond when the digits differ: a scatter of 131,072 keys took 21 us with it, 8 us without.)
__device__ __forceinline__ unsigned same_digit(uint32_t digit) {
    unsigned same = FULL_MASK;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const bool set = (digit >> b) & 1u;
        const unsigned vote = __ballot_sync(FULL_MASK, set);
        same &= set ? vote : ~vote;
    }
    return same;
}

template <bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const RowSortArgs a, const uint32_t* __restrict__ keys, int shift,
                                                                  int digits, int items, int tiles) {
    __shared__ uint32_t hist[MAX_DIGITS];
    if (!FIRST) grid_wait();
    if (FIRST && blockIdx.x == 0 && threadIdx.x < 4) a.counters[threadIdx.x] = 0;
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) hist[d] = 0u;
    __syncthreads();
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * SORT_THREADS * items;
    for (int i = 0; i < items; ++i) {
        const int64_t j = t0 + static_cast<int64_t>(i) * SORT_THREADS + threadIdx.x;
        const bool in = j < a.n;
        const uint32_t key = in ? (FIRST ? source_key(a, j) : keys[j]) : 0u;
        const uint32_t digit = (key >> shift) & (digits - 1);
        const unsigned same = same_digit(digit) & __ballot_sync(FULL_MASK, in);
        // one addition per digit and warp: a frequent id would queue up thirty-two
        if (in && (threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&hist[digit], static_cast<uint32_t>(__popc(same)));
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) a.counts[static_cast<int64_t>(d) * tiles + blockIdx.x] = hist[d];
}

// block d: exclusive scan of digit d's counts over the tiles, in place; the digit's total
__global__ void __launch_bounds__(SORT_THREADS) sort_scan_kernel(const RowSortArgs a, int tiles) {
    __shared__ uint32_t warp_total[SORT_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t* row = a.counts + static_cast<int64_t>(blockIdx.x) * tiles;
    uint32_t carry = 0u;
    grid_wait();
    for (int t0 = 0; t0 < tiles; t0 += SORT_THREADS) {
        const int t = t0 + threadIdx.x;
        const uint32_t v = t < tiles ? row[t] : 0u;
        uint32_t inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(FULL_MASK, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) warp_total[warp] = inc;
        __syncthreads();
        uint32_t before = carry, all = 0u;
#pragma unroll
        for (int i = 0; i < SORT_WARPS; ++i) {
            const uint32_t u = warp_total[i];
            if (i < warp) before += u;
            all += u;
        }
        if (t < tiles) row[t] = before + inc - v;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) a.totals[blockIdx.x] = carry;
}

template <bool FIRST>
__global__ void __launch_bounds__(SORT_THREADS) sort_scatter_kernel(const RowSortArgs a, const uint32_t* __restrict__ keys,
                                                                    const uint32_t* __restrict__ pos, uint32_t* __restrict__ keys_out,
                                                                    uint32_t* __restrict__ pos_out, int shift, int digits, int items,
                                                                    int tiles) {
    __shared__ uint32_t seen[SORT_WARPS][MAX_DIGITS];       // running count per warp and digit, then the warp's first slot
    __shared__ uint32_t warp_total[SORT_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int d = threadIdx.x; d < SORT_WARPS * MAX_DIGITS; d += SORT_THREADS) (&seen[0][0])[d] = 0u;
    __syncthreads();
    grid_wait();
    // a warp owns `items` consecutive groups of 32 keys, in order
    const int64_t w0 = (static_cast<int64_t>(blockIdx.x) * SORT_WARPS + warp) * items * 32;
    uint32_t key[16], rank[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (i >= items) break;
        const int64_t j = w0 + i * 32 + lane;
        const bool in = j < a.n;
        key[i] = in ? (FIRST ? source_key(a, j) : keys[j]) : 0u;
        const uint32_t digit = (key[i] >> shift) & (digits - 1);
        // lanes behind the last key come last in the warp: they count as one digit or another without a rank of theirs
        // ever being used, but must not lead or be counted
        const unsigned same = same_digit(digit) & __ballot_sync(FULL_MASK, in);
        const int leader = in ? __ffs(same) - 1 : lane;
        uint32_t before = 0u;
        if (in && lane == leader) {
            before = seen[warp][digit];
            seen[warp][digit] = before + __popc(same);
        }
        before = __shfl_sync(FULL_MASK, before, leader);
        rank[i] = before + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
    }
    __syncthreads();
    // first slot of digit d: all smaller digits' totals + this digit's earlier tiles + its earlier warps
    {
        const int d = threadIdx.x;
        const uint32_t v = d < digits ? a.totals[d] : 0u;
        uint32_t inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(FULL_MASK, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) warp_total[warp] = inc;
        __syncthreads();
        uint32_t first = inc - v;
#pragma unroll
        for (int i = 0; i < SORT_WARPS; ++i) if (i < warp) first += warp_total[i];
        if (d < digits) {
            first += a.counts[static_cast<int64_t>(d) * tiles + blockIdx.x];
#pragma unroll
            for (int i = 0; i < SORT_WARPS; ++i) { const uint32_t u = seen[i][d]; seen[i][d] = first; first += u; }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (i >= items) break;
        const int64_t j = w0 + i * 32 + lane;
        if (j < a.n) {
            const uint32_t slot = seen[warp][(key[i] >> shift) & (digits - 1)] + rank[i];
            keys_out[slot] = key[i];
            pos_out[slot] = FIRST ? static_cast<uint32_t>(j) : pos[j];
        }
    }
}

// ---- one cluster ------------------------------------------------------------------------------------------------
constexpr int CL_BLOCKS = 8, CL_THREADS = 1024, CL_WARPS = CL_THREADS / 32;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The two halves of a barrier that orders no memory on its way in: behind the wait every block of the cluster has started,
// and its shared memory may be accessed.
__device__ __forceinline__ void cluster_started_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_started_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// address of this block's shared memory location in another block of the cluster
__device__ __forceinline__ uint32_t remote(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void store_remote(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void store_remote(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}

struct ClusterShared {
    uint32_t seen[CL_WARPS][MAX_DIGITS];      // per warp and digit: count, then first slot
    uint32_t totals[CL_BLOCKS][MAX_DIGITS];   // every block's count per digit
    uint32_t quarter[4][MAX_DIGITS];          // this block's count per digit in eight warps each
    uint32_t first[MAX_DIGITS];               // this block's first slot per digit
    uint32_t warp_total[CL_WARPS];
};

// While one cluster sorts, the other SMs set the rows that no id names to zero.  Each block marks the ids of its rows
// in a bitmap (every block reads all ids, from L2) and writes the unmarked rows.  Launched in front of the sort, which
// starts as soon as all of these blocks run (programmatic launch; they leave room for it on every SM) and waits for
// their end only in its last instruction.
// The rows are written by bulk copies from a block of zeros in shared memory: one instruction per 4 KB, so the few warps
// that fit beside the sort are enough: 262 MB in 44 us.  The ids come through shared memory too, 8,192 at a time, because
// the registers for that many loads in flight would not fit.
constexpr int ZERO_THREADS = 256, ZERO_WORDS = 1024;      // 32 registers a thread: eight warps fit beside a block of the sort
constexpr int ZERO_BYTES = 4096, ZERO_IDS = 8192;
__global__ void __launch_bounds__(ZERO_THREADS, 8) zero_unnamed_kernel(const RowSortArgs a) {
    __shared__ uint32_t marks[ZERO_WORDS];
    __shared__ __align__(16) uint4 zeros[ZERO_BYTES / 16];
    extern __shared__ __align__(16) unsigned char staged[];      // [ZERO_IDS] as they come
    grid_release();
    const int64_t each = (a.vocab + gridDim.x - 1) / gridDim.x;
    const int64_t first = each * blockIdx.x, last = first + each < a.vocab ? first + each : a.vocab;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool vec = a.row_bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(a.zero_rows) & 15u) == 0;
    for (int i = threadIdx.x; i < ZERO_BYTES / 16; i += ZERO_THREADS) zeros[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async();                                     // the copies read them
    for (int64_t v0 = first; v0 < last; v0 += ZERO_WORDS * 32) {
        const int64_t v1 = v0 + ZERO_WORDS * 32 < last ? v0 + ZERO_WORDS * 32 : last;
        for (int i = threadIdx.x; i < ZERO_WORDS; i += ZERO_THREADS) marks[i] = 0u;
        __syncthreads();
        for (int64_t i0 = 0; i0 < a.n; i0 += ZERO_IDS) {    // a thread reads only what it copied itself
            const int count = static_cast<int>(a.n - i0 < ZERO_IDS ? a.n - i0 : ZERO_IDS);
            if (a.id_bytes == 8) {
                for (int k = threadIdx.x; k < count; k += ZERO_THREADS)
                    copy_async<8>(smem_u32(staged + k * 8), static_cast<const int64_t*>(a.ids) + i0 + k);
            } else {
                for (int k = threadIdx.x; k < count; k += ZERO_THREADS)
                    copy_async<4>(smem_u32(staged + k * 4), static_cast<const int32_t*>(a.ids) + i0 + k);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            for (int k = threadIdx.x; k < count; k += ZERO_THREADS) {
                const int64_t id = a.id_bytes == 8 ? reinterpret_cast<const int64_t*>(staged)[k] : reinterpret_cast<const int32_t*>(staged)[k];
                if (id >= v0 && id < v1 && id != a.skip) atomicOr(&marks[(id - v0) >> 5], 1u << ((id - v0) & 31));
            }
        }
        __syncthreads();
        if (vec) {
            // lane l of warp w: rows v0 + 256 j + 32 w + l, so a word of marks is one warp's
            for (int64_t v = v0 + threadIdx.x; v < v1; v += ZERO_THREADS) {
                if (marks[(v - v0) >> 5] >> ((v - v0) & 31) & 1u) continue;
                char* row = static_cast<char*>(a.zero_rows) + v * a.row_bytes;
                for (int64_t c = 0; c < a.row_bytes; c += ZERO_BYTES)
                    bulk_s2g(row + c, smem_u32(zeros), static_cast<uint32_t>(a.row_bytes - c < ZERO_BYTES ? a.row_bytes - c : ZERO_BYTES));
            }
        } else {                                             // rows of 2- or 4-byte values at any address
            for (int64_t v = v0 + warp; v < v1; v += ZERO_THREADS / 32) {
                if (marks[(v - v0) >> 5] >> ((v - v0) & 31) & 1u) continue;
                uint16_t* row = reinterpret_cast<uint16_t*>(static_cast<char*>(a.zero_rows) + v * a.row_bytes);
                for (int64_t c = lane * 8 - static_cast<int>(offset16(row) / 2); c < a.row_bytes / 2; c += 256)
                    store_granule(row, c, a.row_bytes / 2, make_uint4(0u, 0u, 0u, 0u));
            }
        }
        __syncthreads();
    }
    bulk_s2g_wait();
}

// pairs i of block b, warp w, round k, lane l:  i = ((b * CL_WARPS + w) * IT + k) * 32 + l
template <int IT>
__global__ void __cluster_dims__(CL_BLOCKS, 1, 1) __launch_bounds__(CL_THREADS, 1) sort_cluster_kernel(const RowSortArgs a, int passes,
                                                                                                       int per, uint32_t* keys_out,
                                                                                                       uint32_t* order_out) {
    cluster_started_arrive();                            // waited for in front of the first store to another block
    extern __shared__ __align__(16) unsigned char cluster_smem[];
    ClusterShared& sh = *reinterpret_cast<ClusterShared*>(cluster_smem);
    uint2* pairs = reinterpret_cast<uint2*>(cluster_smem + sizeof(ClusterShared));      // [CL_THREADS * IT]
    constexpr uint32_t EACH = CL_THREADS * IT;
    const uint32_t rank = cluster_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t local0 = warp * IT * 32 + lane, i0 = rank * EACH + local0;
    const uint32_t n = static_cast<uint32_t>(a.n), digits = 1u << per;
    if (rank == 0 && tid < 4) a.counters[tid] = 0;
    uint32_t key[IT], pos[IT], slot[IT];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        pos[k] = i0 + k * 32;
        key[k] = pos[k] < n ? source_key(a, pos[k]) : 0xffffffffu;      // behind everything, in every digit
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * per;
        for (int d = tid; d < CL_WARPS * MAX_DIGITS; d += CL_THREADS) (&sh.seen[0][0])[d] = 0u;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const uint32_t digit = (key[k] >> shift) & (digits - 1);
            const unsigned same = same_digit(digit);
            const int leader = __ffs(same) - 1;
            uint32_t before = 0u;
            if (lane == leader) {
                before = sh.seen[warp][digit];
                sh.seen[warp][digit] = before + __popc(same);
            }
            before = __shfl_sync(FULL_MASK, before, leader);
            slot[k] = before + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
        }
        __syncthreads();
        // thread (digit, quarter): the quarter's warps of one digit, turned into running sums within the quarter
        const int d = tid & (MAX_DIGITS - 1), q = tid >> 8;
        uint32_t run = 0u;
#pragma unroll
        for (int w = 0; w < CL_WARPS / 4; ++w) {
            const uint32_t v = sh.seen[q * (CL_WARPS / 4) + w][d];
            sh.seen[q * (CL_WARPS / 4) + w][d] = run;
            run += v;
        }
        sh.quarter[q][d] = run;
        __syncthreads();
        const uint32_t t0 = sh.quarter[0][d], t1 = sh.quarter[1][d], t2 = sh.quarter[2][d], t3 = sh.quarter[3][d];
        if (p == 0) cluster_started_wait();             // shared memory of a block that has not started is not there
        {                                               // this block's count of digit d to all eight blocks
            const uint32_t at = smem_u32(&sh.totals[rank][d]);
#pragma unroll
            for (int b = 0; b < CL_BLOCKS / 4; ++b) store_remote(remote(at, q * (CL_BLOCKS / 4) + b), t0 + t1 + t2 + t3);
        }
        cluster_sync();
        // first slot of a digit: smaller digits of all blocks, then this digit of earlier blocks
        uint32_t all = 0u, earlier = 0u;
        if (tid < MAX_DIGITS) {
#pragma unroll
            for (int b = 0; b < CL_BLOCKS; ++b) {
                const uint32_t v = sh.totals[b][tid];
                all += v;
                if (b < static_cast<int>(rank)) earlier += v;
            }
        }
        uint32_t inc = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(FULL_MASK, inc, o);
            if (lane >= o) inc += u;
        }
        if (tid < MAX_DIGITS && lane == 31) sh.warp_total[warp] = inc;
        __syncthreads();
        if (tid < MAX_DIGITS) {
            uint32_t f = inc - all + earlier;
#pragma unroll
            for (int w = 0; w < MAX_DIGITS / 32; ++w) f += w < warp ? sh.warp_total[w] : 0u;
            sh.first[tid] = f;
        }
        __syncthreads();
        const uint32_t base = sh.first[d] + (q > 0 ? t0 : 0u) + (q > 1 ? t1 : 0u) + (q > 2 ? t2 : 0u);
#pragma unroll
        for (int w = 0; w < CL_WARPS / 4; ++w) sh.seen[q * (CL_WARPS / 4) + w][d] += base;
        __syncthreads();
        const bool last = p + 1 == passes;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const uint32_t to = sh.seen[warp][(key[k] >> shift) & (digits - 1)] + slot[k];
            if (last) {
                if (to < n) { keys_out[to] = key[k]; order_out[to] = pos[k]; }
            } else {
                store_remote(remote(smem_u32(pairs + (to & (EACH - 1))), to / EACH), key[k], pos[k]);
            }
        }
        if (last) break;
        cluster_sync();
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const uint2 v = pairs[local0 + k * 32];
            key[k] = v.x;
            pos[k] = v.y;
        }
        // the next pass's counts are exchanged behind these reads and before the next writes to `pairs`; this pass's
        // `totals` were read before the cluster_sync above, so other blocks may write the next ones
    }
    // (the last pass writes to other blocks only before its one cluster_sync: a block may leave when it is done)
    grid_wait();                                         // the zeros of the kernel in front belong to the result
}

int bit_length(int64_t v) { int b = 0; while (v > 0) { ++b; v >>= 1; } return b; }
int items_for(int64_t n) { return n <= (1 << 19) ? 4 : 16; }      // 1,024 or 4,096 keys a tile: a tile per SM and more
int64_t round256(int64_t v) { return (v + 255) & ~static_cast<int64_t>(255); }
int64_t tiles_for(int64_t n) { const int64_t t = SORT_THREADS * items_for(n); return (n + t - 1) / t; }

}  // namespace

int64_t row_sort_bytes(int64_t n) {
    return 4 * round256(n * 4) + round256(tiles_for(n) * MAX_DIGITS * 4) + round256(MAX_DIGITS * 4) + 256;
}

void row_sort_layout(RowSortArgs& a, void* workspace) {
    char* p = static_cast<char*>(workspace);
    const int64_t each = round256(a.n * 4);
    for (int i = 0; i < 2; ++i) { a.keys[i] = reinterpret_cast<uint32_t*>(p); p += each; a.pos[i] = reinterpret_cast<uint32_t*>(p); p += each; }
    a.counts = reinterpret_cast<uint32_t*>(p);
    p += round256(tiles_for(a.n) * MAX_DIGITS * 4);
    a.totals = reinterpret_cast<uint32_t*>(p);
    a.counters = reinterpret_cast<int*>(p + round256(MAX_DIGITS * 4));
}

template <int IT>
static cudaError_t launch_cluster(RowSortArgs& a, int passes, int per, cudaStream_t s) {
    constexpr int SMEM = static_cast<int>(sizeof(ClusterShared)) + CL_THREADS * IT * 8;
    const cudaError_t e = cudaFuncSetAttribute(sort_cluster_kernel<IT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    if (a.zero_rows && IT <= 2) {                        // four and more pairs a thread: the registers of a whole SM
        const int64_t blocks = a.vocab < GRID_SMS ? a.vocab : GRID_SMS;
        const cudaError_t em = cudaFuncSetAttribute(zero_unnamed_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ZERO_IDS * 8);
        if (em != cudaSuccess) return em;
        zero_unnamed_kernel<<<static_cast<unsigned>(blocks), ZERO_THREADS, ZERO_IDS * 8, s>>>(a);
        const cudaError_t ez = launch_behind_smem(sort_cluster_kernel<IT>, dim3(CL_BLOCKS), dim3(CL_THREADS), SMEM, s, a, passes, per, a.keys[0], a.pos[0]);
        if (ez != cudaSuccess) return ez;
    } else {
        sort_cluster_kernel<IT><<<CL_BLOCKS, CL_THREADS, SMEM, s>>>(a, passes, per, a.keys[0], a.pos[0]);
    }
    a.zeroed = a.zero_rows && IT <= 2;
    a.launches = a.zeroed ? 2 : 1;
    a.sorted_keys = a.keys[0];
    a.order = a.pos[0];
    return cudaGetLastError();
}

cudaError_t launch_row_sort(RowSortArgs& a, cudaStream_t s) {
    const int bits = bit_length(a.vocab);                    // keys are 0 .. vocab
    const int passes = (bits + 7) / 8, per = (bits + passes - 1) / passes;
    const int items = items_for(a.n), tiles = static_cast<int>(tiles_for(a.n));
    const int digits = 1 << per;
    if (a.n <= CL_BLOCKS * CL_THREADS * 8) {
        const int64_t it = (a.n + CL_BLOCKS * CL_THREADS - 1) / (CL_BLOCKS * CL_THREADS);
        if (it <= 1) return launch_cluster<1>(a, passes, per, s);
        if (it <= 2) return launch_cluster<2>(a, passes, per, s);
        if (it <= 4) return launch_cluster<4>(a, passes, per, s);
        return launch_cluster<8>(a, passes, per, s);
    }
    a.launches = 3 * passes;
    for (int p = 0; p < passes; ++p) {
        const int in = (p + 1) & 1, out = p & 1, shift = p * per;
        const uint32_t *keys = a.keys[in], *pos = a.pos[in];
        const dim3 block(SORT_THREADS);
        cudaError_t e = cudaSuccess;
        if (p == 0) sort_count_kernel<true><<<tiles, SORT_THREADS, 0, s>>>(a, nullptr, shift, digits, items, tiles);
        else e = launch_behind(sort_count_kernel<false>, dim3(tiles), block, s, a, keys, shift, digits, items, tiles);
        if (e == cudaSuccess) e = launch_behind(sort_scan_kernel, dim3(digits), block, s, a, tiles);
        if (e == cudaSuccess)
            e = p == 0 ? launch_behind(sort_scatter_kernel<true>, dim3(tiles), block, s, a, keys, pos, a.keys[out], a.pos[out], shift, digits, items, tiles)
                       : launch_behind(sort_scatter_kernel<false>, dim3(tiles), block, s, a, keys, pos, a.keys[out], a.pos[out], shift, digits, items, tiles);
        if (e != cudaSuccess) return e;
        a.sorted_keys = a.keys[out];
        a.order = a.pos[out];
    }
    return cudaGetLastError();
}

}  // namespace peer
