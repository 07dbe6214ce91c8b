// Scores of queries against a range of rows held in 8 bits: D[r, b] = sum_i c_r[i] c_b[i] on the tensor cores (int8 x int8
// -> int32, exact), then the pair's scales and the metric.
//
// A tile is 128 held rows (the lanes of the accumulator) by up to 256 queries (its columns): a lane keeps one row, so that
// for every query a warp stores 32 results that lie next to one another.  Which side is which also serves few
// queries: 16 of them still fill all 128 lanes, and the scan is a stream of rows.
//   warp 0, one lane : copies 128-column k-blocks of row tiles (and, where the queries do not fit, of the queries) into a
//                      ring in shared memory.  A block of up to 128 queries stays in shared memory where rows have up to
//                      three k-blocks or the block is all of them (make_plan).
//   warp 1           : issues the products into one of the accumulators
//   warps 2..17      : four groups that finish the scores of an accumulator each and store them
// Waits are bounded; a wait that runs out sets VL_STATUS_TIMEOUT and ends all roles of its CTA (vl_tensor.cuh), whose results
// that are not made by then become NaN.
#include "vl_quant.cuh"
#include "vl_tensor.cuh"

namespace {

constexpr int kTileRows = 128;                 // M: held rows per tile
constexpr int kMaxQueries = 256;               // N: queries per tile, a multiple of 16
constexpr int kBlockK = 128;                   // int8 elements per k-block = one 128-byte swizzle row
constexpr int kStepK = 32;                     // elements per instruction
constexpr int kMaxStages = 12;
constexpr int kMaxAccs = 8;                    // accumulators that tiles take in turn: 512 / nb of them
constexpr int kChunk = 16;                     // accumulator columns (queries) that a finishing group takes at a time: nb is a multiple of it
constexpr int kParts = 4;                      // finishing groups of four warps, one per quarter of the lanes
constexpr int kMostResident = 128;             // queries of a block that stays in shared memory: four accumulators then
constexpr int kFinishWarps = 4 * kParts;
constexpr int kThreads = 64 + 32 * kFinishWarps;
constexpr uint32_t kTileBytes = kTileRows * kBlockK;
constexpr uint32_t kTmemCols = 2 * kMaxQueries;

// A finishing group puts 16 queries' results of a tile into a buffer in shared memory, one row of 128 for each, and copies
// the rows out.  Each group has a tile of its own wherever there are four accumulators: a group that waits for memory
// then keeps no other one waiting (200,000 x 128 x 1,024 queries: four groups on one tile 210 us, two 166, one 154; with 32
// queries at a time 161, and 34 KB less for the operands).
constexpr uint32_t kStageRow = kTileRows * 4 + 15;
constexpr uint32_t kStageBytes = (kChunk * kStageRow + 16 + 127) & ~127u;

// shared memory behind the 1024-byte aligned base: barriers, the block's queries (scales, squared lengths (hi, over), squared
// sums), the finishing groups' buffers; the operands come first
constexpr uint32_t kTailBytes = (8 * (2 * kMaxStages + 2 * kMaxAccs + 3) + 8 + 127) & ~127u;
constexpr uint32_t kOperandBytes = (227 * 1024 - 1024 - kTailBytes - kMaxQueries * 16 - kParts * kStageBytes) & ~1023u;
constexpr uint32_t kOffBars = kOperandBytes;
constexpr uint32_t kOffSlot = kOffBars + 8 * (2 * kMaxStages + 2 * kMaxAccs + 3);
constexpr uint32_t kOffAbort = kOffSlot + 4;
constexpr uint32_t kOffStop = kOffAbort + 4;
constexpr uint32_t kOffQueries = kOffBars + kTailBytes;
static_assert(kOffStop + 8 * kParts <= kOffQueries, "two words for each finishing group");
constexpr uint32_t kOffStage = kOffQueries + kMaxQueries * 16;
constexpr uint32_t kSmemBytes = kOffStage + kParts * kStageBytes + 1024;   // + slack for the alignment
static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
static_assert(3 * kBlockK * kMostResident + 4 * kTileBytes <= kOperandBytes, "blocks of rows of three k-blocks stay in shared memory");
static_assert(VL_QUANT_FEW_QUERIES == kFinishWarps, "a finishing warp for each of few queries");
static_assert(VL_QUANT_FEW_COLUMNS / kBlockK * VL_QUANT_FEW_QUERIES * kBlockK + 4 * kTileBytes <= kOperandBytes, "few queries stay in shared memory");

struct ScanArgs {
    VlQuantRows q, rows;
    const void* queries;           // up to 16 rows that the CTAs hold in 8 bits themselves (q is empty then), or null
    int64_t q_ld;
    int q_type, dim;
    bool fours;                    // groups of four elements of them are aligned
    int64_t nq, row_lo, row_hi;
    int step, lead;                // a tile's window starts at row t * step - lead and is kTileRows high (see store_rows)
    int kblocks, last_steps;       // instructions of the last k-block
    int nb, qblocks;               // queries per block (a multiple of 16) and blocks
    int groups;                    // CTAs that share a block's row tiles
    int stages, accs;
    int parts;                     // finishing warps per quarter that share a tile; kParts / parts tiles are finished side by side
    uint32_t stage_bytes;
    void* out;
    int64_t out_ld;
    int* status;
    int wait_us;                   // longest wait for another role
};

// D[tmem] (+)= A[smem] * B[smem]^T, int8 inputs, int32 accumulate
__device__ __forceinline__ void tc_mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// D int32, A and B signed 8-bit, both K-major
__device__ __forceinline__ uint32_t idesc_i8(int nb)
{
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(nb >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
}

__device__ __forceinline__ int4 ld_shared16(uint32_t at)
{
    int4 v;
    asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
template <typename T>
__device__ __forceinline__ void st_shared(uint32_t at, float r)
{
    if constexpr (sizeof(T) == 4) {
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(r) : "memory");
    } else {
        const T x = vl_from_float<T>(r);
        asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(*reinterpret_cast<const unsigned short*>(&x)) : "memory");
    }
}

// How a chunk's rows, up to 16 queries by the window of tile t, are stored by the 128 threads of a group.
//
// Memory takes whole 32-byte sectors at twice the rate of parts of them (512-byte runs with a 4-byte shift 3.06 TB/s, the
// same runs cut at sectors 4.83), and in a result whose rows are not a multiple of 32 bytes apart each query has its own
// phase, the elements f by which its first result lies behind a sector's start.  So windows overlap by a sector:
// tile t holds the results from t * step - lead on (lead = a sector's elements, step = 128 - lead), and of a query stores
// [t * step - f, (t + 1) * step - f), which are whole sectors.  Results before the first and behind the last whole
// sector of a query go one by one.  Where all rows start on sectors (SECTORS), lead is 0 and step 128.
//
// A row's place in the buffer has the alignment, modulo 16, of its place in the result, so that both take 16 bytes at once.
template <typename T, bool SECTORS>
__device__ __forceinline__ void store_rows(char* at, int64_t ld_bytes, int left, uint32_t stage, uint32_t pitch, int thread)
{
    // (streaming stores: 500,000 x 96 x 1,000 in bf16 287 to 271 us, since the rows stay in L2)
    // all whole sectors: `at` is the place of element t * step of the first query, and t * step is some sectors
    constexpr int kLanes = kTileRows * (int)sizeof(T) / 16;        // lanes that copy a row, 16 bytes each
    constexpr int kRowsPerStep = 128 / kLanes;
    const int piece = (thread % kLanes) * 16, j0 = thread / kLanes;
    if (!SECTORS && piece >= kTileRows * (int)sizeof(T) - 32) return;
    at += j0 * ld_bytes + piece;
    uint32_t from = stage + j0 * pitch + (SECTORS ? 0 : 32) + piece;
    const int64_t at_step = kRowsPerStep * ld_bytes;
    if (left >= kChunk) {
#pragma unroll
        for (int j = 0; j < kChunk; j += kRowsPerStep, at += at_step, from += kRowsPerStep * pitch) {
            const uint32_t f = SECTORS ? 0u : ((uint32_t)(uintptr_t)at - piece) & 31u;
            __stcs(reinterpret_cast<int4*>(at - f), ld_shared16(from - f));
        }
    } else {
#pragma unroll 1
        for (int j = j0; j < left; j += kRowsPerStep, at += at_step, from += kRowsPerStep * pitch) {
            const uint32_t f = SECTORS ? 0u : ((uint32_t)(uintptr_t)at - piece) & 31u;
            __stcs(reinterpret_cast<int4*>(at - f), ld_shared16(from - f));
        }
    }
}
// The first and the last tile, whose queries may begin and end inside a sector.
template <typename T>
__device__ __noinline__ void store_rows_edge(char* out, int64_t ld_bytes, int left, int64_t t, bool last, int64_t count, int step, int lead,
                                             const unsigned char* stage, uint32_t pitch, int thread)
{
    constexpr int kSector = 32 / sizeof(T), kWide = 16 / sizeof(T);
    for (int j = thread >> 3; j < left; j += 16) {
        // elements [lo, hi) of query j in this tile, of which [from, to) are whole sectors
        const int f = (int)((uint32_t)((uintptr_t)out + j * ld_bytes) & 31u) / (int)sizeof(T);
        int64_t lo = t * step - f, hi = lo + step;
        if (last) hi = count;
        int64_t from = lo, to = hi;
        if (t == 0) {
            lo = 0;
            from = f ? kSector - f : 0;
            if (from > hi) from = hi;
        }
        if (last) to = hi - ((hi + f) & (kSector - 1));
        if (to < from) to = from;
        const T* row = reinterpret_cast<const T*>(stage + j * pitch) - (t * step - lead);
        T* o = reinterpret_cast<T*>(out + j * ld_bytes);
        for (int64_t e = lo + (thread & 7); e < from; e += 8) o[e] = row[e];
        for (int64_t e = from + (thread & 7) * kWide; e < to; e += 8 * kWide) *reinterpret_cast<int4*>(o + e) = *reinterpret_cast<const int4*>(row + e);
        for (int64_t e = to + (thread & 7); e < hi; e += 8) o[e] = row[e];
    }
}

// The first of a block's tiles that a way finishes, `behind` tiles after the CTA's first: tiles are dealt to the ways in turn, across blocks.
__device__ __forceinline__ int64_t first_tile(int way, int64_t behind, int ways) { return (way - behind % ways + ways) % ways; }

// NaN as the results that a group has not made when its wait ran out: tile rt of block qb, and what comes after it.
template <typename T, bool SECTORS>
__device__ __noinline__ void store_none(const ScanArgs& a, unsigned char* stage, int qb, int64_t rt, int way, int part, int thread, int barrier)
{
    const int64_t count = a.row_hi - a.row_lo, row_tiles = (count + a.step - 1) / a.step, ld_bytes = a.out_ld * (int64_t)sizeof(T);
    const int qb0 = blockIdx.x / a.groups, qb_step = gridDim.x / a.groups, rt0 = blockIdx.x % a.groups, ways = kParts / a.parts;
    const int64_t mine = rt0 < row_tiles ? (row_tiles - rt0 + a.groups - 1) / a.groups : 0;
    const uint32_t pitch = kTileRows * sizeof(T) + (SECTORS ? 0u : (uint32_t)ld_bytes & 15u);
    for (int i = thread * 4; i < (int)kStageBytes; i += 128 * 4) *reinterpret_cast<uint32_t*>(stage + i) = 0xffffffffu;        // in every type
    barrier_sync(barrier, 128);
#pragma unroll 1
    while (qb < a.qblocks) {
        const int64_t b0 = (int64_t)qb * a.nb;
        const int here = a.nq - b0 < a.nb ? (int)(a.nq - b0) : a.nb;
#pragma unroll 1
        for (; rt < row_tiles; rt += (int64_t)ways * a.groups) {
#pragma unroll 1
            for (int c0 = part * kChunk; c0 < here; c0 += a.parts * kChunk) {
                char* out = reinterpret_cast<char*>(a.out) + (b0 + c0) * ld_bytes;
                const uint32_t off = SECTORS ? 0u : (uint32_t)(uintptr_t)out & 15u;
                store_rows_edge<T>(out, ld_bytes, here - c0 < kChunk ? here - c0 : kChunk, rt, rt + 1 == row_tiles, count, a.step, a.lead, stage + off, pitch, thread);
            }
        }
        qb += qb_step;
        rt = rt0 + first_tile(way, (qb - qb0) / qb_step * mine, ways) * a.groups;
    }
}

// Query b, by one warp, as the products read it: k-blocks of nb rows of 128 bytes, whose 16-byte pieces are swapped by
// the row's number modulo 8.
template <typename T>
__device__ __forceinline__ void hold_query(const ScanArgs& a, int b, unsigned char* at, uint32_t q_bytes, int lane, float& s, int& n)
{
    const T* x[1] = {reinterpret_cast<const T*>(a.queries) + b * a.q_ld};
    float scale[1];
    int norm[1];
    auto put = [&](int, int e, uint32_t word) {
        *reinterpret_cast<uint32_t*>(at + (e / kBlockK) * q_bytes + b * kBlockK + ((((e >> 4) ^ b) & 7) << 4) + (e & 15)) = word;
    };
    if (a.fours) vl_quant_rows<T, true, 6, 1>(x, a.dim, a.kblocks * kBlockK, lane, scale, norm, put);
    else vl_quant_rows<T, false, 1, 1>(x, a.dim, a.kblocks * kBlockK, lane, scale, norm, put);
    s = scale[0];
    n = norm[0];
}
static __device__ __noinline__ void hold_query(const ScanArgs& a, int b, unsigned char* at, uint32_t q_bytes, int lane, float& s, int& n)
{
    s = 0.0f;
    n = 0;
    if (b >= a.nq) {
        for (int e = lane * 4; e < a.kblocks * kBlockK; e += 128)
            *reinterpret_cast<uint32_t*>(at + (e / kBlockK) * q_bytes + b * kBlockK + (e & (kBlockK - 1))) = 0u;
    } else if (a.q_type == VL_TYPE_F32) {
        hold_query<float>(a, b, at, q_bytes, lane, s, n);
    } else if (a.q_type == VL_TYPE_BF16) {
        hold_query<__nv_bfloat16>(a, b, at, q_bytes, lane, s, n);
    } else {
        hold_query<__half>(a, b, at, q_bytes, lane, s, n);
    }
}

// A lane's results of a chunk: 16 queries' values are read four at a time, since shared memory feeds the products too.
template <int METRIC, bool NARROW, bool ALIKE>
__device__ __forceinline__ void finish_chunk(const uint32_t (&v)[kChunk], const float* q_scale, vl_f2 cs, vl_f2 ncs, vl_f2 hi, vl_f2 over,
                                             float (&r)[kChunk], float& least)
{
#pragma unroll
    for (int j = 0; j < kChunk; j += 4) {
        const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(q_scale + j);
        ulonglong2 q_hi = {0ull, 0ull}, q_over = {0ull, 0ull};
        if (METRIC == VL_METRIC_SQL2) {
            q_hi = *reinterpret_cast<const ulonglong2*>(q_scale + kMaxQueries + j);
            q_over = *reinterpret_cast<const ulonglong2*>(q_scale + 2 * kMaxQueries + j);
        }
        vl_quant_pair2<METRIC, NARROW, ALIKE>((int)v[j], (int)v[j + 1], s.x, q_hi.x, q_over.x, cs, ncs, hi, over, r[j], r[j + 1], least);
        vl_quant_pair2<METRIC, NARROW, ALIKE>((int)v[j + 2], (int)v[j + 3], s.y, q_hi.y, q_over.y, cs, ncs, hi, over, r[j + 2], r[j + 3], least);
    }
}
// ... one by one: rows that are not ordinary, and near rows among others
template <int METRIC, bool NARROW>
__device__ __forceinline__ float finish_pair(int dot, const float* q_scale, const VlQuantSide& held)
{
    const int n = *reinterpret_cast<const int*>(q_scale + 3 * kMaxQueries);
    const VlQuantSide q = {*q_scale, q_scale[kMaxQueries], q_scale[2 * kMaxQueries], n, vl_quant_ordinary(*q_scale, n)};
    return vl_quant_pair<METRIC, false, NARROW>(dot, q, held);
}
// ... and put over those in the buffer.  Not inlined: near rows are rare, and the loop over chunks has the registers for itself.
static __device__ __noinline__ void finish_near(int4 d0, int4 d1, int4 d2, int4 d3, const float* q_scale, float row_scale, int row_n, uint32_t at, uint32_t pitch)
{
    const VlQuantSide held = vl_quant_side<VL_METRIC_SQL2>(row_scale, row_n);
    const int dots[kChunk] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w, d2.x, d2.y, d2.z, d2.w, d3.x, d3.y, d3.z, d3.w};
#pragma unroll
    for (int j = 0; j < kChunk; ++j) st_shared<float>(at + j * pitch, finish_pair<VL_METRIC_SQL2, false>(dots[j], q_scale + j, held));
}

template <typename T, int METRIC, bool RESIDENT, bool SECTORS>
__global__ void __launch_bounds__(kThreads, 1)
quant_scan_kernel(const __grid_constant__ CUtensorMap tmap_rows, const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ ScanArgs a)
{
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* base_ptr = smem_raw + (base - raw);
    const uint32_t bar_full = base + kOffBars;
    const uint32_t bar_empty = bar_full + 8 * kMaxStages;
    const uint32_t bar_tfull = bar_empty + 8 * kMaxStages;
    const uint32_t bar_tempty = bar_tfull + 8 * kMaxAccs;
    const uint32_t bar_drain = bar_tempty + 8 * kMaxAccs;
    const uint32_t bar_q_full = bar_drain + 8;
    const uint32_t bar_q_empty = bar_q_full + 8;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(base_ptr + kOffSlot);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + kOffAbort);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // the warp's number: uniform
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMaxStages; ++s) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
        for (int b = 0; b < kMaxAccs; ++b) { mbar_init(bar_tfull + 8 * b, 1); mbar_init(bar_tempty + 8 * b, 4 * a.parts); }
        mbar_init(bar_drain, 1);
        mbar_init(bar_q_full, RESIDENT && a.queries ? kFinishWarps : 1);
        mbar_init(bar_q_empty, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void*)tmem_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int64_t count = a.row_hi - a.row_lo, row_tiles = (count + a.step - 1) / a.step;
    const int qb0 = blockIdx.x / a.groups, qb_step = gridDim.x / a.groups, rt0 = blockIdx.x % a.groups;
    const uint32_t q_bytes = (uint32_t)a.nb * kBlockK;              // one k-block of the queries
    const uint32_t ring = base + (RESIDENT ? a.kblocks * q_bytes : 0u);

    if (warp == 0 && lane == 0) {
        // ---------------- copies ----------------
        uint32_t s = 0, ph = 0, issued = 0, nres = 0;
        bool ok = true;
#pragma unroll 1
        for (int qb = qb0; qb < a.qblocks && ok; qb += qb_step) {
            if (RESIDENT && !a.queries) {
                ok = mbar_wait(bar_q_empty, (nres & 1u) ^ 1u, abort_flag, a.status, a.wait_us);
                if (!ok) break;
                ++nres;
                mbar_expect_tx(bar_q_full, a.kblocks * q_bytes);
                for (int kb = 0; kb < a.kblocks; ++kb) tma_load_2d(base + kb * q_bytes, &tmap_q, kb * kBlockK, qb * a.nb, bar_q_full);
            }
#pragma unroll 1
            for (int64_t rt = rt0; rt < row_tiles && ok; rt += a.groups) {
                const int y = (int)(a.row_lo + rt * a.step - a.lead);        // rows before the first one arrive as zeros, or are not stored
#pragma unroll 1
                for (int kb = 0; kb < a.kblocks; ++kb) {
                    ok = mbar_wait(bar_empty + 8 * s, ph ^ 1u, abort_flag, a.status, a.wait_us);
                    if (!ok) break;
                    mbar_expect_tx(bar_full + 8 * s, a.stage_bytes);
                    tma_load_2d(ring + s * a.stage_bytes, &tmap_rows, kb * kBlockK, y, bar_full + 8 * s);
                    if (!RESIDENT) tma_load_2d(ring + s * a.stage_bytes + kTileBytes, &tmap_q, kb * kBlockK, qb * a.nb, bar_full + 8 * s);
                    ++issued;
                    if (++s == (uint32_t)a.stages) { s = 0; ph ^= 1u; }
                }
            }
        }
        if (!ok) {
            // leaving early: the copies already issued still land in shared memory; wait for them
            const uint32_t open = issued < (uint32_t)a.stages ? issued : (uint32_t)a.stages;
            for (uint32_t j = 0; j < open; ++j) {
                if (s == 0) { s = a.stages; ph ^= 1u; }
                --s;
                const unsigned long long t0 = now_ns();
                while (!mbar_test(bar_full + 8 * s, ph) && now_ns() - t0 < kWaitLimitNs) __nanosleep(100);
            }
            if (RESIDENT && nres) {                                 // (queries that came by a copy)
                const unsigned long long t0 = now_ns();
                while (!mbar_test(bar_q_full, (nres - 1) & 1u) && now_ns() - t0 < kWaitLimitNs) __nanosleep(100);
            }
        }
    } else if (warp == 1) {
        // ---------------- products ----------------
        const uint32_t idesc = idesc_i8(a.nb);
        uint32_t s = 0, ph = 0, nres = 0, buf = 0, tph = 0;
        bool ok = true;
#pragma unroll 1
        for (int qb = qb0; qb < a.qblocks && ok; qb += qb_step) {
            if (RESIDENT) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar_q_full, nres & 1u, abort_flag, a.status, a.wait_us));
                if (!ok) break;
                ++nres;
            }
#pragma unroll 1
            for (int64_t rt = rt0; rt < row_tiles && ok; rt += a.groups) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar_tempty + 8 * buf, tph ^ 1u, abort_flag, a.status, a.wait_us));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + buf * a.nb;
#pragma unroll 1
                for (int kb = 0; kb < a.kblocks; ++kb) {
                    ok = __all_sync(0xffffffffu, mbar_wait(bar_full + 8 * s, ph, abort_flag, a.status, a.wait_us));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t a_desc = smem_desc_sw128(ring + s * a.stage_bytes);
                    const uint64_t b_desc = smem_desc_sw128(RESIDENT ? base + kb * q_bytes : ring + s * a.stage_bytes + kTileBytes);
                    const int steps = kb + 1 < a.kblocks ? kBlockK / kStepK : a.last_steps;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < kBlockK / kStepK; ++kk)     // 32 elements = 2 descriptor units per step
                            if (kk < steps) tc_mma_i8(d_tmem, a_desc + 2 * kk, b_desc + 2 * kk, idesc, (kb | kk) != 0);
                        tc_commit(bar_empty + 8 * s);
                        if (kb + 1 == a.kblocks) tc_commit(bar_tfull + 8 * buf);
                    }
                    __syncwarp();
                    if (++s == (uint32_t)a.stages) { s = 0; ph ^= 1u; }
                }
                if (++buf == (uint32_t)a.accs) { buf = 0; tph ^= 1u; }
            }
            if (RESIDENT && ok && elect_one()) tc_commit(bar_q_empty);
            __syncwarp();
        }
        // every product issued above must have finished before the accumulators are given back
        if (elect_one()) tc_commit(bar_drain);
        __syncwarp();
        const unsigned long long t0 = now_ns();
        while (!mbar_test(bar_drain, 0) && now_ns() - t0 < kWaitLimitNs) __nanosleep(100);
    } else if (warp >= 2) {
        // ---------------- results: one held row per lane ----------------
        const int quarter = warp & 3;                               // the TMEM lanes this warp may read
        const int ways = kParts / a.parts;                          // tiles that are finished side by side
        const int group = (warp - 2) >> 2, way = group / a.parts, part = group % a.parts;
        const int in_group = (warp - 2 - 4 * group) * 32 + lane;    // this thread among the group's 128
        const int64_t ld_bytes = a.out_ld * (int64_t)sizeof(T);
        float* q_scale = reinterpret_cast<float*>(base_ptr + kOffQueries);
        float* q_hi = q_scale + kMaxQueries;
        float* q_over = q_hi + kMaxQueries;
        int* q_n = reinterpret_cast<int*>(q_over + kMaxQueries);
        const uint32_t stage = base + kOffStage + group * kStageBytes;
        volatile int* stop = reinterpret_cast<volatile int*>(base_ptr + kOffStop) + 2 * group;        // the block and tile at which a wait ran out
        const uint32_t pitch = kTileRows * sizeof(T) + (SECTORS ? 0u : (uint32_t)ld_bytes & 15u);
        uint32_t buf = way, tph = 0;
        bool ok = true;
        while (buf >= (uint32_t)a.accs) { buf -= a.accs; tph ^= 1u; }
        // a row's scale and sum of squares are fetched one tile ahead: nothing else covers their way from memory
        auto fetch = [&](int64_t rt, float& cs, int& cn) {
            const int64_t row = a.row_lo + rt * a.step - a.lead + quarter * 32 + lane;
            const bool live = rt < row_tiles && row >= a.row_lo && row < a.row_hi;
            cs = live ? __ldg(a.rows.scales + row) : 0.0f;
            cn = live ? __ldg(a.rows.norms + row) : 0;
        };
        int64_t behind = 0;                                         // tiles of this CTA before the block's
#pragma unroll 1
        for (int qb = qb0; qb < a.qblocks; qb += qb_step) {         // all blocks even after a wait ran out: the barriers count on it
            const int64_t b0 = (int64_t)qb * a.nb;
            const int here = a.nq - b0 < a.nb ? (int)(a.nq - b0) : a.nb;      // queries behind the last one are padding
            const int64_t mine = rt0 < row_tiles ? (row_tiles - rt0 + a.groups - 1) / a.groups : 0;
            const int64_t first = first_tile(way, behind, ways);
            behind += mine;
            barrier_sync(1, 32 * kFinishWarps);
            auto keep = [&](int i, const VlQuantSide& q) {
                q_scale[i] = q.s;
                q_hi[i] = i < here ? q.hi : __int_as_float(0x7f800000);         // padding is near no row
                q_over[i] = q.over;
                q_n[i] = q.n;
            };
            if (RESIDENT && a.queries) {                            // one block, one warp for each of its 16 queries
                float s;
                int n;
                hold_query(a, warp - 2, base_ptr, q_bytes, lane, s, n);
                if (lane == 0) keep(warp - 2, vl_quant_side<METRIC>(s, n));
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_q_full);
            } else {
                for (int i = threadIdx.x - 64; i < a.nb; i += 32 * kFinishWarps) {
                    const bool there = b0 + i < a.nq;
                    keep(i, vl_quant_side<METRIC>(there ? a.q.scales[b0 + i] : 0.0f, there ? a.q.norms[b0 + i] : 0));
                }
            }
            barrier_sync(1, 32 * kFinishWarps);
            bool plain = true;
            uint32_t most = 0u, some = 0x7f7fffffu;                 // bits of the queries' largest squared length and the smallest one but 0
            for (int i = lane; i < here; i += 32) {
                plain = plain && vl_quant_ordinary(q_scale[i], q_n[i]);
                if (METRIC == VL_METRIC_SQL2) {
                    const uint32_t bits = __float_as_uint(q_hi[i]);
                    most = max(most, bits);
                    if (bits) some = min(some, bits);
                }
            }
            plain = __all_sync(0xffffffffu, plain);
            const float q_most = __uint_as_float(__reduce_max_sync(0xffffffffu, most)), q_least = __uint_as_float(__reduce_min_sync(0xffffffffu, some));
            float next_cs;
            int next_cn;
            fetch(rt0 + first * a.groups, next_cs, next_cn);
#pragma unroll 1
            for (int64_t rt = rt0 + first * a.groups; rt < row_tiles && ok; rt += (int64_t)ways * a.groups) {
                const VlQuantSide held = vl_quant_side<METRIC>(next_cs, next_cn);
                fetch(rt + (int64_t)ways * a.groups, next_cs, next_cn);
                ok = mbar_wait(bar_tfull + 8 * buf, tph, abort_flag, a.status, a.wait_us);
                ok = barrier_all(2 + group, 128, ok);               // the group goes on or ends as one
                if (!ok) {
                    stop[0] = qb;
                    stop[1] = (int)rt;
                    break;
                }
                tc_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * a.nb;
                const bool fast = plain && __all_sync(0xffffffffu, held.ordinary);
                const float cs = METRIC == VL_METRIC_COSINE ? 0.5f * held.s : (METRIC == VL_METRIC_SQL2 ? 2.0f * held.s : held.s);
                const vl_f2 cs2 = vl_f2_pack(cs, cs), ncs2 = vl_f2_pack(-cs, -cs), over2 = vl_f2_pack(held.over, held.over), hi2 = vl_f2_pack(held.hi, held.hi);
                const bool alike = METRIC != VL_METRIC_SQL2 || __all_sync(0xffffffffu, held.hi == 0.0f || vl_quant_alike(fminf(q_least, held.hi), fmaxf(q_most, held.hi)));
                const float near = alike ? __fmul_rn(kQuantNear, __fadd_rn(q_most, held.hi)) : 0.0f;          // that of no pair is larger
                const bool edge = !SECTORS && rt == 0 || rt + 1 == row_tiles;
                char* out = reinterpret_cast<char*>(a.out) + (b0 + part * kChunk) * ld_bytes;
                const uint32_t mine = stage + (quarter * 32 + lane) * (uint32_t)sizeof(T);
#pragma unroll 1
                for (int c0 = part * kChunk; c0 < a.nb; c0 += a.parts * kChunk, out += a.parts * kChunk * ld_bytes) {
                    const uint32_t off = SECTORS ? 0u : (uint32_t)(uintptr_t)out & 15u;
                    uint32_t v[kChunk];
                    tc_load16(taddr + c0, v);
                    tc_wait_ld();
                    if (c0 + a.parts * kChunk >= a.nb) {            // the tile's last columns are in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar_tempty + 8 * buf);
                    }
                    constexpr bool kNarrow = sizeof(T) == 2;
                    float r[kChunk], least = __int_as_float(0x7f800000);
                    if (fast && alike) {
                        finish_chunk<METRIC, kNarrow, true>(v, q_scale + c0, cs2, ncs2, hi2, over2, r, least);
                    } else if (fast) {
                        finish_chunk<METRIC, kNarrow, false>(v, q_scale + c0, cs2, ncs2, hi2, over2, r, least);
                    } else {
#pragma unroll
                        for (int j = 0; j < kChunk; ++j) r[j] = finish_pair<METRIC, kNarrow>((int)v[j], q_scale + c0 + j, held);
                    }
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) st_shared<T>(mine + off + j * pitch, r[j]);
                    if (METRIC == VL_METRIC_SQL2 && least <= near)
                        finish_near(make_int4(v[0], v[1], v[2], v[3]), make_int4(v[4], v[5], v[6], v[7]), make_int4(v[8], v[9], v[10], v[11]),
                                    make_int4(v[12], v[13], v[14], v[15]), q_scale + c0, held.s, held.n, mine + off, pitch);
                    barrier_sync(2 + group, 128);
                    const int left = here - c0 < kChunk ? here - c0 : kChunk;
                    if (edge) store_rows_edge<T>(out, ld_bytes, left, rt, rt + 1 == row_tiles, count, a.step, a.lead, base_ptr + (stage - base) + off, pitch, in_group);
                    else store_rows<T, SECTORS>(out + rt * a.step * (int64_t)sizeof(T), ld_bytes, left, stage + off, pitch, in_group);
                    barrier_sync(2 + group, 128);                   // the buffer is free again
                }
                buf += ways;
                while (buf >= (uint32_t)a.accs) { buf -= a.accs; tph ^= 1u; }
            }
        }
        if (!ok) store_none<T, SECTORS>(a, base_ptr + (stage - base), stop[0], stop[1], way, part, in_group, 2 + group);          // for the whole group
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    }
}

// How a scan is divided: blocks of `nb` queries, and `groups` CTAs per block that take its row tiles in turn.
struct ScanPlan {
    bool resident;
    int nb, qblocks, groups, grid, stages;
    uint32_t stage_bytes;
};

ScanPlan make_plan(int64_t nq, int kblocks, int64_t row_tiles, int sms)
{
    ScanPlan p;
    // A block's queries, at most 128, stay in shared memory beside four row stages if they are all of them, or if a row has at most
    // three k-blocks.  Otherwise both sides stream, 256 queries at a time: shared memory feeds the products (128 x 128 x 32 reads
    // 8 KB in 64 cycles, all that it gives) and 256 columns read a quarter less for each.  100,000 rows x 2,560 queries, resident
    // and streaming: 384 elements (200,000 x 2,000) 314 and 320 us; 512 220 and 227, in bf16 210 and 171; 640 274 and 266;
    // 768 336 and 307; 1024 (2,000 queries) 339 and 263.  The result's type is not looked at: at four k-blocks, where it
    // matters, streaming costs 3 % in fp32 and saves 19 % in 16 bits.
    const int fit = (int)((kOperandBytes - 4 * kTileBytes) / ((uint32_t)kblocks * kBlockK)) & ~15;
    const int most = fit < kMostResident ? fit : kMostResident;
    p.resident = kblocks <= 3 || nq <= most;
    const int cap = p.resident ? most : kMaxQueries;
    // Blocks and CTAs: the longest CTA takes `waves` blocks of ceil(row_tiles / groups) tiles, a tile costs its columns and
    // a fixed part (its rows' copies).  More blocks than needed fill SMs where there are few row tiles.
    const int64_t least = (nq + cap - 1) / cap;
    double best = 0.0;
    for (int64_t blocks = least; blocks <= least + sms && blocks <= (nq + 15) / 16; ++blocks) {
        const int nb = (int)(((nq + blocks - 1) / blocks + 15) / 16 * 16);
        if (blocks > least && (nq + nb - 1) / nb != blocks) continue;      // no such number of blocks
        int64_t groups = blocks < sms ? sms / blocks : 1;
        if (groups > row_tiles) groups = row_tiles;
        const int64_t at_once = sms / groups < blocks ? sms / groups : blocks;
        const int64_t waves = (blocks + at_once - 1) / at_once;
        const double cost = (double)(waves * ((row_tiles + groups - 1) / groups)) * (nb + 64);
        if (blocks == least || cost < best) {
            best = cost;
            p.nb = nb;
            p.groups = (int)groups;
            p.grid = (int)(groups * at_once);
        }
    }
    p.qblocks = (int)((nq + p.nb - 1) / p.nb);
    const uint32_t held = p.resident ? (uint32_t)kblocks * p.nb * kBlockK : 0u;
    p.stage_bytes = kTileBytes + (p.resident ? 0u : (uint32_t)p.nb * kBlockK);
    p.stages = (int)((kOperandBytes - held) / p.stage_bytes);
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    return p;
}

template <typename T, int METRIC>
int launch_scan(const ScanPlan& p, const CUtensorMap& rows, const CUtensorMap& q, const ScanArgs& a, cudaStream_t stream)
{
    auto kernel = a.lead == 0 ? (p.resident ? quant_scan_kernel<T, METRIC, true, true> : quant_scan_kernel<T, METRIC, false, true>)
                              : (p.resident ? quant_scan_kernel<T, METRIC, true, false> : quant_scan_kernel<T, METRIC, false, false>);
    const cudaError_t e = vl_allow_smem(kernel);
    VL_CHECK_ARG(e == cudaSuccess, "vl_quant_scores: %s", cudaGetErrorString(e));
    kernel<<<(unsigned)p.grid, kThreads, kSmemBytes, stream>>>(rows, q, a);
    VL_CHECK_LAUNCH("quant_scan_kernel");
    return 0;
}

}  // namespace

int vl_quant_scan(const void* queries, int q_type, int64_t q_ld, const VlQuantRows& q, int64_t nq, const VlQuantRows& rows, int64_t n, int dim, int code_ld, int64_t row_lo, int64_t row_hi,
                  void* out, int type, int64_t out_ld, int metric, int wait_us, int* status, cudaStream_t stream)
{
    const EncodeTiledFn encode = vl_encode_tiled();
    VL_CHECK_ARG(encode, "vl_quant_scores: cuTensorMapEncodeTiled is not available");
    const int kblocks = (code_ld + kBlockK - 1) / kBlockK;
    const int size = type == VL_TYPE_F32 ? 4 : 2;
    const bool sectors = ((uintptr_t)out | (uintptr_t)(out_ld * size)) % 32 == 0 || nq == 1 && (uintptr_t)out % 32 == 0;
    const int lead = sectors ? 0 : 32 / size, tile_step = kTileRows - lead;
    const ScanPlan p = make_plan(nq, kblocks, (row_hi - row_lo + tile_step - 1) / tile_step, vl_sm_count());
    // columns past code_ld and rows past the end arrive as zeros
    CUtensorMap map_rows, map_q;
    const cuuint64_t stride[1] = {(cuuint64_t)code_ld};
    const cuuint32_t step[2] = {1, 1};
    const cuuint64_t dim_rows[2] = {(cuuint64_t)code_ld, (cuuint64_t)n}, dim_q[2] = {(cuuint64_t)code_ld, (cuuint64_t)nq};
    const cuuint32_t box_rows[2] = {kBlockK, kTileRows}, box_q[2] = {kBlockK, (cuuint32_t)p.nb};
    CUresult cr = encode(&map_rows, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(rows.codes), dim_rows, stride, box_rows, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr == CUDA_SUCCESS && queries) map_q = map_rows;             // not used
    else if (cr == CUDA_SUCCESS)
        cr = encode(&map_q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(q.codes), dim_q, stride, box_q, step,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    VL_CHECK_ARG(cr == CUDA_SUCCESS, "vl_quant_scores: cuTensorMapEncodeTiled failed (%d)", (int)cr);
    ScanArgs a;
    a.queries = queries;
    a.q_ld = q_ld;
    a.q_type = q_type;
    a.dim = dim;
    const int q_size = q_type == VL_TYPE_F32 ? 4 : 2;
    a.fours = ((uintptr_t)queries | (uintptr_t)(q_ld * q_size)) % (4 * q_size) == 0;
    a.q = q;
    a.rows = rows;
    a.nq = nq;
    a.row_lo = row_lo;
    a.row_hi = row_hi;
    a.step = tile_step;
    a.lead = lead;
    a.kblocks = kblocks;
    a.last_steps = (code_ld - (kblocks - 1) * kBlockK + kStepK - 1) / kStepK;
    a.nb = p.nb;
    a.qblocks = p.qblocks;
    a.groups = p.groups;
    a.stages = p.stages;
    a.accs = (int)(kTmemCols / p.nb) < kMaxAccs ? (int)(kTmemCols / p.nb) : kMaxAccs;
    a.parts = a.accs >= kParts ? 1 : 2;          // no more tiles are finished side by side than there are accumulators (2: more than 128 queries, enough for both parts)
    a.stage_bytes = p.stage_bytes;
    a.out = out;
    a.out_ld = out_ld;
    a.status = status;
    a.wait_us = wait_us > 0 ? wait_us : (int)(kWaitLimitNs / 1000);
    if (metric == VL_METRIC_COSINE) return launch_scan<float, VL_METRIC_COSINE>(p, map_rows, map_q, a, stream);
    if (metric == VL_METRIC_SQL2) return launch_scan<float, VL_METRIC_SQL2>(p, map_rows, map_q, a, stream);
    if (type == VL_TYPE_F32) return launch_scan<float, VL_QUANT_PRODUCT>(p, map_rows, map_q, a, stream);
    if (type == VL_TYPE_BF16) return launch_scan<__nv_bfloat16, VL_QUANT_PRODUCT>(p, map_rows, map_q, a, stream);
    return launch_scan<__half, VL_QUANT_PRODUCT>(p, map_rows, map_q, a, stream);
}
