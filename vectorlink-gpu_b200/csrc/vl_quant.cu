// Rows held in 8 bits: written, read back, scored against queries at listed ids, and the entry points.  The scan of a
// range of rows is in vl_quant_scan.cu.
#include <initializer_list>

#include "vl_quant.cuh"

namespace {

constexpr int kMaxDim = 131072;       // 127^2 * dim has to fit 32 bits

// ---- write: one warp per row ----
// Wide fp32 rows are bound by memory, 4 bytes in and 1 out for an element: 1M x 768 in 580 us, 6.7 TB/s.  The others are not: the
// time goes by element and row, not by byte.  1M x 768 in bf16 takes 595 us, 3.9 TB/s (issue slots 74 % used, DRAM 45 %);
// 4M x 128 913 and 923 us, 2.8 and 1.7 TB/s; 4M x 64 1,013 and 1,042.  A lane next to a half takes its warp through both ways of
// vl_quant_codes, and the variants of several rows a warp spill 32 to 152 bytes under 64 registers.  To random places
// 1M x 768 takes 665 and 720 us (claims and scattered rows).
struct WriteArgs {
    const void* rows;
    int64_t m, ld;
    int dim;
    const int32_t* ids;               // place of every row, or null: first_row + r
    int64_t first_row;
    int8_t* codes;
    float* scales;
    int32_t* norms;
    int64_t n;
    int code_ld;
    int32_t* owner;                   // with ids and many rows: the last row that names a place, -1 between calls
    int* status;
};

// Which row writes a place that several rows name: the last one.
__global__ void quant_claim_kernel(const int32_t* __restrict__ ids, int64_t m, int64_t n, int32_t* __restrict__ owner)
{
    for (int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; r < m; r += (int64_t)gridDim.x * blockDim.x) {
        const int32_t place = ids[r];
        if (place >= 0 && place < n) atomicMax(owner + place, (int32_t)r);
    }
}

// A handful of rows look through the ids behind their own instead: one launch less (2.5 us of host time).  More rows would
// lose on the device (512 of 50 elements 7.0 us against 3.7 with the claims, 4,096 11.9 against 4.7).
constexpr int64_t kFewRows = 64;

template <typename T, bool VEC, int HELD, int R>
__global__ void __launch_bounds__(256, HELD > 6 ? 2 : 4) quant_write_kernel(const WriteArgs a)
{
    const int lane = threadIdx.x & 31;
    const int64_t warp0 = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int64_t nwarps = ((int64_t)gridDim.x * blockDim.x) >> 5;
    for (int64_t r0 = warp0 * R; r0 < a.m; r0 += nwarps * R) {
        const T* x[R];
        int64_t place[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t r = r0 + k;
            bool mine = r < a.m;
            place[k] = a.first_row + r;
            if (a.ids && mine) {
                place[k] = a.ids[r];
                if (place[k] < 0 || place[k] >= a.n) {
                    if (place[k] != VL_MAXINT && lane == 0) atomicOr(a.status, VL_STATUS_BAD_ID);
                    mine = false;
                } else if (a.owner) {
                    mine = *(volatile int32_t*)(a.owner + place[k]) == (int32_t)r;
                } else {
                    for (int64_t later = r + 1 + lane; later < a.m; later += 32) mine = mine && a.ids[later] != place[k];
                }
                mine = __all_sync(0xffffffffu, mine);
                if (mine && a.owner && lane == 0) a.owner[place[k]] = -1;      // rows that look later are not the owner either way
            }
            x[k] = mine ? reinterpret_cast<const T*>(a.rows) + r * a.ld : nullptr;
        }
        float scale[R];
        int norm[R];
        vl_quant_rows<T, VEC, HELD, R>(x, a.dim, a.code_ld, lane, scale, norm, [&](int k, int e, uint32_t word) {
            *reinterpret_cast<uint32_t*>(a.codes + vl_pick(place, k) * a.code_ld + e) = word;
        });
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (x[k] && lane == k) {
                a.scales[place[k]] = scale[k];
                a.norms[place[k]] = norm[k];
            }
    }
}

// ---- read: one warp per row, four elements per lane and step ----
// The codes of a warp's next row are on their way while the current one is stored (1M x 768 to fp32 610 us, 6.3 TB/s, to
// bf16 374, 6.2; without them 852 and 665; at random ids 623 and 402).  Short rows leave lanes idle: 4M x 128 in 496 us, 5.2 TB/s, and 408,
// 3.8 TB/s.
template <typename T, bool VEC, int HELD>
__global__ void __launch_bounds__(256)
quant_read_kernel(const VlQuantRows rows, int64_t n, int dim, int code_ld, const int32_t* __restrict__ ids, int64_t first_row,
                  int64_t m, T* __restrict__ out, int64_t out_ld, int* __restrict__ status)
{
    const int lane = threadIdx.x & 31;
    const int64_t warp0 = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int64_t nwarps = ((int64_t)gridDim.x * blockDim.x) >> 5;
    // a row that is none has the scale 0; its codes are row 0's, or nothing where there is no row
    auto find = [&](int64_t r, const uint32_t*& words, float& s) {
        int64_t place = r < m ? (ids ? ids[r] : first_row + r) : VL_MAXINT;
        if (place < 0 || place >= n) {
            if (place != VL_MAXINT && lane == 0) atomicOr(status, VL_STATUS_BAD_ID);
            place = -1;
        }
        words = place < 0 ? nullptr : reinterpret_cast<const uint32_t*>(rows.codes + place * code_ld);
        s = place < 0 ? 0.0f : __ldg(rows.scales + place);
    };
    auto value = [](uint32_t w, int k, float s) { return vl_from_float<T>(__fmul_rn((float)(int8_t)(w >> (8 * k)), s)); };
    auto store = [&](T* o, int e, uint32_t w, float s) {
        if (VEC && e + 4 <= dim) {
            T h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = value(w, k, s);
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(o + e) = *reinterpret_cast<const float4*>(h);
            else *reinterpret_cast<uint2*>(o + e) = *reinterpret_cast<const uint2*>(h);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (e + k < dim) o[e + k] = value(w, k, s);
        }
    };
    const uint32_t* next_words;
    float next_s;
    uint32_t next[HELD];
    auto take = [&](int64_t r) {
        find(r, next_words, next_s);
#pragma unroll
        for (int j = 0; j < HELD; ++j) next[j] = next_words && (j * 32 + lane) * 4 < dim ? __ldg(next_words + j * 32 + lane) : 0u;
    };
    take(warp0);
    for (int64_t r = warp0; r < m; r += nwarps) {
        const uint32_t* words = next_words;
        const float s = next_s;
        uint32_t w[HELD];
#pragma unroll
        for (int j = 0; j < HELD; ++j) w[j] = next[j];
        take(r + nwarps);
        T* o = out + r * out_ld;
#pragma unroll
        for (int j = 0; j < HELD; ++j)
            if ((j * 32 + lane) * 4 < dim) store(o, (j * 32 + lane) * 4, w[j], s);
        for (int e = (HELD * 32 + lane) * 4; e < dim; e += 128) store(o, e, words ? __ldg(words + (e >> 2)) : 0u, s);
    }
}

// ---- distances of listed ids ----
// Like the gather of vl_distance.cu with rows of a quarter of the size: a row is fetched by LPR lanes, J chunks of 16 codes
// each, several rows in flight per lane; a warp keeps its query's codes in registers, having rounded the query itself
// (J = 0: longer rows, chunk by chunk, the query's codes from memory).  Bound by the gather of code_ld + 4 bytes per pair
// in sectors of 32: 30,000 lists of 64 ids over 1M x 768 in 272 us (l2; cosine 311), 5.5 TB/s, with queries held before 251; x 128
// in 73 and 64 us, 3.7 and 4.2 TB/s; 10,000 lists over 200,000 x 1536 in 159 us, 6.2 TB/s, and without rows in flight (J = 0) x 2048 in 312,
// 4.2 TB/s, x 4096 in 628, 4.2 TB/s.  A step is requested when the one four (for three chunks two) ahead of it is done; five CTAs per SM for rows of two or three
// chunks (four steps of three chunks, 12 warps per SM: 325 us; ids fetched step by step: 280 to 510, as the compiler orders
// the loads).
struct ListedArgs {
    const void* queries;              // rows to hold first, or null: q has them
    int64_t q_ld;
    VlQuantRows q, rows;
    int64_t nq, n;
    int dim, code_ld;
    const int32_t* ids;               // [nq, w]
    int w, span, spans;               // a query's list is walked in `spans` runs of at most `span` ids
    float* out;
    int* status;
    bool norms;                       // sums of squared codes are needed
};

template <typename T, int LPR, int J, int METRIC, bool VEC>
__global__ void __launch_bounds__(128, J > 1 ? 5 : 8) quant_listed_kernel(const ListedArgs a)
{
    constexpr int G = 32 / LPR;                      // rows per step
    constexpr int JJ = J > 0 ? J : 1;
    constexpr int U = J == 3 ? 2 : 4;                // steps in flight
    constexpr int kUnroll = J == 1 ? 2 : 1;
    const int lane = threadIdx.x & 31, g = lane / LPR, lg = lane % LPR;
    const int chunks = a.code_ld / 16;
    const int64_t warp0 = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), nwarps = (int64_t)gridDim.x * 4;
    for (int64_t task = warp0; task < a.nq * a.spans; task += nwarps) {
        const int64_t b = task / a.spans;
        const int m_lo = (int)(task - b * a.spans) * a.span, m_hi = m_lo + a.span < a.w ? m_lo + a.span : a.w;
        int4 qc[JJ];
        float qs;
        int qn;
        if (J > 0 && a.queries) {
            // every group of LPR lanes rounds the whole query, chunk by chunk as it will meet the rows
            const T* x = reinterpret_cast<const T*>(a.queries) + b * a.q_ld;
            float largest = 0.0f;
#pragma unroll
            for (int j = 0; j < JJ; ++j) {
#pragma unroll
                for (int k = 0; k < 4; ++k) largest = vl_magnitude(largest, vl_widen<T>(vl_load4<T, VEC>(x, (lg + LPR * j) * 16 + 4 * k, a.dim)));
            }
            const VlQuantScale s = vl_quant_scale_of(vl_warp_magnitude(largest));
            int sum = 0;
            uint32_t word[4 * JJ];
            if (!s.tiny) {
#pragma unroll
                for (int k = 0; k < 4 * JJ; ++k) word[k] = vl_quant_codes(vl_widen<T>(vl_load4<T, VEC>(x, (lg + LPR * (k >> 2)) * 16 + 4 * (k & 3), a.dim)), s);
            } else {
#pragma unroll 1
                for (int at = 0; at < 4 * JJ; ++at) {
                    const uint32_t made = vl_quant_codes_tiny(vl_widen<T>(vl_load4<T, VEC>(x, (lg + LPR * (at >> 2)) * 16 + 4 * (at & 3), a.dim)), s.s);
#pragma unroll
                    for (int k = 0; k < 4 * JJ; ++k) word[k] = k == at ? made : word[k];
                }
            }
#pragma unroll
            for (int j = 0; j < JJ; ++j) qc[j] = make_int4(word[4 * j], word[4 * j + 1], word[4 * j + 2], word[4 * j + 3]);
#pragma unroll
            for (int j = 0; j < JJ; ++j) sum = __dp4a(qc[j].x, qc[j].x, __dp4a(qc[j].y, qc[j].y, __dp4a(qc[j].z, qc[j].z, __dp4a(qc[j].w, qc[j].w, sum))));
            qs = s.s;
            qn = __reduce_add_sync(0xffffffffu, g == 0 ? sum : 0);
        } else {
            const int4* c = reinterpret_cast<const int4*>(a.q.codes + b * a.code_ld);
#pragma unroll
            for (int j = 0; j < J; ++j) qc[j] = lg + LPR * j < chunks ? __ldg(c + lg + LPR * j) : make_int4(0, 0, 0, 0);
            qs = a.q.scales[b];
            qn = a.q.norms[b];
        }
        const VlQuantSide q = vl_quant_side<METRIC>(qs, qn);
        // 32 ids at a time, one per lane, which also takes that row's scale and finishes its distance; the next 32 are on
        // their way, since the rows of the steps ahead may be among them
        auto fetch = [&](int m) {
            int32_t id = m < m_hi ? __ldg(a.ids + b * a.w + m) : VL_MAXINT;
            if (id < 0 || id >= a.n) {
                if (id != VL_MAXINT) atomicOr(a.status, VL_STATUS_BAD_ID);
                id = -1;
            }
            return id;
        };
        int4 x[U][JJ];
        auto request = [&](int u, int32_t id) {
            const int4* row = reinterpret_cast<const int4*>(a.rows.codes + (int64_t)id * a.code_ld);
#pragma unroll
            for (int j = 0; j < J; ++j) x[u][j] = id >= 0 && lg + LPR * j < chunks ? __ldg(row + lg + LPR * j) : make_int4(0, 0, 0, 0);
        };
        int32_t cur = fetch(m_lo + lane);
        if (J > 0) {
#pragma unroll
            for (int u = 0; u < U; ++u) request(u, __shfl_sync(0xffffffffu, cur, u * G + g));
        }
        for (int m0 = m_lo; m0 < m_hi; m0 += 32) {
            const int32_t nxt = fetch(m0 + 32 + lane);
            const float cs = cur >= 0 ? __ldg(a.rows.scales + cur) : 0.0f;
            const int cn = cur >= 0 && a.norms ? __ldg(a.rows.norms + cur) : 0;
            int mine = 0;
#pragma unroll kUnroll
            for (int t0 = 0; t0 < 32 / G && m0 + t0 * G < m_hi; t0 += U) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    int dot = 0;
                    if (J > 0) {
#pragma unroll
                        for (int j = 0; j < JJ; ++j)
                            dot = __dp4a(x[u][j].x, qc[j].x, __dp4a(x[u][j].y, qc[j].y, __dp4a(x[u][j].z, qc[j].z, __dp4a(x[u][j].w, qc[j].w, dot))));
                        const int ahead = (t0 + u + U) * G;              // of one block of 32 for the whole warp
                        request(u, __shfl_sync(0xffffffffu, ahead < 32 ? cur : nxt, (ahead & 31) + g));
                    } else {
                        const int32_t id = __shfl_sync(0xffffffffu, cur, (t0 + u) * G + g);
                        const int4* row = reinterpret_cast<const int4*>(a.rows.codes + (int64_t)id * a.code_ld);
                        const int4* c = reinterpret_cast<const int4*>(a.q.codes + b * a.code_ld);
#pragma unroll 4
                        for (int k = lg; k < (id >= 0 ? chunks : 0); k += LPR) {
                            const int4 r = __ldg(row + k), y = __ldg(c + k);
                            dot = __dp4a(r.x, y.x, __dp4a(r.y, y.y, __dp4a(r.z, y.z, __dp4a(r.w, y.w, dot))));
                        }
                        __syncwarp();
                    }
#pragma unroll
                    for (int o = LPR / 2; o >= 1; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                    const int there = __shfl_sync(0xffffffffu, dot, lane % G * LPR);
                    if (lane / G == t0 + u) mine = there;
                }
            }
            if (m0 + lane < m_hi)
                a.out[b * a.w + m0 + lane] = cur >= 0 ? vl_quant_pair<METRIC, true, false>(mine, q, vl_quant_side<METRIC>(cs, cn)) : VL_MAXFLOAT;
            cur = nxt;
        }
    }
}

unsigned warp_blocks(int64_t warps)
{
    const int64_t blocks = (warps + 7) / 8, cap = (int64_t)vl_sm_count() * 32;
    return (unsigned)(blocks < cap ? blocks : cap);
}
// groups of four elements of every row are aligned to their size
bool fours(const void* rows, int64_t ld, int size)
{
    return ((uintptr_t)rows | (uintptr_t)(ld * size)) % (4 * size) == 0;
}

template <typename T>
int write_rows(WriteArgs a, cudaStream_t stream)
{
    if (a.m <= kFewRows) a.owner = nullptr;
    if (a.ids && a.owner) {
        const int64_t blocks = (a.m + 255) / 256, cap = (int64_t)vl_sm_count() * 8;
        quant_claim_kernel<<<(unsigned)(blocks < cap ? blocks : cap), 256, 0, stream>>>(a.ids, a.m, a.n, a.owner);
        VL_CHECK_LAUNCH("quant_claim_kernel");
    }
    const bool vec = fours(a.rows, a.ld, sizeof(T));
    // several rows per warp where they are short and many
#define VL_WRITE(HELD, R)                                                                                        \
    do {                                                                                                         \
        if (vec) quant_write_kernel<T, true, HELD, R><<<warp_blocks((a.m + R - 1) / R), 256, 0, stream>>>(a);    \
        else quant_write_kernel<T, false, HELD, R><<<warp_blocks((a.m + R - 1) / R), 256, 0, stream>>>(a);       \
    } while (0)
    const bool many = a.m > (int64_t)vl_sm_count() * 64;
    constexpr bool kShort = sizeof(T) == 2;      // half the bytes of a row: another row in flight for as many
    if (a.dim <= 128 && many) VL_WRITE(1, 4);
    else if (a.dim <= 256 && many) VL_WRITE(2, (kShort ? 4 : 2));
    else if (a.dim <= 256) VL_WRITE(2, 1);
    else if (a.dim <= 768 && many) VL_WRITE(6, (kShort ? 2 : 1));
    else if (a.dim <= 768) VL_WRITE(6, 1);
    else VL_WRITE(12, 1);
#undef VL_WRITE
    VL_CHECK_LAUNCH("quant_write_kernel");
    return 0;
}
int write_any(const WriteArgs& a, int type, cudaStream_t stream)
{
    return type == VL_TYPE_F32 ? write_rows<float>(a, stream)
                               : type == VL_TYPE_BF16 ? write_rows<__nv_bfloat16>(a, stream) : write_rows<__half>(a, stream);
}

template <typename T>
int read_rows(const VlQuantRows& held, int64_t n, int dim, int code_ld, const int32_t* ids, int64_t first_row, int64_t m, void* out,
              int64_t out_ld, int* status, cudaStream_t s)
{
    const bool vec = fours(out, out_ld, sizeof(T));
#define VL_READ(HELD)                                                                                                                   \
    do {                                                                                                                                \
        if (vec) quant_read_kernel<T, true, HELD><<<warp_blocks(m), 256, 0, s>>>(held, n, dim, code_ld, ids, first_row, m, (T*)out, out_ld, status);   \
        else quant_read_kernel<T, false, HELD><<<warp_blocks(m), 256, 0, s>>>(held, n, dim, code_ld, ids, first_row, m, (T*)out, out_ld, status);      \
    } while (0)
    if (dim <= 128) VL_READ(1);
    else if (dim <= 256) VL_READ(2);
    else if (dim <= 512) VL_READ(4);
    else VL_READ(6);
#undef VL_READ
    VL_CHECK_LAUNCH("quant_read_kernel");
    return 0;
}

// The queries of a scoring call: given as codes, or as floating-point rows that are quantised into the caller's scratch.
int take_queries(const void* queries, int type, int64_t ld, int64_t nq, int dim, int code_ld, int8_t* codes, float* scales,
                 int32_t* norms, int* status, cudaStream_t stream)
{
    if (!queries) return 0;
    const WriteArgs a = {queries, nq, ld, dim, nullptr, 0, codes, scales, norms, nq, code_ld, nullptr, status};
    return write_any(a, type, stream);
}

template <typename T, int METRIC, bool VEC>
void launch_listed(ListedArgs a, cudaStream_t stream)
{
    // a few thousand warps fill the device: with fewer queries a list is divided among warps, 32 ids at least for each
    const int64_t sms = vl_sm_count();
    a.span = a.w;
    if (a.nq < sms * 32) {
        const int64_t want = (sms * 32 + a.nq - 1) / a.nq;
        a.span = (int)(((a.w + want - 1) / want + 31) / 32 * 32);
    }
    a.spans = (a.w + a.span - 1) / a.span;
    const int64_t blocks = (a.nq * a.spans + 3) / 4, cap = sms * 64;
    const unsigned grid = (unsigned)(blocks < cap ? blocks : cap);
    const int chunks = a.code_ld / 16;
#define VL_LISTED(L, J) quant_listed_kernel<T, L, J, METRIC, VEC><<<grid, 128, 0, stream>>>(a)
    if (chunks <= 4) VL_LISTED(4, 1);
    else if (chunks <= 8) VL_LISTED(8, 1);
    else if (chunks <= 16) VL_LISTED(8, 2);
    else if (chunks <= 24) VL_LISTED(8, 3);
    else if (chunks <= 32) VL_LISTED(16, 2);
    else if (chunks <= 48) VL_LISTED(16, 3);
    else if (chunks <= 64) VL_LISTED(32, 2);
    else if (chunks <= 96) VL_LISTED(32, 3);
    else VL_LISTED(32, 0);
#undef VL_LISTED
}
template <typename T, int METRIC>
void launch_listed(const ListedArgs& a, cudaStream_t stream)
{
    if (!a.queries || fours(a.queries, a.q_ld, sizeof(T))) launch_listed<T, METRIC, true>(a, stream);
    else launch_listed<T, METRIC, false>(a, stream);
}
template <typename T>
void launch_listed(const ListedArgs& a, int metric, cudaStream_t stream)
{
    if (metric == VL_METRIC_COSINE) launch_listed<T, VL_METRIC_COSINE>(a, stream);
    else launch_listed<T, VL_METRIC_SQL2>(a, stream);
}
constexpr int kMaxList = 1 << 30;            // places of a list, and those 64 ahead that are asked for, are ints
constexpr int kListedRounds = 96 * 16;       // columns up to which quant_listed_kernel rounds its queries itself

// every place (null ones too) is aligned to elements of `size` bytes
bool aligned(size_t size, std::initializer_list<const void*> places)
{
    uintptr_t bits = 0;
    for (const void* p : places) bits |= (uintptr_t)p;
    return bits % size == 0;
}
size_t type_size(int type) { return type == VL_TYPE_F32 ? 4 : 2; }

#define VL_CHECK_SHAPE(name, n, dim, ld)                                                                                    \
    VL_CHECK_ARG((n) >= 0 && (n) < VL_MAXINT, name ": row count %lld outside int32", (long long)(n));                       \
    VL_CHECK_ARG((dim) > 0 && (dim) <= kMaxDim, name ": dimension %d outside 1..%d", (int)(dim), kMaxDim);                  \
    VL_CHECK_ARG((ld) % 16 == 0 && (ld) >= (dim) && (ld) < (dim) + 16, name ": codes are held %d columns wide, not dim %d to the next multiple of 16", (int)(ld), (int)(dim))

}  // namespace

extern "C" int vl_quant_write(const void* rows, int type, int64_t m, int dim, int64_t ld, const int32_t* ids, int64_t first_row,
                              int8_t* codes, float* scales, int32_t* norms, int64_t n, int code_ld, int32_t* owner, int* status,
                              void* stream)
{
    VL_CHECK_SHAPE("vl_quant_write", n, dim, code_ld);
    VL_CHECK_ARG(m >= 0 && m < VL_MAXINT, "vl_quant_write: bad size");
    VL_CHECK_ARG(type >= VL_TYPE_F32 && type <= VL_TYPE_F16, "vl_quant_write: unknown type %d", type);
    VL_CHECK_ARG(ids || (first_row >= 0 && first_row + m <= n), "vl_quant_write: rows %lld..%lld outside 0..%lld",
                 (long long)first_row, (long long)(first_row + m), (long long)n);
    if (m == 0) return 0;
    VL_CHECK_ARG(rows && status && (n == 0 || (codes && scales && norms && (!ids || owner))), "vl_quant_write: null pointer");
    VL_CHECK_ARG(aligned(16, {codes}), "vl_quant_write: codes must be 16-byte aligned");
    VL_CHECK_ARG(aligned(type_size(type), {rows}) && aligned(4, {ids, scales, norms, owner, status}),
                 "vl_quant_write: a pointer is not aligned to its elements");
    const WriteArgs a = {rows, m, ld, dim, ids, first_row, codes, scales, norms, n, code_ld, owner, status};
    return write_any(a, type, (cudaStream_t)stream);
}

extern "C" int vl_quant_read(const int8_t* codes, const float* scales, int64_t n, int dim, int code_ld, const int32_t* ids,
                             int64_t first_row, int64_t m, void* out, int type, int64_t out_ld, int* status, void* stream)
{
    VL_CHECK_SHAPE("vl_quant_read", n, dim, code_ld);
    VL_CHECK_ARG(m >= 0 && m < VL_MAXINT, "vl_quant_read: bad size");
    VL_CHECK_ARG(type >= VL_TYPE_F32 && type <= VL_TYPE_F16, "vl_quant_read: unknown type %d", type);
    VL_CHECK_ARG(ids || (first_row >= 0 && first_row + m <= n), "vl_quant_read: rows %lld..%lld outside 0..%lld",
                 (long long)first_row, (long long)(first_row + m), (long long)n);
    if (m == 0) return 0;
    VL_CHECK_ARG(out && status && (n == 0 || (codes && scales)), "vl_quant_read: null pointer");
    VL_CHECK_ARG(aligned(16, {codes}), "vl_quant_read: codes must be 16-byte aligned");
    VL_CHECK_ARG(aligned(type_size(type), {out}) && aligned(4, {ids, scales, status}), "vl_quant_read: a pointer is not aligned to its elements");
    VL_CHECK_ARG(out_ld >= dim || m == 1, "vl_quant_read: rows of the result overlap");
    const VlQuantRows held = {codes, scales, nullptr};
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == VL_TYPE_F32) return read_rows<float>(held, n, dim, code_ld, ids, first_row, m, out, out_ld, status, s);
    if (type == VL_TYPE_BF16) return read_rows<__nv_bfloat16>(held, n, dim, code_ld, ids, first_row, m, out, out_ld, status, s);
    return read_rows<__half>(held, n, dim, code_ld, ids, first_row, m, out, out_ld, status, s);
}

extern "C" int vl_quant_scores(const void* queries, int q_type, int64_t q_ld, int8_t* q_codes, float* q_scales, int32_t* q_norms,
                               int64_t nq, const int8_t* codes, const float* scales, const int32_t* norms, int64_t n, int dim,
                               int code_ld, int64_t row_lo, int64_t row_hi, void* out, int type, int64_t out_ld, int metric,
                               int* status, void* stream)
{
    return vl_quant_scores_wait(queries, q_type, q_ld, q_codes, q_scales, q_norms, nq, codes, scales, norms, n, dim, code_ld, row_lo, row_hi, out, type,
                                out_ld, metric, 0, status, stream);
}

extern "C" int vl_quant_scores_wait(const void* queries, int q_type, int64_t q_ld, int8_t* q_codes, float* q_scales, int32_t* q_norms,
                                    int64_t nq, const int8_t* codes, const float* scales, const int32_t* norms, int64_t n, int dim,
                                    int code_ld, int64_t row_lo, int64_t row_hi, void* out, int type, int64_t out_ld, int metric,
                                    int wait_us, int* status, void* stream)
{
    VL_CHECK_SHAPE("vl_quant_scores", n, dim, code_ld);
    VL_CHECK_ARG(nq >= 0 && nq < VL_MAXINT, "vl_quant_scores: bad size");
    VL_CHECK_ARG(wait_us >= 0 && wait_us <= 2000000, "vl_quant_scores: a wait of %d microseconds, not 0..2000000", wait_us);
    VL_CHECK_ARG(0 <= row_lo && row_lo <= row_hi && row_hi <= n, "vl_quant_scores: bad row range");
    VL_CHECK_ARG(!queries || (q_type >= VL_TYPE_F32 && q_type <= VL_TYPE_F16), "vl_quant_scores: unknown type %d", q_type);
    VL_CHECK_ARG(metric == VL_METRIC_COSINE || metric == VL_METRIC_SQL2 || metric == VL_QUANT_PRODUCT, "vl_quant_scores: unknown metric %d", metric);
    VL_CHECK_ARG(type == VL_TYPE_F32 || (metric == VL_QUANT_PRODUCT && type > VL_TYPE_F32 && type <= VL_TYPE_F16),
                 "vl_quant_scores: distances are 32-bit numbers, products of a known type (got %d)", type);
    if (nq == 0 || row_lo == row_hi) return 0;
    const bool few = queries && nq <= VL_QUANT_FEW_QUERIES && code_ld <= VL_QUANT_FEW_COLUMNS;      // no need of the scratch
    VL_CHECK_ARG((few || (q_codes && q_scales && q_norms)) && codes && scales && norms && out && status, "vl_quant_scores: null pointer");
    VL_CHECK_ARG(aligned(16, {codes, q_codes}), "vl_quant_scores: codes must be 16-byte aligned");
    VL_CHECK_ARG((!queries || aligned(type_size(q_type), {queries})) && aligned(type_size(type), {out}) &&
                 aligned(4, {q_scales, q_norms, scales, norms, status}), "vl_quant_scores: a pointer is not aligned to its elements");
    VL_CHECK_ARG(out_ld >= row_hi - row_lo || nq == 1, "vl_quant_scores: rows of the result overlap");
    const cudaStream_t s = (cudaStream_t)stream;
    if (!few) {
        const int rc = take_queries(queries, q_type, q_ld, nq, dim, code_ld, q_codes, q_scales, q_norms, status, s);
        if (rc) return rc;
        queries = nullptr;
    }
    return vl_quant_scan(queries, q_type, q_ld, {q_codes, q_scales, q_norms}, nq, {codes, scales, norms}, n, dim, code_ld, row_lo, row_hi, out,
                         type, out_ld, metric, wait_us, status, s);
}

extern "C" int vl_quant_listed(const void* queries, int q_type, int64_t q_ld, int8_t* q_codes, float* q_scales, int32_t* q_norms,
                               int64_t nq, const int8_t* codes, const float* scales, const int32_t* norms, int64_t n, int dim,
                               int code_ld, const int32_t* ids, int w, float* out, int metric, int* status, void* stream)
{
    VL_CHECK_SHAPE("vl_quant_listed", n, dim, code_ld);
    VL_CHECK_ARG(nq >= 0 && nq < VL_MAXINT && w >= 0 && w <= kMaxList, "vl_quant_listed: bad size");
    VL_CHECK_ARG(!queries || (q_type >= VL_TYPE_F32 && q_type <= VL_TYPE_F16), "vl_quant_listed: unknown type %d", q_type);
    VL_CHECK_ARG(metric == VL_METRIC_COSINE || metric == VL_METRIC_SQL2, "vl_quant_listed: unknown metric %d", metric);
    if (nq == 0 || w == 0) return 0;
    const bool rounds = queries && code_ld <= kListedRounds;      // no need of the scratch
    VL_CHECK_ARG((rounds || (q_codes && q_scales && q_norms)) && ids && out && status && (n == 0 || (codes && scales && norms)), "vl_quant_listed: null pointer");
    VL_CHECK_ARG(aligned(16, {codes, q_codes}), "vl_quant_listed: codes must be 16-byte aligned");
    VL_CHECK_ARG((!queries || aligned(type_size(q_type), {queries})) && aligned(4, {q_scales, q_norms, scales, norms, ids, out, status}),
                 "vl_quant_listed: a pointer is not aligned to its elements");
    const cudaStream_t s = (cudaStream_t)stream;
    if (!rounds) {
        const int rc = take_queries(queries, q_type, q_ld, nq, dim, code_ld, q_codes, q_scales, q_norms, status, s);
        if (rc) return rc;
        queries = nullptr;
    }
    // 127^2 * 1040 is below 2^24: without l2, sums of squared codes are looked at in wider rows only
    const ListedArgs a = {queries, q_ld, {q_codes, q_scales, q_norms}, {codes, scales, norms}, nq, n, dim, code_ld, ids, w, 0, 0, out, status,
                          metric == VL_METRIC_SQL2 || dim > 1040};
    if (!queries || q_type == VL_TYPE_F32) launch_listed<float>(a, metric, s);
    else if (q_type == VL_TYPE_BF16) launch_listed<__nv_bfloat16>(a, metric, s);
    else launch_listed<__half>(a, metric, s);
    VL_CHECK_LAUNCH("quant_listed_kernel");
    return 0;
}
