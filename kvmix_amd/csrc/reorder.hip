// The first dimension of many tensors reordered in place:  t[i] = old t[index[i]], the same index for all of them (the states of beams
// that go on).
//
// Bound by memory: rows that stay are neither read nor written, and a row that several others become is read by the same thread
// for all of them, from HBM once.  A thread takes one piece of sixteen bytes of a row, at the same place of all rows, so that no other
// thread reads what it writes and nothing has to be waited for.  Up to 64 rows are a wave's lanes, their sets bits of a mask.  Where what
// is written is read by no other row (beams placed so that the first child stays where its parent was), sixteen rows go at once;
// where not, up to 32 rows' old values are in registers before the first is written.  Otherwise old values that are still wanted
// when their place is written are put in the LDS first, each by the thread that will want it; where they are too many for
// all threads of a block, fewer take a turn.
// 2.2 GB of states in 32 rows: 440 us where half of them stay (1.1 GB read, 1.1 written, 5.0 TB/s), 895 us where all are moved round (2.2 GB each,
// 4.9 TB/s).  Through the LDS less: 40 rows of 1.4 GB moved round 1.6 ms (1.8 TB/s), 128 of 1.3 GB 4.1 ms.
#include <algorithm>
#include <numeric>
#include <vector>

#include "copy_rows.h"

namespace kvmix {

constexpr int kReorderItems = 40, kReorderThreads = 256, kReorderAhead = 8;
constexpr int kReorderRows = 1024, kReorderStage = 2048;  // rows at most; pieces in the LDS

struct ReorderItem {
    uint8_t *base;
    int64_t batch, outer, inner;  // bytes from one to the next
    int64_t row_bytes;
    uint32_t pieces;              // of one i of the first dimension
    CopyDiv per_row, rows;        // pieces of a row, rows of an outer one
};

struct ReorderArgs {
    ReorderItem item[kReorderItems];
    uint32_t first[kReorderItems + 1];
    const int64_t *index;
    int count, rows;
};

typedef uint32_t word4 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t word2 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t word1 __attribute__((aligned(1)));
typedef uint16_t half1 __attribute__((aligned(1)));

typedef uint32_t Bytes16 __attribute__((ext_vector_type(4)));

// Sixteen bytes, or the first n of them, piece by piece: the last of a row is followed by what another thread writes.  STREAM: whole ones
// as what nobody wants again soon.
template <bool STREAM>
__device__ __forceinline__ Bytes16 load_bytes(const uint8_t *p, int n)
{
    if (n == 16) return STREAM ? __builtin_nontemporal_load((const word4 *)p) : *(const word4 *)p;
    uint32_t first[2] = {0, 0}, four = 0, tail = 0;
    if (n & 8) {
        const word2 x = *(const word2 *)p;
        first[0] = x[0], first[1] = x[1];
    }
    if (n & 4) four = *(const word1 *)(p + (n & 8));
    if (n & 2) tail = *(const half1 *)(p + (n & 12));
    if (n & 1) tail |= (uint32_t)p[n & 14] << (n & 2) * 8;
    return Bytes16{first[0], first[1], four, tail};
}

template <bool STREAM>
__device__ __forceinline__ void store_bytes(uint8_t *p, Bytes16 v, int n)
{
    if (n == 16) {
        if constexpr (STREAM) __builtin_nontemporal_store((word4)v, (word4 *)p);
        else *(word4 *)p = v;
        return;
    }
    if (n & 8) *(word2 *)p = word2{v[0], v[1]};
    if (n & 4) *(word1 *)(p + (n & 8)) = v[2];
    if (n & 2) *(half1 *)(p + (n & 12)) = (uint16_t)v[3];
    if (n & 1) p[n & 14] = (uint8_t)(v[3] >> (n & 2) * 8);
}

struct Piece16 {
    uint8_t *at;  // of the first row
    int64_t batch;
    int bytes;
};

__device__ __forceinline__ Piece16 piece_of(const ReorderItem &it, uint32_t p)
{
    const uint32_t row = copy_div(p, it.per_row), o = copy_div(row, it.rows);
    const int64_t in = (int64_t)(p - row * it.per_row.d) * 16;
    return {it.base + o * it.outer + (row - o * it.rows.d) * it.inner + in, it.batch, (int)(it.row_bytes - in < 16 ? it.row_bytes - in : 16)};
}

// Rows `change` (a bit each) become their sources, N at once: every old value of these is read before the first is written.  All lanes
// come here, since each has the source of a row in its register; those that have no piece of their own (`mine`) write nothing.
template <int N, bool STREAM>
__device__ __forceinline__ void move_rows(uint8_t *at, int64_t batch, int bytes, bool mine, uint64_t change, int source)
{
    while (change) {
        Bytes16 v[N];
        uint64_t left = change;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (left) {
                v[j] = load_bytes<STREAM>(at + __builtin_amdgcn_readlane(source, __builtin_ctzll(left)) * batch, bytes);
                left &= left - 1;
            }
        if (mine) {
            uint64_t to = change;
#pragma unroll
            for (int j = 0; j < N; j++)
                if (to) {
                    store_bytes<STREAM>(at + __builtin_ctzll(to) * batch, v[j], bytes);
                    to &= to - 1;
                }
        }
        change = left;
    }
}

template <bool STREAM>
__global__ void __launch_bounds__(kReorderThreads) reorder_rows(ReorderArgs a)
{
    const int t = threadIdx.x, lane = t % kWave;
    const int64_t own = a.rows <= kWave && lane < a.rows ? a.index[lane] : lane;
    const int nth = __popcll(__ballot(lane < a.count && blockIdx.x >= a.first[min(lane, kReorderItems)])) - 1;
    const ReorderItem it = a.item[nth];
    const uint32_t begin = (blockIdx.x - a.first[nth]) * kReorderThreads;
    const uint32_t end = begin + kReorderThreads < it.pieces ? begin + kReorderThreads : it.pieces;

    if (a.rows <= kWave) {
        // every wave has all rows in its lanes
        const int source = own >= 0 && own < a.rows ? (int)own : lane;  // (an index that is none changes nothing)
        const uint64_t change = __ballot(source != lane);
        if (!change) return;
        uint64_t wanted = 0;
        for (uint64_t left = change; left; left &= left - 1) wanted |= 1ull << __builtin_amdgcn_readlane(source, __builtin_ctzll(left));
        const bool apart = !(wanted & change);  // nothing that is written is read
        if (apart || __popcll(change) <= 32) {
            if (begin + __builtin_amdgcn_readfirstlane(t - lane) >= end) return;  // (a wave in which no lane has a piece)
            const bool mine = begin + t < end;
            const Piece16 piece = piece_of(it, mine ? begin + t : end - 1);
            auto move = [&](int bytes) {
                if (__popcll(change) <= 8) move_rows<8, STREAM>(piece.at, piece.batch, bytes, mine, change, source);
                else if (apart) move_rows<16, STREAM>(piece.at, piece.batch, bytes, mine, change, source);
                else move_rows<32, STREAM>(piece.at, piece.batch, bytes, mine, change, source);
            };
            if (__all(piece.bytes == 16)) move(16);
            else move(piece.bytes);
            return;
        }
    }

    // many rows, or many that are written and read
    __shared__ Bytes16 stage[kReorderStage];
    extern __shared__ int16_t lists[];  // of a.rows each
    int16_t *source = lists, *change = source + a.rows, *early = change + a.rows, *slot = early + a.rows;  // slot: of an old value in the LDS, or -1
    int16_t *wanted = slot + a.rows;
    __shared__ int changes, earlies;
    if (t == 0) changes = earlies = 0;
    for (int i = t; i < a.rows; i += kReorderThreads) {
        const int64_t from = a.index[i];
        source[i] = (int16_t)(from >= 0 && from < a.rows ? from : i);
        wanted[i] = 0;
    }
    __syncthreads();
    for (int i = t; i < a.rows; i += kReorderThreads)
        if (source[i] != i) wanted[source[i]] = 1;
    __syncthreads();
    for (int i = t; i < a.rows; i += kReorderThreads) {
        slot[i] = -1;
        if (source[i] == i) continue;
        change[atomicAdd(&changes, 1)] = (int16_t)i;
        if (wanted[i]) {
            const int s = atomicAdd(&earlies, 1);
            early[s] = (int16_t)i, slot[i] = (int16_t)s;
        }
    }
    __syncthreads();
    const int n = __builtin_amdgcn_readfirstlane(changes), staged = __builtin_amdgcn_readfirstlane(earlies);
    if (n == 0) return;
    const int at_once = staged * kReorderThreads > kReorderStage ? kReorderStage / staged : kReorderThreads;
    if (t >= at_once) return;
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    for (uint32_t p = begin + t; p < end; p += at_once) {
        const Piece16 piece = piece_of(it, p);
        Bytes16 v[kReorderAhead];
        for (int i = 0; i < staged; i += kReorderAhead) {
#pragma unroll
            for (int j = 0; j < kReorderAhead; j++)
                if (i + j < staged) v[j] = load_bytes<STREAM>(piece.at + uniform(early[i + j]) * piece.batch, piece.bytes);
#pragma unroll
            for (int j = 0; j < kReorderAhead; j++)
                if (i + j < staged) stage[(i + j) * at_once + t] = v[j];
        }
        for (int i = 0; i < n; i += kReorderAhead) {
#pragma unroll
            for (int j = 0; j < kReorderAhead; j++) {
                if (i + j < n) {
                    const int from = uniform(source[uniform(change[i + j])]), s = uniform(slot[from]);
                    v[j] = s >= 0 ? stage[s * at_once + t] : load_bytes<STREAM>(piece.at + from * piece.batch, piece.bytes);
                }
            }
#pragma unroll
            for (int j = 0; j < kReorderAhead; j++)
                if (i + j < n) store_bytes<STREAM>(piece.at + uniform(change[i + j]) * piece.batch, v[j], piece.bytes);
        }
    }
}

namespace {

// What a tensor takes of memory: runs of bytes, every stride[i] bytes of each dimension, larger strides first.
struct Layout {
    int64_t at;              // of the first byte
    int64_t size[3], stride[3];
    int64_t extent[4];       // what is left of it from dimension i on spans; the last: a run
    int dims;
};

// Bytes from the first to behind the last.
__int128 extent_of(const kvmix_reorder_t &p, int64_t rows)
{
    return (__int128)(rows - 1) * p.batch_stride + (__int128)(p.outer - 1) * p.outer_stride + (__int128)(p.inner - 1) * p.inner_stride + p.row_bytes;
}

Layout layout_of(const kvmix_reorder_t &p, int64_t rows)
{
    struct Dim {
        int64_t size, stride;
    } dim[3] = {{rows, p.batch_stride}, {p.outer, p.outer_stride}, {p.inner, p.inner_stride}};
    std::sort(dim, dim + 3, [](const Dim &a, const Dim &b) { return a.stride > b.stride; });
    Layout l{};
    l.at = (int64_t)p.base;
    for (const Dim &d : dim)
        if (d.size > 1) l.size[l.dims] = d.size, l.stride[l.dims++] = d.stride;
    l.extent[l.dims] = p.row_bytes;
    for (int i = l.dims - 1; i >= 0; i--) l.extent[i] = (l.size[i] - 1) * l.stride[i] + l.extent[i + 1];
    return l;
}

int64_t down(int64_t a, int64_t b) { return a / b - (a % b < 0); }

// Columns beside one another of the same wider rows: the runs of both begin at one place each of a stride that all of theirs are multiples
// of, and fit beside one another there.
bool columns_apart(const Layout &a, int i, const Layout &b, int j, int64_t d)
{
    int64_t stride = 0;
    while (i < a.dims) stride = std::gcd(stride, a.stride[i++]);
    while (j < b.dims) stride = std::gcd(stride, b.stride[j++]);
    d = (d % stride + stride) % stride;
    return d >= a.extent[a.dims] && d + b.extent[b.dims] <= stride;
}

// Whether what is left of a from dimension i on and of b from j on, which begins `d` bytes after a's, have a byte in common.  Where their strides
// are alike only the distance of their indexes matters, and few distances bring them near one another; where not, the larger
// stride's entries are looked at one by one.  That ends after `steps`: then they count as meeting.
bool meet(const Layout &a, int i, const Layout &b, int j, int64_t d, int &steps)
{
    if (d >= a.extent[i] || -d >= b.extent[j]) return false;
    if ((i == a.dims && j == b.dims) || --steps < 0) return true;
    const bool both = i < a.dims && j < b.dims && a.stride[i] == b.stride[j], of_a = both || j == b.dims || (i < a.dims && a.stride[i] > b.stride[j]);
    const bool of_b = both || !of_a;
    if (!both && i < a.dims && j < b.dims && columns_apart(a, i, b, j, d)) return false;
    const int64_t stride = of_a ? a.stride[i] : b.stride[j], ea = a.extent[i + of_a], eb = b.extent[j + of_b];
    const int64_t least = of_a ? -(a.size[i] - 1) : 0, most = of_b ? b.size[j] - 1 : 0;  // of the index of b less that of a
    for (int64_t m = std::max(least, down(-eb - d, stride) + 1); m <= std::min(most, down(ea - d - 1, stride)); m++)
        if (meet(a, i + of_a, b, j + of_b, d + m * stride, steps)) return true;
    return false;
}

// Whether two of the tensors have memory in common, or a code of its own.
int check_apart(const kvmix_reorder_t *items, int64_t count, int64_t rows)
{
    struct Span {
        int64_t from, to;
        const kvmix_reorder_t *item;
    };
    std::vector<Span> all;
    all.reserve(count);
    for (int64_t i = 0; i < count; i++) {
        const kvmix_reorder_t &p = items[i];
        if (p.outer == 0 || p.inner == 0 || p.row_bytes == 0) continue;
        const __int128 extent = extent_of(p, rows);
        if (extent < 0 || extent > (int64_t)1 << 60) return KVMIX_ERR_UNSUPPORTED;  // (nothing that an address space could hold)
        all.push_back({(int64_t)p.base, (int64_t)p.base + (int64_t)extent, &p});
    }
    std::sort(all.begin(), all.end(), [](const Span &a, const Span &b) { return a.from < b.from; });
    bool apart = true;
    for (size_t i = 0; i + 1 < all.size(); i++) apart = apart && all[i].to <= all[i + 1].from;
    if (apart) return KVMIX_OK;

    std::vector<Layout> l;
    l.reserve(all.size());
    for (const Span &span : all) l.push_back(layout_of(*span.item, rows));
    auto in_common = [&](size_t i, size_t j) {
        int steps = 1 << 16;
        return meet(l[i], 0, l[j], 0, l[j].at - l[i].at, steps);
    };
    const int64_t stride = l[0].stride[0];
    if (std::all_of(l.begin(), l.end(), [&](const Layout &a) { return a.stride[0] == stride && a.extent[1] <= stride; })) {
        // Views of one storage, or of several alike: each is near those alone that begin in its part of the stride.
        std::sort(l.begin(), l.end(), [&](const Layout &a, const Layout &b) { return a.at % stride < b.at % stride; });
        for (size_t i = 0; i < l.size(); i++)
            for (size_t k = 1; k < l.size(); k++) {
                const size_t j = (i + k) % l.size();
                const int64_t off = l[j].at % stride - l[i].at % stride;
                if ((j < i ? off + stride : off) >= l[i].extent[1]) break;
                if (in_common(i, j)) return KVMIX_ERR_OVERLAP;
            }
        return KVMIX_OK;
    }
    for (size_t i = 0; i < all.size(); i++)
        for (size_t j = i + 1; j < all.size() && all[j].from < all[i].to; j++)
            if (in_common(i, j)) return KVMIX_ERR_OVERLAP;
    return KVMIX_OK;
}

}  // namespace
}  // namespace kvmix

using namespace kvmix;

extern "C" int kvmix_reorder_rows(const kvmix_reorder_t *items, int64_t count, const int64_t *index, int64_t rows, kvmix_stream_t stream)
{
    if (count < 0 || rows < 0) return KVMIX_ERR_SHAPE;
    if (count && !items) return KVMIX_ERR_NULL;
    if (rows > kReorderRows) return KVMIX_ERR_UNSUPPORTED;
    auto empty = [](const kvmix_reorder_t &p) { return p.outer == 0 || p.inner == 0 || p.row_bytes == 0; };
    for (int64_t i = 0; i < count; i++) {
        const kvmix_reorder_t &p = items[i];
        if (p.outer < 0 || p.inner < 0 || p.row_bytes < 0) return KVMIX_ERR_SHAPE;
        if (empty(p) || rows <= 1) continue;
        if (!p.base) return KVMIX_ERR_NULL;
        if ((p.inner > 1 && p.inner_stride < p.row_bytes) || (p.outer > 1 && p.outer_stride < p.row_bytes) || p.batch_stride < p.row_bytes) return KVMIX_ERR_SHAPE;
        if (p.outer > (1ll << 31) || p.inner > (1ll << 31) || p.row_bytes > (1ll << 40) ||
            (__int128)p.outer * p.inner * ((p.row_bytes + 15) / 16) > 0x7fffffff - kReorderThreads)
            return KVMIX_ERR_UNSUPPORTED;
    }
    if (rows <= 1 || count == 0) return KVMIX_OK;  // (one row is itself)
    int rc = KVMIX_OK;
    try {
        rc = check_apart(items, count, rows);
    } catch (...) {  // (what a vector throws)
        return KVMIX_ERR_MEMORY;
    }
    if (rc != KVMIX_OK) return rc;
    if (!index) return KVMIX_ERR_NULL;
    // Tensors of more than the 256 MB that the cache before the memory holds go by the caches.  Half of 32 rows, 1 GB in all: 189 instead of 204 us,
    // 181 instead of 198 before a kernel that reads them; 256 MB: 46 instead of 39, 128 MB before one that reads them 33 instead of 22.
    __int128 total = 0;
    for (int64_t i = 0; i < count; i++) total += empty(items[i]) ? 0 : (__int128)rows * items[i].outer * items[i].inner * items[i].row_bytes;
    const bool stream_by = total > 1 << 28;
    for (int64_t i = 0; i < count;) {
        ReorderArgs a{};
        a.index = index, a.rows = (int)rows;
        for (; i < count && a.count < kReorderItems; i++) {
            const kvmix_reorder_t &p = items[i];
            if (empty(p)) continue;
            ReorderItem &it = a.item[a.count];
            it.base = (uint8_t *)p.base, it.batch = p.batch_stride, it.outer = p.outer_stride, it.inner = p.inner_stride, it.row_bytes = p.row_bytes;
            it.per_row = copy_divisor((uint32_t)((p.row_bytes + 15) / 16)), it.rows = copy_divisor((uint32_t)p.inner);
            it.pieces = (uint32_t)(p.outer * p.inner) * it.per_row.d;
            const uint32_t blocks = (it.pieces + kReorderThreads - 1) / kReorderThreads;
            if (a.first[a.count] + (uint64_t)blocks >= 1u << 24) break;  // (a launch of 2^32 threads or more runs modulo 2^32)
            a.first[a.count + 1] = a.first[a.count] + blocks;
            a.count++;
        }
        if (!a.count) continue;
        const size_t lists = (size_t)rows * 5 * sizeof(int16_t);
        if (stream_by) reorder_rows<true><<<a.first[a.count], kReorderThreads, lists, (hipStream_t)stream>>>(a);
        else reorder_rows<false><<<a.first[a.count], kReorderThreads, lists, (hipStream_t)stream>>>(a);
        rc = launch_status();
        if (rc != KVMIX_OK) break;
    }
    return rc;
}
