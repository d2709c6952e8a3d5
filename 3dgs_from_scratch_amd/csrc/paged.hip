// A paged cache's bookkeeping: new keys and values into its pages, and the keys that matter
// moved to fewer pages.

#include "paged.h"
#include "wave_ops.h"

namespace gs {

using Chunk = __attribute__((ext_vector_type(4))) uint32_t;  // 8 elements

// --------------------------------------------------------------------- append
// A thread copies 8 elements of a row's keys and values; a row's threads are neighbours.  The
// row's sequence is found by bisection of the offsets.
__global__ __launch_bounds__(256) void paged_append_kernel(
    GsPages p, const uint16_t *__restrict__ k, int64_t k_row, int64_t k_head,
    const uint16_t *__restrict__ v, int64_t v_row, int64_t v_head, int64_t rows,
    const int32_t *__restrict__ offsets, uint16_t *__restrict__ k_pages,
    uint16_t *__restrict__ v_pages, float *__restrict__ weights) {
    const int chunks = p.dim / 8, a_row = chunks * p.heads;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = at / a_row;
    if (row >= rows) return;
    const int rest = (int)(at - row * a_row), head = rest / chunks, chunk = rest - head * chunks;
    int low = 0, high = p.sequences + 1;  // offsets that are at most row
    while (low < high) {
        const int middle = (low + high) / 2;
        if (offsets[middle] <= row)
            low = middle + 1;
        else
            high = middle;
    }
    const int b = low - 1;
    if (b < 0 || b >= p.sequences) return;
    const int64_t end = offsets[b + 1] < rows ? offsets[b + 1] : rows;
    const int64_t slot = filled_slots(p, b) - (end - row);
    if (slot < 0) return;
    const int index = (int)(slot / p.page_size), place = (int)(slot - (int64_t)index * p.page_size);
    const int page = page_of(p, b, index);
    if (page < 0) return;
    const Chunk key = *(const Chunk *)(k + row * k_row + head * k_head + chunk * 8);
    const Chunk value = *(const Chunk *)(v + row * v_row + head * v_head + chunk * 8);
    const int64_t to = row_at(p, page, place) + head * p.head_stride + chunk * 8;
    *(Chunk *)(k_pages + to) = key;
    *(Chunk *)(v_pages + to) = value;
    if (weights && chunk == 0) weights[sum_at(p, page, place, head)] = 0.0f;
}

// --------------------------------------------------------------------- evict
// A weight's place in the order of all floats: larger is larger, both zeros are one, NaN is above
// infinity.
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);  // -0 + 0 = 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kPick = 1024;  // threads

// Which slots stay: a workgroup a sequence and head.  The smallest order that stays is found
// by its bytes, from the highest, with a histogram of the slots that agree so far; then the
// slots are walked in order.
__global__ __launch_bounds__(kPick) void paged_pick_kernel(GsPages p,
                                                           const float *__restrict__ weights,
                                                           int32_t keep, int32_t recent,
                                                           int32_t *__restrict__ new_lengths,
                                                           int32_t *__restrict__ kept) {
    __shared__ uint32_t histogram[256];
    __shared__ uint32_t scan[kPick / kWave + 1];
    __shared__ uint32_t found[2];
    const int b = blockIdx.x / p.heads, head = blockIdx.x % p.heads, t = threadIdx.x;
    const int filled = filled_slots(p, b), old = max(filled - recent, 0);
    int32_t *out = kept + (int64_t)blockIdx.x * keep;
    const auto sum_of = [&](int slot, uint32_t *order) {  // false: the slot is not there
        const int index = slot / p.page_size, page = page_of(p, b, index);
        if (page < 0) return false;
        *order = order_of(weights[sum_at(p, page, slot - index * p.page_size, head)]);
        return true;
    };
    // slots that are there: recent ones and others
    uint32_t there = 0, there_old = 0, order;
    for (int slot = t; slot < filled; slot += kPick)
        if (sum_of(slot, &order)) {
            ++there;
            there_old += slot < old;
        }
    uint32_t all, all_old;
    block_exclusive_scan<uint32_t, kPick>(there, scan, all);
    block_exclusive_scan<uint32_t, kPick>(there_old, scan, all_old);
    // the old slots that stay: `want` of all_old
    const uint32_t want = min((uint32_t)keep - (all - all_old), all_old);
    uint32_t threshold = 0, need = want;  // those above it stay, and the first `need` equal to it
    if (want > 0 && want < all_old) {
        uint32_t mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (t < 256) histogram[t] = 0;
            __syncthreads();
            for (int slot = t; slot < old; slot += kPick)
                if (sum_of(slot, &order) && (order & mask) == threshold)
                    atomicAdd(&histogram[order >> shift & 255], 1u);
            __syncthreads();
            if (t == 0) {
                uint32_t above = 0;
                int byte = 255;
                while (above + histogram[byte] < need) above += histogram[byte--];
                found[0] = byte;
                found[1] = need - above;
            }
            __syncthreads();
            threshold |= found[0] << shift;
            need = found[1];
            mask |= 255u << shift;
            __syncthreads();
        }
    }
    const bool none = want == 0, every = want == all_old;
    uint32_t written = 0, equal = 0;
    for (int first = 0; first < filled; first += kPick) {
        const int slot = first + t;
        const bool is = slot < filled && sum_of(slot, &order), late = slot >= old;
        const bool same = is && !late && !none && !every && order == threshold;
        uint32_t total;
        const uint32_t before = equal + block_exclusive_scan<uint32_t, kPick>(same, scan, total);
        equal += total;
        const bool stays = is && (late || every || (!none && (order > threshold || (same && before < need))));
        const uint32_t to = written + block_exclusive_scan<uint32_t, kPick>(stays, scan, total);
        written += total;
        if (stays && to < (uint32_t)keep) out[to] = slot;
    }
    for (int j = written + t; j < keep; j += kPick) out[j] = -1;
    if (head == 0 && t == 0) new_lengths[b] = (int32_t)written;
}

// The picked slots to the new pages: a thread moves 8 elements of a key and a value.
__global__ __launch_bounds__(256) void paged_move_kernel(GsPages p, uint16_t *k_pages,
                                                         uint16_t *v_pages, float *weights,
                                                         const int32_t *__restrict__ new_tables,
                                                         int64_t new_stride, int32_t keep,
                                                         const int32_t *__restrict__ kept) {
    const int chunks = p.dim / 8, a_row = chunks * p.heads, b = blockIdx.y;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = at / a_row;
    if (row >= keep) return;
    const int rest = (int)(at - row * a_row), head = rest / chunks, chunk = rest - head * chunks;
    const int j = (int)row;
    const int slot = kept[((int64_t)b * p.heads + head) * keep + j];
    if (slot < 0) return;
    const int to_page = new_tables[b * new_stride + j / p.page_size], to_place = j % p.page_size;
    if ((uint32_t)to_page >= (uint64_t)p.pages) return;
    const int page = page_of(p, b, slot / p.page_size), place = slot % p.page_size;
    const int64_t from = row_at(p, page, place) + head * p.head_stride + chunk * 8;
    const int64_t to = row_at(p, to_page, to_place) + head * p.head_stride + chunk * 8;
    *(Chunk *)(k_pages + to) = *(const Chunk *)(k_pages + from);
    *(Chunk *)(v_pages + to) = *(const Chunk *)(v_pages + from);
    if (chunk == 0)
        weights[sum_at(p, to_page, to_place, head)] = weights[sum_at(p, page, place, head)];
}

int check_pages(const GsPages *p, bool weights) {
    if (!p || p->pages < 0 || p->sequences < 0 || p->page_size < 1 || p->heads < 1 || p->dim < 1 ||
        p->table_width < 0 || p->table_stride < 0 || p->page_stride < 0 || p->slot_stride < 0 ||
        p->head_stride < 0 || !element_type(p->type))
        return GS_ERR_INVALID_ARGUMENT;
    if (weights && (p->sum_page < 0 || p->sum_slot < 0 || p->sum_head < 0))
        return GS_ERR_INVALID_ARGUMENT;
    if (p->sequences > 0 && (!p->lengths || (p->table_width > 0 && !p->tables)))
        return GS_ERR_INVALID_ARGUMENT;
    if (p->type == GS_F32 || p->dim % 8 != 0 || p->dim > GS_MAX_HEAD_DIM ||
        p->pages > 0x7fffffffLL || (int64_t)p->page_size * p->table_width > kMaxSlots ||
        p->slot_stride < p->dim || p->slot_stride > (1 << 23) ||
        (p->page_stride | p->slot_stride | p->head_stride) % 8 != 0)
        return GS_ERR_UNSUPPORTED;
    return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" int gs_paged_append(const GsPages *p, const void *k, int64_t k_row, int64_t k_head,
                               const void *v, int64_t v_row, int64_t v_head, int64_t rows,
                               const int32_t *offsets, void *k_pages, void *v_pages, float *weights,
                               hipStream_t stream) {
    const int st = check_pages(p, weights != nullptr);
    if (st) return st;
    if (rows < 0 || k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0 || !offsets)
        return GS_ERR_INVALID_ARGUMENT;
    if (rows == 0 || p->sequences == 0 || p->pages == 0 || p->table_width == 0) return GS_OK;
    if (!k || !v || !k_pages || !v_pages) return GS_ERR_INVALID_ARGUMENT;
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) ||
        (k_row | k_head | v_row | v_head) % 8 != 0)
        return GS_ERR_UNSUPPORTED;
    const int64_t groups = (rows * (p->dim / 8) * p->heads + 255) / 256;
    if (rows > kMaxSlots || groups > 0x7fffffffLL) return GS_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)groups), dim3(256), 0, stream, *p,
                       (const uint16_t *)k, k_row, k_head, (const uint16_t *)v, v_row, v_head, rows,
                       offsets, (uint16_t *)k_pages, (uint16_t *)v_pages, weights);
    return launch_status();
}

extern "C" int gs_paged_evict(const GsPages *p, void *k_pages, void *v_pages, float *weights,
                              const int32_t *new_tables, int64_t new_stride, int32_t new_width,
                              int32_t keep, int32_t recent, int32_t *new_lengths, int32_t *kept,
                              hipStream_t stream) {
    const int st = check_pages(p, true);
    if (st) return st;
    if (keep < 1 || recent < 0 || recent > keep || new_stride < 0 || new_width < 0 ||
        (int64_t)new_width * p->page_size < keep)
        return GS_ERR_INVALID_ARGUMENT;
    if (p->sequences == 0) return GS_OK;
    if (!new_tables || !new_lengths || !kept || (p->pages > 0 && (!k_pages || !v_pages || !weights)))
        return GS_ERR_INVALID_ARGUMENT;
    if (!aligned16(k_pages) || !aligned16(v_pages)) return GS_ERR_UNSUPPORTED;
    const int64_t pick = (int64_t)p->sequences * p->heads;
    const int64_t groups = ((int64_t)keep * (p->dim / 8) * p->heads + 255) / 256;
    if (pick > 0x7fffffffLL || groups > 0x7fffffffLL || p->sequences > 65535)
        return GS_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(paged_pick_kernel, dim3((unsigned)pick), dim3(kPick), 0, stream, *p,
                       (const float *)weights, keep, recent, new_lengths, kept);
    hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)groups, (unsigned)p->sequences), dim3(256),
                       0, stream, *p, (uint16_t *)k_pages, (uint16_t *)v_pages, weights, new_tables,
                       new_stride, keep, (const int32_t *)kept);
    return launch_status();
}
