// A paged cache's bookkeeping: new keys and values into its pages, and the keys that matter
// moved to fewer pages.

#include "paged.h"
#include "wave_ops.h"

namespace gs {

using Chunk = __attribute__((ext_vector_type(4))) uint32_t;  // 8 elements

// --------------------------------------------------------------------- append
// A thread copies 8 elements of a row's keys and values; a row's threads are neighbours.  The
// row's sequence is found by bisection of the offsets.  Bound by memory: 65280 rows of 4 heads of
// 128, 53 us, 5.1 TB/s, a large copy's rate; 16 rows 3.3 us.
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
        const int middle = low + (high - low) / 2;  // (the sum of both may pass 32 bits)
        if (offsets[middle] <= row)
            low = middle + 1;
        else
            high = middle;
    }
    const int b = low - 1;
    if (b < 0 || b >= p.sequences) return;
    const int64_t end = offsets[b + 1] < rows ? offsets[b + 1] : rows;
    // (not by the length as the table clamps it, which would be an earlier token's slot)
    const int64_t slot = p.lengths[b] - (end - row);
    if (slot < 0 || slot >= (int64_t)p.page_size * p.table_width) return;
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
// infinity.  No weight's is 0, nor kRecent, which is above all.
constexpr uint32_t kRecent = 0xffffffffu, kLargest = 0xfffffffeu;
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return kLargest;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);  // -0 + 0 = 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kPick = 1024, kPickWaves = kPick / kWave;
constexpr int kDigit = 11, kBins = 1 << kDigit;
constexpr int kHeld = 32 * kPick;  // slots whose orders fit in LDS
constexpr int kUnroll = 4;

// Of 64 slots, for each of the waves, to cover so many.
__host__ __device__ __forceinline__ int rounds_of(int64_t slots) {
    return (int)((slots + kUnroll * kPick - 1) / (kUnroll * kPick)) * kUnroll;
}

struct PickShared {
    uint32_t histogram[kBins];
    uint32_t waves[2][kPickWaves];  // counts of each wave
    uint32_t found[3];
};

// Sums over the waves before this one, or all, of a count that each wave has left.
__device__ __forceinline__ uint32_t sum_of_waves(const uint32_t *counts, int before) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kPickWaves; ++w) sum += w < before ? counts[w] : 0;
    return sum;
}

// How many of the lanes before this one are in a mask.
__device__ __forceinline__ uint32_t lanes_before(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Which slots of a sequence and head stay: a workgroup, each wave a stretch of slots that follow
// one another, 64 at a time.  HELD: the slots' orders stay in LDS, else they are read again for
// every pass.  WHOLE: 64 slots lie in one page, which a lane of the wave finds for all of them.  The
// smallest order that stays is found by its digits from the highest, with a histogram of the slots
// that agree so far; then each wave counts what it keeps, and writes it behind what the waves before
// it keep.
//
// Bound by the instructions of one CU: reading and the first histogram are a third of the time for
// 32640 slots, then its scan, a second histogram, counting and writing.  64 heads of 2500 to 32640 slots
// 25 us, 3 of 16320 in pages of 40 16, 18 of up to 60 10.  For the first, orders in registers, whose
// loops have to be unrolled, took 64 us, a page found for every slot 45, and digits under masks, with the
// recent slots told by their numbers, 29.
template <bool HELD, bool WHOLE>
__device__ __forceinline__ void pick(const GsPages &p, const float *weights, int b, int head, int filled,
                                     int32_t keep, int32_t recent, int32_t *new_lengths, int32_t *out,
                                     PickShared &shared, uint32_t *orders) {
    const int t = threadIdx.x, lane = t % kWave, wave = uniform(t / kWave);
    const int old = max(filled - recent, 0);
    const int rounds = rounds_of(filled);            // of a wave
    const int first = wave * rounds * kWave + lane;  // the lane's first slot
    const int more_pages = kWave / p.page_size, more_places = kWave - more_pages * p.page_size;
    // f(slot, order) for the lane's slots in turn; the order of a slot that is not there is 0, that of
    // a recent one kRecent.  Pages and weights of BATCH slots are on their way at a time.
    const auto from_memory = [&](auto f) {
        constexpr int BATCH = 16;
        const auto put = [&](int slot, bool is, float w) {
            f(slot, !is ? 0u : slot >= old ? kRecent : order_of(w));
        };
        if constexpr (WHOLE) {
            // a lane looks for the page of a round's 64 slots
            for (int i0 = 0; i0 < rounds; i0 += kWave) {
                const int begin = (wave * rounds + i0 + lane) * kWave, index = begin / p.page_size;
                const bool is = i0 + lane < rounds && begin < filled;
                const int mine = is ? page_of(p, b, index) : -1, place = begin - index * p.page_size;
                const float *line = weights + lane * p.sum_slot;
                for (int j0 = 0; j0 < kWave && i0 + j0 < rounds; j0 += BATCH) {
                    float w[BATCH];
                    bool has[BATCH];
#pragma unroll
                    for (int j = 0; j < BATCH; ++j) {
                        const int page = __builtin_amdgcn_readlane(mine, j0 + j);
                        has[j] = page >= 0 && first + (i0 + j0 + j) * kWave < filled;
                        const int64_t at = sum_at(p, page, __builtin_amdgcn_readlane(place, j0 + j), head);
                        w[j] = has[j] ? line[at] : 0.0f;
                    }
#pragma unroll
                    for (int j = 0; j < BATCH; ++j)
                        if (i0 + j0 + j < rounds)
                            put(first + (i0 + j0 + j) * kWave, has[j], w[j]);
                }
            }
        } else {
            int index = first / p.page_size, place = first - index * p.page_size;
            for (int i0 = 0; i0 < rounds; i0 += BATCH) {
                int pages[BATCH], places[BATCH];
                float w[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const bool is = i0 + i < rounds && first + (i0 + i) * kWave < filled;
                    pages[i] = is ? page_of(p, b, index) : -1;
                    places[i] = place;
                    index += more_pages;
                    place += more_places;
                    if (place >= p.page_size) place -= p.page_size, ++index;
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i)
                    w[i] = pages[i] >= 0 ? weights[sum_at(p, pages[i], places[i], head)] : 0.0f;
#pragma unroll
                for (int i = 0; i < BATCH; ++i)
                    if (i0 + i < rounds) put(first + (i0 + i) * kWave, pages[i] >= 0, w[i]);
            }
        }
    };
    const auto each = [&](auto f) {
        if constexpr (HELD) {
            for (int slot = first, i = 0; i < rounds; i += kUnroll, slot += kUnroll * kWave) {
                uint32_t some[kUnroll];
#pragma unroll
                for (int n = 0; n < kUnroll; ++n) some[n] = orders[slot + n * kWave];
#pragma unroll
                for (int n = 0; n < kUnroll; ++n) f(slot + n * kWave, some[n]);
            }
        } else {
            from_memory(f);
        }
    };
    // orders, how many there are, and the histogram of the highest digit
    for (int i = t; i < kBins; i += kPick) shared.histogram[i] = 0;
    __syncthreads();
    uint32_t there = 0, there_old = 0;
    from_memory([&](int slot, uint32_t order) {
        if (HELD) orders[slot] = order;
        const bool counts = order - 1 < kRecent - 1;
        there += __popcll(__ballot(order != 0));
        there_old += __popcll(__ballot(counts));
        if (counts) atomicAdd(&shared.histogram[order >> (32 - kDigit)], 1u);
    });
    if (lane == 0) shared.waves[0][wave] = there, shared.waves[1][wave] = there_old;
    __syncthreads();
    const uint32_t all = sum_of_waves(shared.waves[0], kPickWaves);
    const uint32_t all_old = sum_of_waves(shared.waves[1], kPickWaves);
    __syncthreads();
    // `want` of the old slots stay: orders above `high`, and the first `need` from `low` to `high`
    const uint32_t want = min((uint32_t)keep - (all - all_old), all_old);
    uint32_t low = kLargest, high = kLargest, need = 0;  // none
    if (want == all_old) low = high = 0;                 // all
    if (want > 0 && want < all_old) {
        low = 0;
        need = want;
        for (int shift = 32 - kDigit, digit = kDigit;;) {
            // bins from the largest down, two a thread: the one in which the count passes need
            const int bin = kBins - 1 - 2 * t;
            const uint32_t one = shared.histogram[bin], two = shared.histogram[bin - 1];
            shared.histogram[bin] = shared.histogram[bin - 1] = 0;
            const uint32_t upto = lanes_sum_upto(one + two);
            if (lane == kWave - 1) shared.waves[0][wave] = upto;
            __syncthreads();
            const uint32_t before = upto - one - two + sum_of_waves(shared.waves[0], wave);
            if (before < need && need <= before + one + two) {
                const bool second = need > before + one;
                shared.found[0] = second ? bin - 1 : bin;
                shared.found[1] = need - before - (second ? one : 0);
                shared.found[2] = second ? two : one;
            }
            __syncthreads();
            low |= shared.found[0] << shift;
            high = min(low | ((1u << shift) - 1), kLargest);
            need = shared.found[1];
            // (done too where all with these digits stay)
            if (shift == 0 || need == shared.found[2]) break;
            digit = min(shift, kDigit);
            shift -= digit;
            const auto bin_of = [&](uint32_t order) { return order >> shift & ((1u << digit) - 1); };
            if (shared.found[2] > all_old / 4) {
                // (they may all be alike, such as zeros, and additions to one place follow one
                // another: one for a wave whose lanes agree.  With all weights alike the eviction of
                // up to 32640 slots takes 124 us and 167 without; taken always, this costs the others 5)
                each([&](int, uint32_t order) {
                    const bool counts = order - low <= high - low;
                    const uint32_t mine = bin_of(order), first_bin = uniform((int)mine);
                    const uint64_t some = __ballot(counts);
                    if (!__ballot(counts && mine != first_bin)) {
                        if (lane == 0 && some)
                            atomicAdd(&shared.histogram[first_bin], (uint32_t)__popcll(some));
                    } else if (counts) {
                        atomicAdd(&shared.histogram[mine], 1u);
                    }
                });
            } else {
                each([&](int, uint32_t order) {
                    if (order - low <= high - low) atomicAdd(&shared.histogram[bin_of(order)], 1u);
                });
            }
            __syncthreads();
        }
    }
    uint32_t sure = 0, equal = 0;
    each([&](int, uint32_t order) {
        sure += __popcll(__ballot(order > high));
        equal += __popcll(__ballot(order - low <= high - low));
    });
    __syncthreads();
    if (lane == 0) shared.waves[0][wave] = sure, shared.waves[1][wave] = equal;
    __syncthreads();
    uint32_t equals = sum_of_waves(shared.waves[1], wave);
    uint32_t written = sum_of_waves(shared.waves[0], wave) + min(equals, need);
    each([&](int slot, uint32_t order) {
        bool stays = order > high;
        const bool same = order - low <= high - low;
        const uint64_t alike = __ballot(same);
        if (alike && equals < need) {
            stays = stays || (same && equals + lanes_before(alike) < need);
            equals += __popcll(alike);
        }
        const uint64_t stay = __ballot(stays);
        const uint32_t to = written + lanes_before(stay);
        if (stays && to < (uint32_t)keep) out[to] = slot;
        written += __popcll(stay);
    });
    const uint32_t stayed = all - all_old + want;
    for (int j = stayed + t; j < keep; j += kPick) out[j] = -1;
    if (head == 0 && t == 0) new_lengths[b] = (int32_t)stayed;
}

template <bool HELD, bool WHOLE>
__global__ __launch_bounds__(kPick) void paged_pick_kernel(GsPages p,
                                                           const float *__restrict__ weights,
                                                           int32_t keep, int32_t recent,
                                                           int32_t *__restrict__ new_lengths,
                                                           int32_t *__restrict__ kept) {
    __shared__ PickShared shared;
    extern __shared__ uint32_t orders[];
    const int b = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
    pick<HELD, WHOLE>(p, weights, b, head, filled_slots(p, b), keep, recent, new_lengths,
               kept + (int64_t)blockIdx.x * keep, shared, orders);
}

// The picked slots to the new pages: a thread moves 8 elements of a key and a value.  Bound by memory:
// 8160 of 32640 slots and fewer in 16 sequences, 4 heads of 128, 76 us, 4.8 TB/s, 95% of a large copy's rate.
__global__ __launch_bounds__(256) void paged_move_kernel(GsPages p, uint16_t *k_pages,
                                                         uint16_t *v_pages, float *weights,
                                                         const int32_t *__restrict__ new_tables,
                                                         int64_t new_stride, int32_t keep,
                                                         const int32_t *__restrict__ kept) {
    const int chunks = p.dim / 8, a_row = chunks * p.heads;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = at / a_row;
    if (row >= keep) return;
    const int rest = (int)(at - row * a_row), head = rest / chunks, chunk = rest - head * chunks;
    const int j = (int)row, index = j / p.page_size, to_place = j - index * p.page_size;
    const int64_t b = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    if (b >= p.sequences) return;
    const int slot = kept[(b * p.heads + head) * keep + j];
    const int to_page = new_tables[b * new_stride + index];
    if (slot < 0 || (uint32_t)to_page >= (uint64_t)p.pages) return;
    const int page = page_of(p, (int)b, slot / p.page_size), place = slot % p.page_size;
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
    constexpr int64_t most = 0x7fffffff;
    if (p->page_stride > most || p->head_stride > most ||
        (weights && (p->sum_page > most || p->sum_slot > most || p->sum_head > most)))
        return GS_ERR_UNSUPPORTED;
    if (p->type == GS_F32 || p->dim % 8 != 0 || p->dim > GS_MAX_HEAD_DIM ||
        p->pages > 0x7fffffffLL || (int64_t)p->page_size * p->table_width > kMaxSlots ||
        p->sequences > kMaxSlots || p->page_size > kMaxSlots || (int64_t)p->heads * (p->dim / 8) > kMaxSlots ||
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
    if (rows > kMaxSlots || !launchable(groups, 256)) return GS_ERR_UNSUPPORTED;
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
    const int64_t picks = (int64_t)p->sequences * p->heads;
    const int64_t groups = ((int64_t)keep * (p->dim / 8) * p->heads + 255) / 256;
    if (keep > kMaxSlots || !launchable(picks, kPick) || !launchable(groups, 256)) return GS_ERR_UNSUPPORTED;
    // (by the slots that a table could hold: what is filled is not known here)
    const int64_t slots = (int64_t)p->page_size * p->table_width;
    const bool held = slots <= kHeld, whole = p->page_size % kWave == 0;
    const unsigned lds = held ? (unsigned)(rounds_of(slots) * kPick * sizeof(uint32_t)) : 0;
    const auto kernel = held ? whole ? paged_pick_kernel<true, true> : paged_pick_kernel<true, false>
                             : whole ? paged_pick_kernel<false, true> : paged_pick_kernel<false, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)picks), dim3(kPick), lds, stream, *p,
                       (const float *)weights, keep, recent, new_lengths, kept);
    const int picked = launch_status();
    if (picked) return picked;  // (what moves is what has been picked)
    const int32_t rows = p->sequences < 65535 ? p->sequences : 65535;  // of the grid's second dimension
    hipLaunchKernelGGL(paged_move_kernel,
                       dim3((unsigned)groups, (unsigned)rows, (unsigned)((p->sequences + rows - 1) / rows)),
                       dim3(256), 0, stream, *p, (uint16_t *)k_pages, (uint16_t *)v_pages, weights, new_tables,
                       new_stride, keep, (const int32_t *)kept);
    return launch_status();
}
