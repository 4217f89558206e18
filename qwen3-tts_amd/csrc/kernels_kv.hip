// The paged key/value cache of the token-step operators: rows written (as they are or in 8 bits) and read back.
//
// Mathematics: 8-bit rows hold x ~ code * s with one s = max|x| * (1 / TOP) per token and key head (ops_device.h).  Both kernels are one
// pass over the rows and are bound by memory: a write reads A and writes S bytes per value (+ 4 per row), a read the reverse.
// Layout: head_dim / 8 lanes hold a row, eight values each, so the row's maximum is a butterfly over 8 or 16 neighbouring lanes and
// every access is 16 bytes (8 for 8-bit codes) of a contiguous row.  A wave has one token and 64 / lanes-per-row of its 2 * kv_heads
// rows: which sequence the token belongs to is then one question per wave, answered by a ballot over up to 64 of `cu` at a time
// (no chain of dependent loads as in a binary search), while the rows' own loads are already in flight.
#include "ops_device.h"

namespace hipvoc {

struct KvSlot { bool in; int64_t row, scale; };      // in: the token exists and its place is sound; row / scale: of key head 0

// Sequence and place of token `t` (the same for the whole wave); `lane` 0 .. 63
__device__ __forceinline__ KvSlot kv_slot(const KvMoveArgs &a, int t, int lane, bool &padding) {
    KvSlot s = {false, 0, 0};
    int seq = 0;
    for (int b0 = 0; b0 < a.r.n_seqs; b0 += 64) {
        const int b = b0 + lane;
        const bool before = b < a.r.n_seqs && a.r.cu[b + 1] <= t;
        const int n = __popcll(__ballot(before));
        seq += n;
        if (n < 64) break;
    }
    padding = seq >= a.r.n_seqs;
    if (padding) return s;
    const int64_t pos = row_position(t, a.r.cu[seq], a.r.first[seq], a.r.table_width, a.page_shift);
    if (pos < 0) {
        if (lane == 0) raise(a.err, OPS_ERR_POSITION);
        return s;
    }
    const int page = a.r.table[seq * a.r.table_stride + (pos >> a.page_shift)], at = (int)(pos & (a.c.page - 1));
    if (!page_ok(page, a.c.n_pages)) {
        if (lane == 0) raise(a.err, OPS_ERR_PAGE);
        return s;
    }
    s.in = true;
    s.row = page * a.c.page_stride + (int64_t)at * a.c.head_dim;
    s.scale = (int64_t)page * a.c.kv_heads * a.c.page + at;
    return s;
}

// A wave takes KV_U times 64 lanes' worth of its token's rows, all their loads ahead of the question where they belong.
template <int ACT, int ST, int HD>
__global__ __launch_bounds__(256) void kv_write_kernel(KvMoveArgs a, int parts) {
    constexpr int LPR = HD / 8, RPW = 64 / LPR;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, t = (int)(w / parts), row0 = (int)(w % parts) * RPW * KV_U + lane / LPR, d = (lane % LPR) * 8;
    if (t >= a.n_rows) return;
    typedef typename Store<ACT>::type act_t;
    typedef typename Store<ST>::type st_t;
    Raw8<ACT> raw[KV_U];
#pragma unroll
    for (int u = 0; u < KV_U; u++) {
        const int row = row0 + u * RPW, value = row >= a.c.kv_heads, head = value ? row - a.c.kv_heads : row;
        if (row < 2 * a.c.kv_heads) raw[u] = load_raw8<ACT>((const act_t *)(value ? a.v : a.k) + t * (value ? a.v_stride : a.k_stride) + head * HD + d);
    }
    bool padding;
    const KvSlot s = kv_slot(a, t, lane, padding);
    if (!s.in) return;                                                   // the whole wave: a wave has one token
#pragma unroll
    for (int u = 0; u < KV_U; u++) {
        const int row = row0 + u * RPW, value = row >= a.c.kv_heads, head = value ? row - a.c.kv_heads : row;
        const bool mine = row < 2 * a.c.kv_heads;
        st_t *dst = (st_t *)(value ? a.c.v : a.c.k) + s.row + (int64_t)head * a.c.page * HD + d;
        if constexpr (ST == ACT) {
            if (mine) store_raw8<ACT>(dst, raw[u]);
        } else {
            float x[8];
            load8<ACT>(&raw[u], x);
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) m = amax_bits(m, x[i]);
            const float scale = scale8<ST>(__uint_as_float(amax_lanes(m, LPR)));
            if (mine) {
                *(u32x2 *)dst = Coder<ST>(scale).eight(x);
                if (d == 0) (value ? a.c.v_scale : a.c.k_scale)[s.scale + (int64_t)head * a.c.page] = scale;
            }
        }
    }
}

template <int ACT, int ST, int HD>
__global__ __launch_bounds__(256) void kv_read_kernel(KvMoveArgs a, int parts) {
    constexpr int LPR = HD / 8, RPW = 64 / LPR;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, t = (int)(w / parts), row0 = (int)(w % parts) * RPW * KV_U + lane / LPR, d = (lane % LPR) * 8;
    if (t >= a.n_rows) return;
    bool padding;
    const KvSlot s = kv_slot(a, t, lane, padding);
    if (padding) return;
    typedef typename Store<ACT>::type act_t;
    typedef typename Store<ST>::type st_t;
    Raw8<ST == ACT ? ACT : HIPVOC_T_BF16> raw[KV_U];
    u32x2 codes[KV_U];
    float scale[KV_U];
#pragma unroll
    for (int u = 0; u < KV_U; u++) {
        const int row = row0 + u * RPW, value = row >= a.c.kv_heads, head = value ? row - a.c.kv_heads : row;
        if (row < 2 * a.c.kv_heads && s.in) {
            const st_t *src = (const st_t *)(value ? a.c.v : a.c.k) + s.row + (int64_t)head * a.c.page * HD + d;
            if constexpr (ST == ACT) {
                raw[u] = load_raw8<ACT>(src);
            } else {
                codes[u] = *(const u32x2 *)src;
                scale[u] = (value ? a.c.v_scale : a.c.k_scale)[s.scale + (int64_t)head * a.c.page];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < KV_U; u++) {
        const int row = row0 + u * RPW, value = row >= a.c.kv_heads, head = value ? row - a.c.kv_heads : row;
        if (row >= 2 * a.c.kv_heads) continue;
        act_t *dst = (act_t *)(value ? a.v : a.k) + t * (value ? a.v_stride : a.k_stride) + head * HD + d;
        float x[8];
        if (s.in) {
            if constexpr (ST == ACT) {
                store_raw8<ACT>(dst, raw[u]);
                continue;
            } else {
                load8<ST>(&codes[u], x);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] *= scale[u];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __builtin_nanf("");
        }
        store8<ACT>(dst, x);
    }
}

template <int ACT, int ST, int HD> static hipError_t kv_go(const KvMoveArgs &a, bool write, hipStream_t s) {
    const int parts = kv_parts(a.c.kv_heads, HD);
    const unsigned blocks = (unsigned)(((int64_t)a.n_rows * parts + 3) / 4);
    if (write) kv_write_kernel<ACT, ST, HD><<<blocks, 256, 0, s>>>(a, parts);
    else kv_read_kernel<ACT, ST, HD><<<blocks, 256, 0, s>>>(a, parts);
    return hipGetLastError();
}
template <int ACT, int ST> static hipError_t kv_hd(const KvMoveArgs &a, bool write, hipStream_t s) {
    return a.c.head_dim == 64 ? kv_go<ACT, ST, 64>(a, write, s) : kv_go<ACT, ST, 128>(a, write, s);
}
template <int ACT> static hipError_t kv_st(const KvMoveArgs &a, bool write, hipStream_t s) {
    if (a.c.dtype == HIPVOC_T_INT8) return kv_hd<ACT, HIPVOC_T_INT8>(a, write, s);
    if (a.c.dtype == HIPVOC_T_E4M3) return kv_hd<ACT, HIPVOC_T_E4M3>(a, write, s);
    return kv_hd<ACT, ACT>(a, write, s);
}
static hipError_t kv_act(const KvMoveArgs &a, bool write, hipStream_t s) {
    if (a.dtype == HIPVOC_T_F32) return kv_st<HIPVOC_T_F32>(a, write, s);
    if (a.dtype == HIPVOC_T_F16) return kv_st<HIPVOC_T_F16>(a, write, s);
    return kv_st<HIPVOC_T_BF16>(a, write, s);
}

__global__ void take_error_kernel(int *err, int word) { err[word] = atomicExch(err, 0); }
hipError_t launch_take_error(int *err, int word, hipStream_t s) {
    take_error_kernel<<<1, 1, 0, s>>>(err, word);
    return hipGetLastError();
}

hipError_t launch_kv_write(const KvMoveArgs &a, hipStream_t s) { return kv_act(a, true, s); }
hipError_t launch_kv_read(const KvMoveArgs &a, hipStream_t s) { return kv_act(a, false, s); }

}  // namespace hipvoc
