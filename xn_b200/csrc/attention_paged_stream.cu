// Attention of few query rows over a paged cache, or of small calls: the keys and values stream through once for 16 rows, from HBM.
//
// Work is counted in units of 16 keys of one (sequence, tile of rows, key head) item, all items laid end to end, and dealt out
// evenly to the warps of the machine, whatever the lengths: a long context is shared by many warps, short ones follow one
// another in a warp.  The rows of an item are the query heads of one key head, for one or more tokens: up to 8 x NT of them.
//
// A warp keeps its own ring of units in shared memory, filled with 16-byte asynchronous copies (rows of a unit may lie in any
// pages) and never waits for another warp while it streams.  Per unit, on mma.sync:
//   S^T = K Q^T   16 keys x 8 rows per product, Q's fragments stay in registers
//   running maximum and sum of every row (a lane owns two rows' columns), p = 2^(s - m)
//   O^T += V^T P^T, V's fragments by transposing loads, P^T turned in registers
// Keys ride the 16-row dimension, rows the 8-column one: with one to eight rows (a token's heads) half of what the other way
// round would cost, which keeps the products well below the time that the unit's bytes take to arrive.  P is rounded to the
// element type for the second product (half a step, 2^-8 of each in bf16 and 2^-11 in f16, as the output's own rounding); scores,
// maxima, sums and O stay in f32.
//
// A warp that holds the whole of an item writes its rows; parts are joined within the CTA through shared memory, and what
// crosses CTAs (at most two records of each) by a second kernel.
#include "paged.cuh"

namespace xn {
namespace {

__device__ __forceinline__ unsigned smem_addr(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(unsigned dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
    unsigned y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int UNIT = 16;  // keys

// The units of a sequence: kv_heads * tiles items of U units each.
struct SequenceUnits {
    Sequence s;
    int lo;      // first key that any row sees
    int base;    // the same, down to a multiple of the unit
    int U, tiles;
    __device__ __forceinline__ unsigned long long total(const PagedArgs &a) const {
        return (unsigned long long)U * (unsigned)tiles * (unsigned)a.kv_heads;
    }
};
template <int TR> __device__ __forceinline__ SequenceUnits sequence_units(const PagedArgs &a, int b) {
    SequenceUnits u;
    u.s = load_sequence(a, b);
    u.lo = first_key(a, u.s.off);
    u.base = u.lo / UNIT * UNIT;
    u.U = max(1, (u.s.ctx - u.base + UNIT - 1) / UNIT);  // rows that see nothing get their zeros from an empty unit
    u.tiles = (int)(((long long)u.s.n * a.group + TR - 1) / TR);
    return u;
}

// A place in the line of all units.
struct Cursor {
    unsigned long long pos;
    int b, head, tile, unit;
    SequenceUnits u;
};
template <int TR> __device__ __forceinline__ void next_sequence(const PagedArgs &a, Cursor &c) {
    for (++c.b; c.b < a.batch; ++c.b) {
        c.u = sequence_units<TR>(a, c.b);
        if (c.u.tiles) break;
    }
    c.head = c.tile = c.unit = 0;
}
template <int TR> __device__ __forceinline__ void advance(const PagedArgs &a, Cursor &c) {
    ++c.pos;
    if (++c.unit < c.u.U) return;
    c.unit = 0;
    if (++c.tile < c.u.tiles) return;
    c.tile = 0;
    if (++c.head < a.kv_heads) return;
    next_sequence<TR>(a, c);
}

// One warp's or CTA's part of an item, in shared memory: O [rows][HD], then m, l
struct PartHead {
    unsigned long long begin, end;  // units of the item; end == 0: none
    int q0, rows, tile_row, head;
};

template <typename T, int HD, int NT, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) paged_stream_kernel(const PagedArgs a) {
    constexpr int TR = 8 * NT, CHUNKS = HD / 8, ROWS_AT_ONCE = 32 / CHUNKS;
    constexpr int ROW_BYTES = HD * 2, TILE = UNIT * ROW_BYTES, STAGE = 2 * TILE;
    constexpr int REC = TR * (HD + 2);
    static_assert(REC * 4 <= STAGES * STAGE, "a warp's last part takes the place of its ring");
    extern __shared__ __align__(1024) unsigned char smem[];
    float *recs = reinterpret_cast<float *>(smem + WARPS * STAGES * STAGE);  // first parts, one per warp
    __shared__ unsigned long long scan[WARPS + 1];
    __shared__ unsigned long long start_base[WARPS];
    __shared__ int start_b[WARPS];
    __shared__ PartHead heads[2 * WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    dependent_begin();

    // ---- where every warp's share begins: all sequences' units, added up in order ----
    unsigned long long total = 0;
    auto block_scan = [&](unsigned long long x, unsigned long long &sum) {  // exclusive
        unsigned long long inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = inc;
        __syncthreads();
        unsigned long long before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += scan[w];
            all += scan[w];
        }
        sum = all;
        return before + inc - x;
    };
    const int rounds = (a.batch + WARPS * 32 - 1) / (WARPS * 32);
    unsigned long long mine = 0, at = 0;
    for (int r = 0; r < rounds; ++r) {
        const int b = r * WARPS * 32 + (int)threadIdx.x;
        mine = b < a.batch ? sequence_units<TR>(a, b).total(a) : 0;
        unsigned long long sum;
        at = block_scan(mine, sum);
        total += sum;
    }
    const Shares shares(total, gridDim.x * WARPS);
    const unsigned long long bound = shares.begin(blockIdx.x * WARPS + min(lane, WARPS));  // lane w: where warp w's share begins
    unsigned long long seen = 0;
    for (int r = 0; r < rounds; ++r) {
        const int b = r * WARPS * 32 + (int)threadIdx.x;
        unsigned long long sum = total;
        if (rounds > 1) {
            mine = b < a.batch ? sequence_units<TR>(a, b).total(a) : 0;
            at = block_scan(mine, sum);
        }
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const unsigned long long p = __shfl_sync(0xffffffffu, bound, w);
            if (p >= seen + at && p < seen + at + mine) {
                start_b[w] = b;
                start_base[w] = seen + at;
            }
        }
        seen += sum;
    }
    if (lane == 0) heads[2 * warp].end = heads[2 * warp + 1].end = 0;
    __syncthreads();
    const unsigned long long first = __shfl_sync(0xffffffffu, bound, warp), last = __shfl_sync(0xffffffffu, bound, warp + 1);

    unsigned char *ring = smem + warp * STAGES * STAGE;
    auto store_part = [&](int which, const Cursor &c, const float (&o)[HD / 16][NT][4], const float (&m)[NT][2], const float (&l)[NT][2]) {
        float *rec = which == 0 ? recs + warp * REC : reinterpret_cast<float *>(ring);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = nt * 8 + (lane & 3) * 2 + e;
#pragma unroll
                for (int mt = 0; mt < HD / 16; ++mt) {
                    rec[row * HD + mt * 16 + (lane >> 2)] = o[mt][nt][e];
                    rec[row * HD + mt * 16 + 8 + (lane >> 2)] = o[mt][nt][2 + e];
                }
                if (lane < 4) {
                    rec[TR * HD + row] = m[nt][e];
                    rec[TR * HD + TR + row] = l[nt][e];
                }
            }
    };
    if (first < last) {
        Cursor pc;  // what is loaded next
        pc.pos = first;
        pc.b = start_b[warp];
        pc.u = sequence_units<TR>(a, pc.b);
        {
            unsigned long long item, unit;
            divide(first - start_base[warp], (unsigned)pc.u.U, item, unit);
            pc.unit = (int)unit;
            pc.head = (int)((unsigned)item / (unsigned)pc.u.tiles);
            pc.tile = (int)((unsigned)item % (unsigned)pc.u.tiles);
        }
        Cursor cc = pc;  // what is computed next
        int page = -1;   // the page of this lane's key in the unit at pc: read one unit ahead
        auto key_of = [&](const Cursor &c) { return c.u.base + c.unit * UNIT + (lane & 15); };
        auto page_of = [&](int key) { return a.page_shift >= 0 ? key >> a.page_shift : (int)((unsigned)key / (unsigned)a.page_size); };
        auto fetch_page = [&](const Cursor &c) {
            const int key = key_of(c);
            return c.pos < last && key >= c.u.lo && key < c.u.s.ctx ? a.table[(long long)c.b * a.table_stride + page_of(key)] : -1;
        };
        auto issue = [&](int slot, int page) {
            if (pc.pos < last) {
                const int key = key_of(pc);
                const bool there = page >= 0 && page < a.num_pages;
                const long long at_row = there ? (long long)page * a.page_stride + (long long)pc.head * a.head_stride +
                                                     (long long)(key - page_of(key) * a.page_size) * a.row_stride
                                               : -1;
                const unsigned kdst = smem_addr(ring + slot * STAGE), vdst = kdst + TILE;
                const int chunk = lane % CHUNKS;
#pragma unroll
                for (int i = 0; i < UNIT / ROWS_AT_ONCE; ++i) {
                    const int row = i * ROWS_AT_ONCE + lane / CHUNKS;
                    const long long off = __shfl_sync(0xffffffffu, at_row, row);
                    const bool valid = off >= 0;
                    const long long e = valid ? off + chunk * 8 : 0;
                    const unsigned d = (unsigned)(row * ROW_BYTES + ((chunk ^ (row & 7)) << 4));
                    cp_async16(kdst + d, static_cast<const T *>(a.k) + e, valid);
                    cp_async16(vdst + d, static_cast<const T *>(a.v) + e, valid);
                }
                advance<TR>(a, pc);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        {
            int pages[STAGES];
            Cursor c = pc;
#pragma unroll
            for (int s = 0; s < STAGES; ++s) {
                pages[s] = fetch_page(c);
                if (c.pos < last) advance<TR>(a, c);
            }
#pragma unroll
            for (int s = 0; s < STAGES - 1; ++s) issue(s, pages[s]);
            page = pages[STAGES - 1];
        }

        unsigned qf[HD / 16][NT][2];
        float o[HD / 16][NT][4], m[NT][2], l[NT][2];
        int hi_key[NT][2], lo_key[NT][2];
        int sure_hi = 0, sure_lo = 0;  // the keys that all rows of the item see
        bool fresh = true;
        unsigned long long item_begin = 0;
        int slot = 0;
        while (cc.pos < last) {
            if (fresh) {
                fresh = false;
                item_begin = cc.pos - (unsigned)cc.unit;
                const int rows = (int)min((long long)cc.u.s.n * a.group - (long long)cc.tile * TR, (long long)TR);
                sure_hi = cc.u.s.off + (int)((unsigned)(cc.tile * TR) / (unsigned)a.group);
                sure_lo = first_key(a, cc.u.s.off + (int)((unsigned)(cc.tile * TR + rows - 1) / (unsigned)a.group));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int rq = nt * 8 + (lane >> 2);  // the row of this lane's Q fragments
                    const unsigned r = (unsigned)(cc.tile * TR + rq);
                    const T *qp = static_cast<const T *>(a.q) + (long long)(cc.u.s.q0 + (int)(r / (unsigned)a.group)) * a.q_token +
                                  (long long)(cc.head * a.group + (int)(r % (unsigned)a.group)) * a.q_head + (lane & 3) * 2;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        qf[kk][nt][0] = rq < rows ? *reinterpret_cast<const unsigned *>(qp + kk * 16) : 0u;
                        qf[kk][nt][1] = rq < rows ? *reinterpret_cast<const unsigned *>(qp + kk * 16 + 8) : 0u;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int rs = nt * 8 + (lane & 3) * 2 + e;  // the row of this lane's scores
                        const int i = (int)((unsigned)(cc.tile * TR + rs) / (unsigned)a.group);
                        hi_key[nt][e] = rs < rows ? min(cc.u.s.ctx - 1, cc.u.s.off + i) : -1;
                        lo_key[nt][e] = first_key(a, cc.u.s.off + i);
                        m[nt][e] = -INFINITY;
                        l[nt][e] = 0.0f;
                    }
#pragma unroll
                    for (int mt = 0; mt < HD / 16; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.0f;
                }
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();
            issue(slot == 0 ? STAGES - 1 : slot - 1, page);  // the slot of the unit before this one
            page = fetch_page(pc);

            const unsigned kt = smem_addr(ring + slot * STAGE), vt = kt + TILE;
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                unsigned kf[4];
                const int row = lane & 15, chunk = kk * 2 + (lane >> 4);
                ldmatrix_x4(kf, kt + row * ROW_BYTES + ((chunk ^ (row & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<T>(s[nt], kf, qf[kk][nt][0], qf[kk][nt][1]);
            }
            const int key0 = cc.u.base + cc.unit * UNIT + (lane >> 2), key1 = key0 + 8;
            unsigned pf[NT][2];
            bool moved = false;
            float alpha[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x0 = key0 <= hi_key[nt][e] && key0 >= lo_key[nt][e] ? s[nt][e] * a.c : -INFINITY;
                    const float x1 = key1 <= hi_key[nt][e] && key1 >= lo_key[nt][e] ? s[nt][2 + e] * a.c : -INFINITY;
                    float top = fmaxf(x0, x1);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float mn = fmaxf(m[nt][e], top);
                    alpha[nt][e] = mn == m[nt][e] ? 1.0f : exp2_fast(m[nt][e] - mn);
                    moved |= mn != m[nt][e];
                    m[nt][e] = mn;
                    const float ref = mn == -INFINITY ? 0.0f : mn;
                    p[e] = exp2_fast(x0 - ref);
                    p[2 + e] = exp2_fast(x1 - ref);
                    l[nt][e] = l[nt][e] * alpha[nt][e] + (p[e] + p[2 + e]);
                }
                pf[nt][0] = transpose8x8(pack2<T>(p[0], p[1]));
                pf[nt][1] = transpose8x8(pack2<T>(p[2], p[3]));
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int mt = 0; mt < HD / 16; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[mt][nt][e] *= alpha[nt][e & 1];
            }
            // A row of V that some rows see and others do not, and that is not finite, is taken for zeros (a product with the probability 0
            // would be NaN), and the rows that see it become NaN.  Beyond the context and before all windows it is zeros anyway.
            const int unit0 = cc.u.base + cc.unit * UNIT;
            if ((unit0 + UNIT - 1 > sure_hi && sure_hi < cc.u.s.ctx - 1) || (unit0 < sure_lo && cc.u.lo < sure_lo)) {
                const int key = unit0 + (lane & 15);  // two lanes a key
                unsigned char *row = ring + slot * STAGE + TILE + (lane & 15) * ROW_BYTES;
                NotFinite<T> check;
#pragma unroll
                for (int i = 0; i < CHUNKS / 2; ++i)
                    check.see(*reinterpret_cast<const uint4 *>(row + (((lane >> 4) * (CHUNKS / 2) + ((i ^ lane) & (CHUNKS / 2 - 1))) << 4)));
                unsigned which = __ballot_sync(0xffffffffu, check.any() && (key > sure_hi || key < sure_lo));
                if (which) {
                    which = (which | which >> 16) & 0xffffu;
                    if (which >> (lane & 15) & 1)
#pragma unroll
                        for (int i = 0; i < CHUNKS / 2; ++i)
                            *reinterpret_cast<uint4 *>(row + (((lane >> 4) * (CHUNKS / 2) + ((i ^ lane) & (CHUNKS / 2 - 1))) << 4)) = make_uint4(0, 0, 0, 0);
                    __syncwarp();
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            for (unsigned k = which; k; k &= k - 1) {
                                const int bad_key = unit0 + __ffs(k) - 1;
                                if (bad_key <= hi_key[nt][e] && bad_key >= lo_key[nt][e]) l[nt][e] = NAN;
                            }
                }
            }
#pragma unroll
            for (int mt = 0; mt < HD / 16; ++mt) {
                unsigned vf[4];
                const int row = (lane & 7) + ((lane >> 4) << 3), chunk = mt * 2 + ((lane >> 3) & 1);
                ldmatrix_x4_trans(vf, vt + row * ROW_BYTES + ((chunk ^ (row & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[mt][nt], vf, pf[nt][0], pf[nt][1]);
            }
            slot = slot + 1 == STAGES ? 0 : slot + 1;

            // ---- the end of the item, or of the share ----
            const bool item_done = cc.unit + 1 == cc.u.U;
            if (item_done || cc.pos + 1 == last) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
                const unsigned long long item_end = item_begin + (unsigned)cc.u.U;
                const long long all_rows = (long long)cc.u.s.n * a.group;
                if (item_begin >= first && item_end <= last) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const long long r = (long long)cc.tile * TR + nt * 8 + (lane & 3) * 2 + e;
                            if (r >= all_rows) continue;
                            const float inv = l[nt][e] == 0.0f ? 0.0f : 1.0f / l[nt][e];
                            T *dst = static_cast<T *>(a.out) + (long long)(cc.u.s.q0 + (int)((unsigned)r / (unsigned)a.group)) * a.out_token +
                                     (long long)(cc.head * a.group + (int)((unsigned)r % (unsigned)a.group)) * a.out_head + (lane >> 2);
#pragma unroll
                            for (int mt = 0; mt < HD / 16; ++mt) {
                                dst[mt * 16] = from_f32<T>(o[mt][nt][e] * inv);
                                dst[mt * 16 + 8] = from_f32<T>(o[mt][nt][2 + e] * inv);
                            }
                        }
                } else {
                    // the first part if the share begins inside the item, otherwise the last: by then the ring is drained
                    const int which = item_begin < first ? 0 : 1;
                    if (which == 1) {
                        asm volatile("cp.async.wait_group 0;" ::: "memory");
                        __syncwarp();
                    }
                    store_part(which, cc, o, m, l);
                    if (lane == 0)
                        heads[2 * warp + which] = PartHead{item_begin, item_end, cc.u.s.q0, (int)all_rows, cc.tile * TR, cc.head};
                }
                fresh = true;
            }
            advance<TR>(a, cc);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();

    // ---- parts of one item within the CTA are joined; what began before it or goes on behind it becomes a record ----
    const unsigned long long cta_first = __shfl_sync(0xffffffffu, bound, 0), cta_last = __shfl_sync(0xffffffffu, bound, WARPS);
    float *out_rec = part_records(a.ws, gridDim.x) + (size_t)blockIdx.x * 2 * REC;
    PartNote said{};
    auto rec_at = [&](int i) { return (i & 1) ? reinterpret_cast<const float *>(smem + (i >> 1) * STAGES * STAGE) : recs + (i >> 1) * REC; };
    // lane i looks after record i of the 2 * WARPS: those of one item follow one another
    const PartHead own = heads[min(lane, 2 * WARPS - 1)];
    const unsigned there = __ballot_sync(0xffffffffu, lane < 2 * WARPS && own.end != 0);
    const unsigned before = there & ((1u << lane) - 1);
    const unsigned long long begin_before = __shfl_sync(0xffffffffu, own.begin, before ? 31 - __clz(before) : 0);
    const unsigned leads = __ballot_sync(0xffffffffu, (there >> lane & 1) && (!before || begin_before != own.begin));
    for (unsigned todo = leads; todo; todo &= todo - 1) {
        const int i = __ffs(todo) - 1, j = todo & (todo - 1) ? __ffs(todo & (todo - 1)) - 1 : 32;
        const unsigned members = there & (j < 32 ? (1u << j) - 1 : ~0u) & ~((1u << i) - 1);
        const PartHead h = heads[i];
        const bool whole = h.begin >= cta_first && h.end <= cta_last;
        const int which = h.begin < cta_first ? 0 : 1;
        const int rows = min(h.rows - h.tile_row, TR);
        for (int row = warp; row < rows; row += WARPS) {
            const bool member = members >> lane & 1;
            const float *mine_rec = rec_at(member ? lane : i);
            const float m = member ? mine_rec[TR * HD + row] : -INFINITY, l = member ? mine_rec[TR * HD + TR + row] : 0.0f;
            const float mm = warp_max(m), w = mm == -INFINITY ? 0.0f : exp2_fast(m - mm), ll = warp_sum(w * l);
            float acc[HD / 32];
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) acc[e] = 0.0f;
            for (unsigned k = members; k; k &= k - 1) {
                const int at = __ffs(k) - 1;
                const float wk = __shfl_sync(0xffffffffu, w, at);
                const float *rec = rec_at(at) + row * HD + lane;
#pragma unroll
                for (int e = 0; e < HD / 32; ++e) acc[e] += wk * rec[e * 32];
            }
            if (whole) {
                const unsigned r = (unsigned)(h.tile_row + row);
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                T *dst = static_cast<T *>(a.out) + (long long)(h.q0 + (int)(r / (unsigned)a.group)) * a.out_token +
                         (long long)(h.head * a.group + (int)(r % (unsigned)a.group)) * a.out_head;
#pragma unroll
                for (int e = 0; e < HD / 32; ++e) dst[e * 32 + lane] = from_f32<T>(acc[e] * inv);
            } else {
                float *rec = out_rec + which * REC;
#pragma unroll
                for (int e = 0; e < HD / 32; ++e) rec[row * HD + e * 32 + lane] = acc[e];
                if (lane == 0) {
                    rec[TR * HD + row] = mm;
                    rec[TR * HD + TR + row] = ll;
                }
            }
        }
        if (!whole && which == 0) said.joined = 1;
        if (!whole && which == 1 && threadIdx.x == 0)
            said = PartNote{said.joined, (int)(shares.of(h.end - 1) / WARPS), h.q0, h.rows, h.tile_row, h.head};
    }
    if (threadIdx.x == 0) static_cast<PartNote *>(a.ws)[blockIdx.x] = said;
}

// Joins the records of the items that begin in one CTA of the kernel before and go on in others: record 1 of the first and the records 0
// of the CTAs behind it.  A thread holds 4 * NV columns of AT rows at once, a group of HD / (4 * NV) threads the rows.  Where an item has
// few records, the blocks of its first CTA join it and their groups take rows of their own.  Where it has many (a long context of few
// rows has one from every CTA), several groups share the records of the same rows, and the blocks of all its CTAs take rows of it; records
// are read a few at a time, before it is known whether they are there.  64 rows of 2 heads over 30000 keys on the tensor-memory kernel:
// 99 us with a row's records read one after another, 62 shared among groups, 22 among blocks too.  16 columns a thread in that kernel's
// case (4: twice the instructions for the weights of the records, a batch of chunks 65 to 68 us).
constexpr int MERGE_NT = 256, MANY_RECORDS = 8;
template <typename T, int HD, int NV, int AT, bool ALWAYS_SHARED>
__global__ void __launch_bounds__(MERGE_NT) paged_merge_kernel(const PagedArgs a, int rec_rows, int used) {
    constexpr int LANES = HD / (4 * NV), GROUPS = MERGE_NT / LANES, AHEAD = ALWAYS_SHARED ? 4 : 2;
    constexpr int SLICES = ALWAYS_SHARED ? GROUPS : MANY_RECORDS, TEAMS = GROUPS / SLICES;  // groups that share a row; rows at a time then
    __shared__ float sm[GROUPS][AT], sl[GROUPS][AT];
    __shared__ float4 so[GROUPS][AT][NV][LANES];
    __shared__ int helps;  // the first CTA of the item that goes on here and has many records
    const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    dependent_begin();
    const PartNote *notes = static_cast<const PartNote *>(a.ws);
    // threads look for an item that goes on here (there is one at most) while the block's own one is joined
    int found = -1;
    if (!ALWAYS_SHARED)
        for (int c = threadIdx.x; c < (int)blockIdx.x; c += MERGE_NT) {
            const int last = notes[c].last;
            if (last >= (int)blockIdx.x && last - c >= MANY_RECORDS) found = c;
        }
    const size_t rec_floats = part_record_floats(rec_rows, HD);
    const float *recs = part_records(a.ws, a.parts);
    struct Part {  // of a row
        float m, l;
        float4 o[NV];
    };
    auto join = [](Part &x, const Part &y) {
        const float mn = fmaxf(x.m, y.m), ref = mn == -INFINITY ? 0.0f : mn;
        const float w0 = exp2_fast(x.m - ref), w1 = exp2_fast(y.m - ref);
        x.l = x.l * w0 + y.l * w1;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            x.o[v].x = x.o[v].x * w0 + y.o[v].x * w1;
            x.o[v].y = x.o[v].y * w0 + y.o[v].y * w1;
            x.o[v].z = x.o[v].z * w0 + y.o[v].z * w1;
            x.o[v].w = x.o[v].w * w0 + y.o[v].w * w1;
        }
        x.m = mn;
    };
    for (int turn = 0; turn < (ALWAYS_SHARED ? 1 : 2); ++turn) {
        int first = blockIdx.x;
        if (turn == 1) {
            if (!__syncthreads_or(found >= 0)) break;
            if (found >= 0) helps = found;
            __syncthreads();
            first = helps;
        }
        const PartNote n = notes[first];
        if (n.last == 0) continue;
        const bool shared = ALWAYS_SHARED || n.last - first >= MANY_RECORDS;
        const int slices = shared ? SLICES : 1, slice = shared ? group % SLICES : 0;
        // rows: AT of every team at a time, dealt out to the blocks of the item's CTAs, or AT of every group
        const int teams = shared ? TEAMS : GROUPS, team = shared ? group / SLICES : group;
        const int turns_of = shared && !ALWAYS_SHARED ? n.last - first + 1 : 1;
        const int begin = ((turns_of == 1 ? 0 : (int)blockIdx.x - first) * (int)gridDim.y + (int)blockIdx.y) * teams * AT;
        auto is_row = [&](int row) { return row < rec_rows && (row & 127) < used && n.tile_row + (row >> 7) * used + (row & 127) < n.rows; };
        for (int b0 = begin; b0 < rec_rows; b0 += turns_of * (int)gridDim.y * teams * AT) {
            Part mine[AT];
            int rows[AT], item_rows[AT];
            bool any = false;
#pragma unroll
            for (int i = 0; i < AT; ++i) {
                const int row = b0 + team * AT + i;
                any |= is_row(row);
                rows[i] = is_row(row) ? row : -1;
                item_rows[i] = n.tile_row + (row >> 7) * used + (row & 127);
                mine[i].m = -INFINITY;
                mine[i].l = 0.0f;
#pragma unroll
                for (int v = 0; v < NV; ++v) mine[i].o[v] = make_float4(0, 0, 0, 0);
            }
            if (shared && !ALWAYS_SHARED ? !__syncthreads_or(any) : !any) continue;
            for (int c0 = first + slice; c0 <= n.last; c0 += AHEAD * slices) {
                int there[AHEAD];
                Part read[AHEAD][AT];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    const int c = min(c0 + k * slices, n.last);
                    const float *rec = recs + ((size_t)c * 2 + (c == first)) * rec_floats;
                    // not there: a share in which no key block of the item begins
                    there[k] = c0 + k * slices <= n.last && (c == first || notes[c].joined);
#pragma unroll
                    for (int i = 0; i < AT; ++i) {
                        const int row = max(rows[i], 0);
                        read[k][i].m = rec[rec_rows * HD + row];
                        read[k][i].l = rec[rec_rows * HD + rec_rows + row];
#pragma unroll
                        for (int v = 0; v < NV; ++v) read[k][i].o[v] = reinterpret_cast<const float4 *>(rec + (size_t)row * HD)[v * LANES + lane];
                    }
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                    if (there[k]) {
#pragma unroll
                        for (int i = 0; i < AT; ++i) {
                            if (k == 0 && !ALWAYS_SHARED && c0 == first) mine[i] = read[k][i];
                            else join(mine[i], read[k][i]);
                        }
                    }
            }
            if (shared) {  // group i of a team joins and writes the i-th of its rows
#pragma unroll
                for (int i = 0; i < AT; ++i) {
#pragma unroll
                    for (int v = 0; v < NV; ++v) so[group][i][v][lane] = mine[i].o[v];
                    if (lane == 0) { sm[group][i] = mine[i].m; sl[group][i] = mine[i].l; }
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < AT; ++i) {
                    if (i != slice) {
                        rows[i] = -1;
                        continue;
                    }
                    for (int g = 0; g < SLICES; ++g) {
                        Part other;
                        const int at = team * SLICES + g;
                        other.m = sm[at][i];
                        other.l = sl[at][i];
#pragma unroll
                        for (int v = 0; v < NV; ++v) other.o[v] = so[at][i][v][lane];
                        if (g == 0) mine[i] = other;
                        else join(mine[i], other);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < AT; ++i) {
                if (rows[i] < 0) continue;
                const unsigned r = (unsigned)item_rows[i];
                T *dst = static_cast<T *>(a.out) + (long long)(n.q0 + (int)(r / (unsigned)a.group)) * a.out_token +
                         (long long)(n.head * a.group + (int)(r % (unsigned)a.group)) * a.out_head;
                const float inv = mine[i].l == 0.0f ? 0.0f : 1.0f / mine[i].l;
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    uint2 w;
                    w.x = pack2<T>(mine[i].o[v].x * inv, mine[i].o[v].y * inv);
                    w.y = pack2<T>(mine[i].o[v].z * inv, mine[i].o[v].w * inv);
                    reinterpret_cast<uint2 *>(dst)[v * LANES + lane] = w;
                }
            }
        }
    }
}

template <int HD, int NT> struct StreamShape {
    // eight warps of three (head_dim 64: six) units each hold 192 KB in flight; 16 rows need the room for their records
    static constexpr int WARPS = NT == 1 ? 8 : 6, STAGES = 384 / HD;
    static constexpr size_t SMEM = (size_t)WARPS * STAGES * 2 * UNIT * HD * 2 + (size_t)WARPS * 8 * NT * (HD + 2) * sizeof(float);
};

template <typename T, int HD, int NT> int launch_stream(PagedArgs &a, cudaStream_t st) {
    using S = StreamShape<HD, NT>;
    auto kern = paged_stream_kernel<T, HD, NT, S::WARPS, S::STAGES>;
    XN_ENSURE_SMEM(kern, S::SMEM);
    a.parts = sm_count();
    if (int rc = launch_dependent(kern, dim3((unsigned)a.parts), dim3(S::WARPS * 32), S::SMEM, st, a)) return rc;
    return launch_paged_merge(FMT_OF<T>, HD, 8 * NT, 8 * NT, a, st);
}

}  // namespace

namespace {
template <typename T, int HD> int launch_merge(int rows, int used, const PagedArgs &a, cudaStream_t st) {
    constexpr int NV = 4, AT = 1, BLOCK = MERGE_NT * 4 * NV / HD * AT;
    if (rows <= 16)
        return launch_dependent(paged_merge_kernel<T, HD, 1, 1, true>, dim3((unsigned)a.parts, (unsigned)rows), dim3(MERGE_NT), 0, st, a, rows, used);
    return launch_dependent(paged_merge_kernel<T, HD, NV, AT, false>, dim3((unsigned)a.parts, (unsigned)((rows + BLOCK - 1) / BLOCK)), dim3(MERGE_NT),
                            0, st, a, rows, used);
}
}  // namespace

int launch_paged_merge(xn_dtype dt, int head_dim, int rows, int used, const PagedArgs &a, cudaStream_t st) {
    if (dt == XN_F16) return head_dim == 64 ? launch_merge<__half, 64>(rows, used, a, st) : launch_merge<__half, 128>(rows, used, a, st);
    return head_dim == 64 ? launch_merge<__nv_bfloat16, 64>(rows, used, a, st) : launch_merge<__nv_bfloat16, 128>(rows, used, a, st);
}

size_t paged_stream_workspace(int head_dim) { return part_bytes(sm_count(), 16, head_dim); }

int launch_paged_stream(xn_dtype dt, int head_dim, int rows, PagedArgs &a, cudaStream_t st) {
    const bool wide = rows > 8;
    if (dt == XN_F16) {
        if (head_dim == 64) return wide ? launch_stream<__half, 64, 2>(a, st) : launch_stream<__half, 64, 1>(a, st);
        return wide ? launch_stream<__half, 128, 2>(a, st) : launch_stream<__half, 128, 1>(a, st);
    }
    if (head_dim == 64) return wide ? launch_stream<__nv_bfloat16, 64, 2>(a, st) : launch_stream<__nv_bfloat16, 64, 1>(a, st);
    return wide ? launch_stream<__nv_bfloat16, 128, 2>(a, st) : launch_stream<__nv_bfloat16, 128, 1>(a, st);
}

}  // namespace xn
