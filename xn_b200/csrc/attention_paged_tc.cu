// Attention of chunks of query rows over a paged cache, on the tensor-memory MMAs.
//
// An item is up to 256 rows of one key head: two tiles A and B of 128 rows, a tile holding the query heads of the key head for
// 128 / group consecutive tokens, one TMA box.  Per block of 128 keys and tile:
//   S = Q K^T into tensor memory; a softmax thread owns a row of its tile: p = 2^((s - m) c) with m the row's reference point, sum
//   in f32, P rounded to the element type and written back over the scores; O += P V with P from tensor memory and V from shared memory
//   as it lies in memory.
// The two tiles take turns: while the tensor cores work on one tile's products, the softmax of the other tile runs.  Both
// read the same K and V stages, so a block costs 64 KB of L2 reads for 256 rows (head_dim 128).  An item of at most 128 rows has one
// tile only: then A and B are two streams over the even and the odd key blocks, each with its own maximum, sum and accumulator, merged
// at the end.
//
// Pages: a key block is a few TMA boxes of consecutive rows of a page, their page indexes read one block ahead.  Boxes beyond the
// context are not loaded, keys beyond it are masked, and the rows of V beyond it are overwritten with zeros in shared memory before a
// product reads them: whatever the page holds there does not matter.  The same is done where a causal or window border runs through
// the block and a row of V is not finite; rows of the result that see it become NaN, the others are as if it were not there.  Blocks
// go from the last key down: a causal item's border block comes first, when its V has time to be looked over (measured: 4 us of
// 68 in a batch of chunks with the border last, none so).
//
// Work is counted in key blocks (twice for items of two tiles), all items laid end to end and dealt out evenly to one persistent CTA per
// SM; what a CTA holds of an item that it shares with its neighbours becomes a record, joined by the merge kernel.  So a long context
// with few rows, a batch of chunks and single tokens, and a triangle all fill the machine.
#include "paged.cuh"
#include "tc05.cuh"

namespace xn {
namespace {

typedef unsigned long long u64;
constexpr int TC_THREADS = 128 + 256;      // two TMA producers, MMA issuer, segment walker; two softmax warpgroups
constexpr int KEYS = 128;
constexpr int HALF = KEYS * BKB;           // 128 rows of 64 elements: 16 KB
constexpr int K_STAGES = 2, V_STAGES = 2;
constexpr int TC_ROWS = 256;               // rows of an item and of a record
constexpr u64 SNAP = 4 * 2 * KEYS;          // units, see tc_weight
constexpr int SEGS = 4;                    // segments that the walker may be ahead

struct TcArgs {
    PagedArgs p;
    int tile_tokens;  // 128 / group
    int box;          // rows of a page that one TMA box loads
    WaitCtx wait;
};

struct TcSequence {
    Sequence s;
    int supers;  // items per key head
};
struct TcItem {
    int tok0, ntok;  // tokens of the sequence
    int kb0, kb1;    // key blocks that any of its rows sees (one at least)
    int lo;          // first key that any of its rows sees
    int dual;        // two tiles
};
__device__ __forceinline__ TcSequence tc_sequence(const TcArgs &a, int b) {
    TcSequence t;
    t.s = load_sequence(a.p, b);
    t.supers = (t.s.n + 2 * a.tile_tokens - 1) / (2 * a.tile_tokens);
    return t;
}
__device__ __forceinline__ TcItem tc_item(const TcArgs &a, int n, int off, int index) {
    TcItem i;
    i.tok0 = index * 2 * a.tile_tokens;
    i.ntok = min(n - i.tok0, 2 * a.tile_tokens);
    i.dual = i.ntok > a.tile_tokens;
    const int last = off + i.tok0 + i.ntok - 1;
    i.lo = first_key(a.p, off + i.tok0);
    i.kb0 = i.lo / KEYS;
    i.kb1 = max(last >= 0 ? last / KEYS + 1 : 0, i.kb0 + 1);
    return i;
}
// Units of work, by what it takes: an item weighs its keys and a block more, times 4 with two tiles (3450 cycles a block) and times 3 with
// one (2500: its two streams wait for memory as much as for one another).  In closed form, so that a share's beginning is found
// without a look at every item.
__device__ __forceinline__ u64 tc_weight(const TcArgs &a, const TcSequence &q, int index) {
    const int step = 2 * a.tile_tokens, end = min((index + 1) * step, q.s.n);
    const long long keys = (long long)max(q.s.off, 0) + end;
    return (u64)(min(keys, a.p.window ? (long long)a.p.window + step : keys) + KEYS) * (end - index * step > a.tile_tokens ? 4 : 3);
}
__device__ __forceinline__ u64 tc_before(const TcArgs &a, const TcSequence &q, int index) {  // of the items before this one, none the last
    const long long step = 2 * a.tile_tokens, off = max(q.s.off, 0);
    // the first `growing` of them see a block of tokens more each, the others a window
    const long long growing = a.p.window ? min((long long)index, max(0ll, (a.p.window - off + step - 1) / step)) : index;
    return 4 * (u64)(growing * (off + KEYS) + step * growing * (growing + 1) / 2 + (index - growing) * (a.p.window + step + KEYS));
}
__device__ __forceinline__ u64 tc_total(const TcArgs &a, const TcSequence &q) {
    return q.supers ? tc_before(a, q, q.supers - 1) + tc_weight(a, q, q.supers - 1) : 0;
}

// What a CTA does of an item: `nb` key blocks from block kb0 on (nb == 0: there is nothing more).
struct Segment {
    int nb, kb0;
    int b, head;
    int row0, tok0, n, ctx, off;  // first query row of the item, its first token, tokens and keys of the sequence, key of token 0
    int lo;                       // first key that any of the item's rows sees
    int dual;                     // two tiles
    int record;                   // -1: the whole item; otherwise the record that this part of it becomes
};
// The keys that all rows of the segment's item see, and the last that any does.
struct Sure {
    int lo, hi, last;
    __device__ __forceinline__ Sure(const TcArgs &a, const Segment &g) {
        const int end = min(g.tok0 + (1 + g.dual) * a.tile_tokens, g.n);
        lo = first_key(a.p, g.off + end - 1);
        hi = min(g.ctx - 1, g.off + g.tok0);
        last = min(g.ctx, g.off + end) - 1;
    }
};
struct Walk {
    int b, head, index;
    u64 pos;  // where the item begins
    u64 first, last;
    TcSequence q;
    // *end: where the item's units end
    __device__ __forceinline__ bool next(const TcArgs &a, Segment &g, u64 *end) {
        while (pos < last) {
            if (index >= q.supers) {
                index = 0;
                if (++head >= a.p.kv_heads) {
                    head = 0;
                    do {
                        if (++b >= a.p.batch) return false;
                        q = tc_sequence(a, b);
                    } while (q.supers == 0);
                }
                continue;
            }
            const TcItem it = tc_item(a, q.s.n, q.s.off, index);
            const int nkb = it.kb1 - it.kb0, dual = it.dual;
            const u64 units = tc_weight(a, q, index);
            *end = pos + units;
            // The blocks that begin in this share, if they lie evenly in the item's units.  A share's end that is near one of the item's is
            // moved there: a part of an item costs a record of its rows, as much as two blocks.
            auto cut = [&](u64 at) {
                if (at >= *end) return nkb;
                if (at <= pos || at - pos < SNAP) return 0;
                if (*end - at < SNAP) return nkb;
                return (int)(((at - pos) * (unsigned)nkb + units - 1) / units);
            };
            const int from = cut(first), to = cut(last);
            g = Segment{to - from, it.kb0 + from, b, head, q.s.q0 + it.tok0, it.tok0, q.s.n, q.s.ctx, q.s.off, it.lo, dual,
                        from == 0 && to == nkb ? -1 : (from > 0 ? 0 : 1)};
            pos = *end;
            ++index;
            if (from < to) return true;
        }
        return false;
    }
};

struct Border {  // a block of V that a causal or window border runs through
    int key0, sure_hi, sure_lo, first, last;  // first, last: the first and last key that any row of the item sees
    unsigned slot;
};
struct TcShared {
    uint64_t q_full, q_empty, k_full[K_STAGES], k_empty[K_STAGES], v_raw[V_STAGES], v_full[V_STAGES], v_empty[V_STAGES];
    uint64_t s_full[2], p_full[2][2], o_full[2], o_empty, red_full, red_empty, seg_full[SEGS], seg_empty[SEGS];
    Segment segs[SEGS];
    // keys of the segment that some rows see and others do not, and whose values are not finite: those above Sure::hi upwards, those below
    // Sure::lo downwards (a row's borders lie at most 255 keys from another's)
    uint32_t bad[SEGS][2][TC_ROWS / 32], any_bad[SEGS];
    Border border[V_STAGES];
    uint32_t tmem_slot;
    float red_m[2][128], red_l[2][128];
};

__device__ __forceinline__ bool mbar_test(uint64_t *bar, unsigned parity) {
    unsigned done;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
// D += A * B with A in tensor memory (lane = row, two 16-bit elements per column, 8 columns per MMA)
__device__ __forceinline__ void umma_from_tmem(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 b;\nmov.b64 b, {%2, %5};\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}" ::"r"(tmem_d),
        "r"(tmem_a), "r"(b_desc), "r"(idesc), "r"(acc), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ u64 pack_f32x2(float lo, float hi) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f32x2(u64 v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ u64 fma_f32x2(u64 a, u64 b, u64 c) {
    u64 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ u64 add_f32x2(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <typename T, int HD>
__global__ void __launch_bounds__(TC_THREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const TcArgs args) {
    constexpr int H = HD / 64, STAGE = H * HALF;
    constexpr int FMT = std::is_same<T, __half>::value ? 0 : 1;
    constexpr uint32_t IDESC_S = instr_desc(FMT, FMT, KEYS), IDESC_O = instr_desc(FMT, FMT, HD) | (1u << 16);
    const PagedArgs &p = args.p;
    extern __shared__ __align__(1024) unsigned char smem[];  // the kernel has no other shared memory: it begins on a swizzle atom
    unsigned char *sQ = smem;                     // two tiles
    unsigned char *sK = sQ + 2 * STAGE;
    unsigned char *sV = sK + K_STAGES * STAGE;
    unsigned char *sOut = sV + V_STAGES * STAGE;  // 4 KB for each softmax warp
    TcShared &sh = *reinterpret_cast<TcShared *>(sOut + 8 * 4096);
    const int warp = warp_id(), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        prefetch_tmap(&map_q);
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
        mbar_init(&sh.q_full, 1); mbar_init(&sh.q_empty, 1);
        for (int i = 0; i < K_STAGES; ++i) { mbar_init(&sh.k_full[i], 1); mbar_init(&sh.k_empty[i], 1); }
        for (int i = 0; i < V_STAGES; ++i) { mbar_init(&sh.v_raw[i], 1); mbar_init(&sh.v_full[i], 1); mbar_init(&sh.v_empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i][0], 4);
            mbar_init(&sh.p_full[i][1], 4);
            mbar_init(&sh.o_full[i], 1);
        }
        for (int i = 0; i < SEGS; ++i) {
            sh.any_bad[i] = 0;
            for (int w = 0; w < 2 * (TC_ROWS / 32); ++w) sh.bad[i][w >> 3][w & 7] = 0;
        }
        mbar_init(&sh.o_empty, 8);
        mbar_init(&sh.red_full, 8);
        mbar_init(&sh.red_empty, 8);
        for (int i = 0; i < SEGS; ++i) { mbar_init(&sh.seg_full[i], 1); mbar_init(&sh.seg_empty[i], 11); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = sh.tmem_slot;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // A wait's outcome is the warp's: one that ran out for some lanes only would part lanes that go on together.
    auto wait_all = [&](uint64_t *bar, unsigned parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, args.wait)) != 0; };

    // A softmax thread holds a row's 128 scores: registers move from the first warpgroup (128 x 56) to the other two (256 x 224), all
    // that the launch has (384 x 168).
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0 || warp == 3) {
            // ---- producers, one of Q and K, one of V: lane i looks after piece i of a key block ----
            asm volatile("griddepcontrol.wait;" ::: "memory");
            const bool keys = warp == 0;
            const CUtensorMap *map = keys ? &map_k : &map_v;
            bool ok = true;
            unsigned n_block = 0;
            const int pieces = KEYS / args.box;
            const unsigned tile_bytes = (unsigned)(args.tile_tokens * p.group * BKB * H);
            static_assert(K_STAGES == 2 && V_STAGES == 2, "of a ring's blocks one at most waits while another is issued");
            // stages of V whose blocks a border runs through, issued and not looked over yet, the older one first; -1: none
            int waits = -1, waits_next = -1;
            unsigned raw_phase = 0;
            for (unsigned n_seg = 0; ok; ++n_seg) {
                const unsigned slot = n_seg % SEGS;
                if (!wait_all(&sh.seg_full[slot], (n_seg / SEGS) & 1u)) break;
                const Segment g = sh.segs[slot];
                int page = -1, row = 0;
                auto fetch = [&](int kb) {  // the page of this lane's piece
                    const int key = kb * KEYS + lane * args.box;
                    page = -1;
                    row = 0;
                    if (lane < pieces && kb >= g.kb0 && key < g.ctx) {
                        const int at_page = p.page_shift >= 0 ? key >> p.page_shift : (int)((unsigned)key / (unsigned)p.page_size);
                        row = key - at_page * p.page_size;
                        page = p.table[(long long)g.b * p.table_stride + at_page];
                    }
                };
                fetch(g.kb0 + g.nb - 1);
                if (keys && g.nb) {  // while the first page's index is on its way
                    ok = wait_all(&sh.q_empty, (n_seg & 1u) ^ 1u);
                    if (!ok) break;
                    if (elect_one()) {
                        mbar_expect_tx(&sh.q_full, tile_bytes << g.dual);
                        for (int t = 0; t <= g.dual; ++t)
#pragma unroll
                            for (int h = 0; h < H; ++h)
                                tma_load_3d(sQ + t * STAGE + h * HALF, &map_q, h * 64, g.head * p.group, g.row0 + t * args.tile_tokens, &sh.q_full);
                    }
                }
                const Sure sure(args, g);
                for (int j = 0; ok;) {
                    if (waits < 0) {
                        waits = waits_next;
                        waits_next = -1;
                    }
                    if (j == g.nb && (waits < 0 || g.nb)) break;
                    const unsigned n = n_block + (unsigned)j, stage = n % K_STAGES, parity = ((n / K_STAGES) & 1u) ^ 1u;
                    uint64_t *room = keys ? &sh.k_empty[stage] : &sh.v_empty[stage];
                    // looked over as soon as it is there, or nothing else can be done
                    if (waits >= 0 && (j == g.nb || waits_next >= 0 ||
                                       __any_sync(0xffffffffu, mbar_test(&sh.v_raw[waits], raw_phase >> waits & 1u) || !mbar_test(room, parity)))) {
                        // Rows of V that no row of the item sees become zeros, and so do those that some see and others do not, if they are not
                        // finite: a product with the probability 0 would be NaN.  This warp has the time for it, while the next loads
                        // are on their way.
                        ok = wait_all(&sh.v_raw[waits], raw_phase >> waits & 1u);
                        if (!ok) break;
                        raw_phase ^= 1u << waits;
                        const Border e = sh.border[waits];
                        // rows [0, below) and [above, KEYS)
                        const int below = min(max(e.sure_lo - e.key0, 0), KEYS), above = min(max(e.sure_hi + 1 - e.key0, below), KEYS);
#pragma unroll 1
                        for (int i = lane; i < below + KEYS - above; i += 32) {
                            const int r = i < below ? i : above + i - below, key = e.key0 + r;
                            unsigned char *vrow = sV + waits * STAGE + r * BKB;
                            bool clear = key > e.last || key < e.first;
                            if (!clear) {
                                NotFinite<T> check;
#pragma unroll 8
                                for (int c = 0; c < H * 8; ++c)  // lanes in turned order: eight rows' pieces cover all banks
                                    check.see(*reinterpret_cast<const uint4 *>(vrow + (c >> 3) * HALF + ((c ^ r) & 7) * 16));
                                clear = check.any();
                                if (clear) {
                                    const int side = key > e.sure_hi ? 0 : 1, at = side ? e.sure_lo - 1 - key : key - e.sure_hi - 1;
                                    atomicOr(&sh.bad[e.slot][side][at >> 5], 1u << (at & 31));
                                    sh.any_bad[e.slot] = 1;
                                }
                            }
                            if (clear)
#pragma unroll
                                for (int c = 0; c < H * 8; ++c)
                                    *reinterpret_cast<uint4 *>(vrow + (c >> 3) * HALF + ((c ^ r) & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.v_full[waits]);
                        waits = -1;
                        continue;
                    }
                    const int kb = g.kb0 + g.nb - 1 - j, used = min(pieces, max(0, (g.ctx - kb * KEYS + args.box - 1) / args.box));
                    const int now_page = page, now_row = row;
                    fetch(kb - 1);
                    ok = wait_all(room, parity);
                    if (!ok) break;
                    const bool border = !keys && (kb * KEYS + KEYS - 1 > sure.hi || kb * KEYS < sure.lo);
                    uint64_t *full = keys ? &sh.k_full[stage] : border ? &sh.v_raw[stage] : &sh.v_full[stage];
                    unsigned char *dst = (keys ? sK : sV) + stage * STAGE;
                    if (elect_one()) mbar_expect_tx(full, (unsigned)(used * args.box * BKB * H));
                    for (int i = 0; i < used; ++i) {
                        const int pg = __shfl_sync(0xffffffffu, now_page, i), rw = __shfl_sync(0xffffffffu, now_row, i);
                        if (elect_one()) {
#pragma unroll
                            for (int h = 0; h < H; ++h) tma_load_4d(dst + h * HALF + i * args.box * BKB, map, h * 64, rw, g.head, pg, full);
                        }
                    }
                    if (border) {
                        (waits < 0 ? waits : waits_next) = (int)stage;
                        if (lane == 0) sh.border[stage] = Border{kb * KEYS, sure.hi, sure.lo, g.lo, sure.last, slot};
                        __syncwarp();
                    }
                    ++j;
                }
                if (g.nb == 0) break;
                n_block += (unsigned)g.nb;
                if (lane == 0) mbar_arrive(&sh.seg_empty[slot]);
            }
        } else if (warp == 2) {
            // ---- walker: the segments of this CTA's share, a few ahead of the others ----
            asm volatile("griddepcontrol.wait;" ::: "memory");
            auto warp_scan = [&](u64 x) {  // inclusive
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                return x;
            };
            auto warp_sum = [&](u64 x) {
#pragma unroll
                for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                return x;
            };
            // a sequence a lane and its units, of all key heads
            TcSequence q;
            u64 sum, total = 0, seen = 0;
            auto look_at = [&](int b0) {
                q = TcSequence{};
                if (b0 + lane < p.batch) q = tc_sequence(args, b0 + lane);
                sum = tc_total(args, q) * (unsigned)p.kv_heads;
            };
            for (int b0 = 0; b0 < p.batch; b0 += 32) {
                look_at(b0);
                total += warp_sum(sum);
            }
            const Shares shares(total, gridDim.x);
            Walk walk{};
            walk.first = shares.begin(blockIdx.x);
            walk.last = shares.begin(blockIdx.x + 1);
            for (int b0 = 0; b0 < p.batch && walk.first < walk.last; b0 += 32) {  // the item that the share begins in
                if (p.batch > 32) look_at(b0);
                const u64 inc = seen + warp_scan(sum);
                const bool here = inc - sum <= walk.first && walk.first < inc;
                const unsigned hit = __ballot_sync(0xffffffffu, here);
                seen = __shfl_sync(0xffffffffu, inc, 31);
                if (!hit) continue;
                const int src = __ffs(hit) - 1;
                int head = 0, index = 0;
                u64 pos = 0;
                if (here) {
                    u64 heads, in_head;
                    divide(walk.first - (inc - sum), tc_total(args, q), heads, in_head);
                    int hi = q.supers - 1;
                    while (index < hi) {
                        const int mid = (index + hi + 1) >> 1;
                        if (tc_before(args, q, mid) <= in_head) index = mid;
                        else hi = mid - 1;
                    }
                    head = (int)heads;
                    pos = walk.first - in_head + tc_before(args, q, index);
                }
                walk.b = b0 + src;
                walk.head = __shfl_sync(0xffffffffu, head, src);
                walk.index = __shfl_sync(0xffffffffu, index, src);
                walk.pos = __shfl_sync(0xffffffffu, pos, src);
                walk.q.s.q0 = __shfl_sync(0xffffffffu, q.s.q0, src);
                walk.q.s.n = __shfl_sync(0xffffffffu, q.s.n, src);
                walk.q.s.ctx = __shfl_sync(0xffffffffu, q.s.ctx, src);
                walk.q.s.off = __shfl_sync(0xffffffffu, q.s.off, src);
                walk.q.supers = __shfl_sync(0xffffffffu, q.supers, src);
                break;
            }
            if (walk.first >= walk.last) walk.last = 0;
            PartNote note{};
            u64 goes_to = 0;  // the last unit of the item that the share does not end
            if (lane == 0) {
                for (unsigned n_seg = 0;; ++n_seg) {
                    Segment g{};
                    u64 end;
                    const bool more = walk.next(args, g, &end);
                    if (more && g.record == 0) note.joined = 1;
                    if (more && g.record == 1) {
                        note = PartNote{note.joined, 0, g.row0 - g.tok0, g.n * p.group, g.tok0 * p.group, g.head};
                        goes_to = end - 1;
                    }
                    if (!more) g.nb = 0;
                    const unsigned slot = n_seg % SEGS;
                    if (!mbar_wait(&sh.seg_empty[slot], ((n_seg / SEGS) & 1u) ^ 1u, args.wait)) break;
                    sh.segs[slot] = g;
                    if (sh.any_bad[slot]) {
                        sh.any_bad[slot] = 0;
                        for (int i = 0; i < 2 * (TC_ROWS / 32); ++i) sh.bad[slot][i >> 3][i & 7] = 0;
                    }
                    mbar_arrive(&sh.seg_full[slot]);
                    if (!more) break;
                }
                if (goes_to) note.last = (int)shares.of(goes_to);
                static_cast<PartNote *>(p.ws)[blockIdx.x] = note;
            }
        } else if (warp == 1) {
            // ---- MMA issuer ----
            asm volatile("griddepcontrol.wait;" ::: "memory");  // ahead of the first wait: its limit is not for what earlier kernels take
            if (elect_one()) {
                bool ok = true;
                unsigned nk = 0, nv = 0, np[2] = {0, 0};
                auto scores = [&](int t, int q_tile, unsigned stage) {  // S_t = Q K^T
    #pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const uint32_t da = smem_desc(sQ + q_tile * STAGE + h * HALF), db = smem_desc(sK + stage * STAGE + h * HALF);
    #pragma unroll
                        for (int ks = 0; ks < BKB / UMMA_KB; ++ks) {
                            const uint32_t adv = (uint32_t)(ks * UMMA_KB >> 4);
                            umma<false>(tmem_base + t * KEYS, da + adv, db + adv, IDESC_S, (h | ks) != 0);
                        }
                    }
                    umma_commit(&sh.s_full[t]);
                };
                auto after = [] { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); };
                // O_t (+)= P_t V, the first 64 keys as soon as their probabilities are there
                auto product = [&](int t, unsigned stage, bool add) -> bool {
                    const uint32_t db = smem_desc_mn(sV + stage * STAGE, HALF);
                    const unsigned n = np[t]++;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (!mbar_wait(&sh.p_full[t][half], n & 1u, args.wait)) return false;
                        after();
#pragma unroll
                        for (int ks = 4 * half; ks < 4 * half + 4; ++ks)
                            umma_from_tmem(tmem_base + 256 + t * HD, tmem_base + t * KEYS + ks * 8, db + ks * (uint32_t)(16 * BKB >> 4), IDESC_O,
                                           add || ks != 0);
                    }
                    return true;
                };
                auto wait_k = [&](unsigned n) { return mbar_wait(&sh.k_full[n % K_STAGES], (n / K_STAGES) & 1u, args.wait); };
                auto wait_v = [&](unsigned n) { return mbar_wait(&sh.v_full[n % V_STAGES], (n / V_STAGES) & 1u, args.wait); };
                for (unsigned n_seg = 0; ok; ++n_seg) {
                    const unsigned slot = n_seg % SEGS;
                    if (!mbar_wait(&sh.seg_full[slot], (n_seg / SEGS) & 1u, args.wait)) break;
                    const int nb = sh.segs[slot].nb, dual = sh.segs[slot].dual;
                    if (nb == 0) break;
                    mbar_arrive(&sh.seg_empty[slot]);
                    const unsigned o_phase = (n_seg & 1u) ^ 1u;
                    if (!mbar_wait(&sh.q_full, n_seg & 1u, args.wait) || !wait_k(nk)) { ok = false; break; }
                    after();
                    if (dual) {
                        scores(0, 0, nk % K_STAGES);
                        scores(1, 1, nk % K_STAGES);
                        umma_commit(&sh.k_empty[nk % K_STAGES]);
                        if (nb == 1) umma_commit(&sh.q_empty);
                        ++nk;
                        for (int j = 0; j < nb && ok; ++j, ++nv) {
                            const bool more = j + 1 < nb;
                            for (int t = 0; t < 2 && ok; ++t) {
                                // the first products of an item overwrite the accumulators: the rows before must have been read
                                ok = (t || (wait_v(nv) && (j || mbar_wait(&sh.o_empty, o_phase, args.wait)))) && product(t, nv % V_STAGES, j != 0);
                                if (!ok) break;
                                if (t) umma_commit(&sh.v_empty[nv % V_STAGES]);
                                if (!more) umma_commit(&sh.o_full[t]);
                                else {
                                    if (t == 0 && !wait_k(nk)) { ok = false; break; }
                                    after();
                                    scores(t, t, nk % K_STAGES);
                                    if (t) {
                                        umma_commit(&sh.k_empty[nk % K_STAGES]);
                                        if (j + 2 == nb) umma_commit(&sh.q_empty);
                                        ++nk;
                                    }
                                }
                            }
                        }
                    } else {
                        scores(0, 0, nk % K_STAGES);
                        umma_commit(&sh.k_empty[nk % K_STAGES]);
                        ++nk;
                        if (nb > 1) {
                            if (!wait_k(nk)) { ok = false; break; }
                            after();
                            scores(1, 0, nk % K_STAGES);
                            umma_commit(&sh.k_empty[nk % K_STAGES]);
                            ++nk;
                        }
                        if (nb <= 2) umma_commit(&sh.q_empty);
                        for (int j = 0; j < nb && ok; ++j, ++nv) {
                            const int t = j & 1;
                            ok = wait_v(nv) && (j || mbar_wait(&sh.o_empty, o_phase, args.wait)) && product(t, nv % V_STAGES, j > 1);
                            if (!ok) break;
                            umma_commit(&sh.v_empty[nv % V_STAGES]);
                            if (j + 2 < nb) {
                                if (!wait_k(nk)) { ok = false; break; }
                                after();
                                scores(t, 0, nk % K_STAGES);
                                umma_commit(&sh.k_empty[nk % K_STAGES]);
                                if (j + 3 == nb) umma_commit(&sh.q_empty);
                                ++nk;
                            }
                        }
                        if (ok) {
                            umma_commit(&sh.o_full[0]);
                            umma_commit(&sh.o_full[1]);
                        }
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---- softmax: tile t, row r ----
        const int t = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_addr = lanes + (uint32_t)(t * KEYS);
        const uint32_t o_addr = lanes + 256 + (uint32_t)(t * HD);
        const int tile_rows = args.tile_tokens * p.group;
        const int r_token = r / p.group, r_head = r % p.group;
        bool ok = true;
        unsigned n_mine = 0, n_split = 0;
        // The first turn is a dry one, with nothing to wait for and nothing written: it brings the code into the instruction cache while the
        // first segment, its keys and its scores are on their way (cold, a first block took 5000 to 9000 cycles instead of 3500).
        bool dry = true;
        for (unsigned n_seg = 0; ok; dry ? (void)(dry = false) : (void)++n_seg) {
            const unsigned slot = n_seg % SEGS;
            if (!dry && !wait_all(&sh.seg_full[slot], (n_seg / SEGS) & 1u)) break;
            const Segment g = dry ? Segment{1, 0, 0, 0, 0, 0, 1, KEYS, 0, 0, 1, -1} : sh.segs[slot];
            const int nb = g.nb, dual = g.dual, ctx = g.ctx, kb0 = g.kb0;
            if (nb == 0) break;
            const int tok = g.tok0 + (dual ? t * args.tile_tokens : 0) + r_token;
            const bool real = r < tile_rows && tok < g.n && !dry;
            const bool any_real = __any_sync(0xffffffffu, real) || dry;
            const int horizon = min(ctx - 1, g.off + tok);
            const int low = first_key(p, g.off + tok);
            float m = real ? -INFINITY : 0.0f;  // rows of nobody never move their reference
            u64 l2[2] = {0, 0};
            bool begun = false;
            for (int j = 0; j < nb; ++j) {
                if (!dual && (j & 1) != t) continue;
                const int key0 = (kb0 + nb - 1 - j) * KEYS;
                if (!dry) {
                    ok = wait_all(&sh.s_full[t], n_mine & 1u);
                    if (!ok) break;
                    ++n_mine;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (any_real) {
                    uint32_t v[4][32];
#pragma unroll
                    for (int i = 0; i < 4; ++i) tmem_ld32_nowait(s_addr + i * 32, v[i]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if ((real || dry) && (key0 + KEYS - 1 > horizon || key0 < low)) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            // bits [from, to) of the chunk's columns are seen
                            const int from = min(max(low - key0 - 32 * c, 0), 32), to = min(max(horizon + 1 - key0 - 32 * c, 0), 32);
                            const uint32_t seen = (uint32_t)((1ull << to) - 1) & ~(uint32_t)((1ull << from) - 1);
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!(seen & (1u << i))) v[c][i] = 0xff800000u;
                        }
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < KEYS; i += 2)
                        top[(i >> 1) & 3] = fmaxf(fmaxf(top[(i >> 1) & 3], __uint_as_float(v[i >> 5][i & 31])),
                                                  __uint_as_float(v[(i + 1) >> 5][(i + 1) & 31]));
                    const float bm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                    // The reference moves only when a block exceeds it by 2^8: any reference gives the same quotient, values up to 256
                    // are harmless in f32 and in the 16-bit types, and rescaling the accumulator becomes rare.
                    const float m_new = real && (bm - m) * p.c > 8.0f ? bm : m;
                    if (__any_sync(0xffffffffu, m_new != m)) {
                        const float alpha = m_new != m ? exp2_fast((m - m_new) * p.c) : 1.0f;  // m = -inf: 0
                        if (begun) {  // S is complete, so the products before it are too: the accumulator is this thread's
#pragma unroll 1
                            for (int i = 0; i < HD / 32; ++i) {
                                uint32_t o[32];
                                tmem_ld32(o_addr + i * 32, o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                                tmem_st32(o_addr + i * 32, o);
                            }
                        }
                        const u64 a2 = pack_f32x2(alpha, alpha);
                        l2[0] = fma_f32x2(l2[0], a2, 0);
                        l2[1] = fma_f32x2(l2[1], a2, 0);
                        m = m_new;
                    }
                    begun = true;
                    const float mc = m == -INFINITY ? 0.0f : -m * p.c;
                    const u64 c2 = pack_f32x2(p.c, p.c), m2 = pack_f32x2(mc, mc);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t packed[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int e = half * 64 + 2 * i;
                            float x, y;
                            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[e >> 5][e & 31]), __uint_as_float(v[(e + 1) >> 5][(e + 1) & 31])),
                                                   c2, m2), x, y);
                            x = exp2_fast(x);
                            y = exp2_fast(y);
                            l2[i & 1] = add_f32x2(l2[i & 1], pack_f32x2(x, y));
                            packed[i] = pack2<T>(x, y);
                        }
                        if (!dry) tmem_st32(s_addr + half * 32, packed);
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0 && !dry) mbar_arrive(&sh.p_full[t][half]);
                    }
                } else {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane < 2) mbar_arrive(&sh.p_full[t][lane]);
                }
            }
            float l;
            {
                float x, y;
                unpack_f32x2(add_f32x2(l2[0], l2[1]), x, y);
                l = x + y;
            }
            // the weights of the two accumulators in this row; with two tiles there is only the row's own
            float w0 = 1.0f, w1 = 0.0f, mm = m;
            if (!dual && ok) {
                const unsigned turn = n_split++ & 1u;
                ok = wait_all(&sh.red_empty, turn ^ 1u);  // the rows of the item before have been read
                sh.red_m[t][r] = m;
                sh.red_l[t][r] = l;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.red_full);
                ok = ok && wait_all(&sh.red_full, turn);
                const float m0 = sh.red_m[0][r], m1 = sh.red_m[1][r];
                mm = fmaxf(m0, m1);
                const float l0 = sh.red_l[0][r], l1 = sh.red_l[1][r];
                w0 = l0 == 0.0f ? 0.0f : exp2_fast((m0 - mm) * p.c);  // nothing seen: 0; nothing but NaN: NaN
                w1 = l1 == 0.0f ? 0.0f : exp2_fast((m1 - mm) * p.c);
                l = w0 * l0 + w1 * l1;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.red_empty);
            }
            // a tile's own accumulator, or both of a row's
            if (ok && !dry && (!dual || t == 0)) ok = wait_all(&sh.o_full[0], n_seg & 1u);
            if (ok && !dry && (!dual || t == 1)) ok = wait_all(&sh.o_full[1], n_seg & 1u);
            if (ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (!dry && sh.any_bad[slot]) {
                    const Sure sure(args, g);
                    for (int i = 0; i < 2 * TC_ROWS; ++i) {  // a key that the row sees was taken for zeros
                        const int key = i < TC_ROWS ? sure.hi + 1 + i : sure.lo - 1 - (i - TC_ROWS);
                        if ((sh.bad[slot][i >> 8][(i & 255) >> 5] >> (i & 31) & 1) && key <= horizon && key >= low) l = NAN;
                    }
                }
                const bool empty = l == 0.0f;
                const float inv = empty ? 0.0f : 1.0f / l;
                // Columns of the row that this thread reads: all of its tile's accumulator, or half of both.  32 at a time go through shared
                // memory, so that eight threads write 32 columns of one row together: a thread that wrote its own row would touch a line
                // of its own with every store.
                const int c0 = dual ? 0 : t * (HD / 2), ncols = dual ? HD : HD / 2;
                const int record = g.record;
                float *rec = part_records(p.ws, gridDim.x) + ((size_t)blockIdx.x * 2 + max(record, 0)) * part_record_floats(TC_ROWS, HD);
                const int rec_row = dual ? t * 128 + r : r;
                const long long own_row = !real ? -1
                                          : record >= 0 ? (long long)rec_row * HD
                                                        : (long long)(g.row0 - g.tok0 + tok) * p.out_token + (long long)(g.head * p.group + r_head) * p.out_head;
                if (any_real) {
                    const float scale0 = record >= 0 ? w0 : w0 * inv, scale1 = record >= 0 ? w1 : w1 * inv;
                    float4 *mine = reinterpret_cast<float4 *>(sOut + (warp - 4) * 4096);
                    long long rows[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) rows[i] = __shfl_sync(0xffffffffu, own_row, 4 * i + (lane >> 3));
#pragma unroll 1
                    for (int c = c0; c < c0 + ncols; c += 32) {
                        uint32_t x[32], y[32];
                        if (dual) {
                            tmem_ld32(o_addr + c, x);
                        } else {
                            tmem_ld32_nowait(lanes + 256 + c, x);
                            tmem_ld32_nowait(lanes + 256 + HD + c, y);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float f[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                f[e] = scale0 == 0.0f || empty ? 0.0f : __uint_as_float(x[4 * i + e]) * scale0;
                                if (!dual && scale1 != 0.0f && !empty) f[e] += __uint_as_float(y[4 * i + e]) * scale1;
                            }
                            mine[lane * 8 + (i ^ (lane & 7))] = make_float4(f[0], f[1], f[2], f[3]);
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int row = 4 * i + (lane >> 3), piece = lane & 7;
                            const float4 f = mine[row * 8 + (piece ^ (row & 7))];
                            if (rows[i] < 0) continue;
                            if (record >= 0) *reinterpret_cast<float4 *>(rec + rows[i] + c + piece * 4) = f;
                            else
                                *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + rows[i] + c + piece * 4) = make_uint2(pack2<T>(f.x, f.y), pack2<T>(f.z, f.w));
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0 && !dry) mbar_arrive(&sh.o_empty);
                if (record >= 0 && real && (dual || t == 0)) {
                    rec[TC_ROWS * HD + rec_row] = mm == -INFINITY ? -INFINITY : mm * p.c;
                    rec[TC_ROWS * HD + TC_ROWS + rec_row] = l;
                }
                if (lane == 0 && !dry) mbar_arrive(&sh.seg_empty[slot]);
            }
            if (dry) {
                asm volatile("griddepcontrol.wait;" ::: "memory");  // from here on memory that earlier kernels may use is written
            }
        }
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    }
}

template <typename T, int HD>
int launch_tc(TcArgs &a, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t st) {
    auto kern = paged_tc_kernel<T, HD>;
    const size_t smem = (size_t)(2 + K_STAGES + V_STAGES) * (HD / 64) * HALF + 8 * 4096 + sizeof(TcShared);
    XN_ENSURE_SMEM(kern, smem);
    a.p.parts = sm_count();
    if (int rc = launch_dependent(kern, dim3((unsigned)a.p.parts), dim3(TC_THREADS), smem, st, mq, mk, mv, a)) return rc;
    return launch_paged_merge(FMT_OF<T>, HD, TC_ROWS, a.tile_tokens * a.p.group, a.p, st);
}

}  // namespace

size_t paged_tc_workspace(int head_dim) { return part_bytes(sm_count(), TC_ROWS, head_dim); }

bool paged_tc_fits(const PagedArgs &a) {
    const long long most = 1ll << 38;  // strides that a tensor map holds
    return a.q_token < most && a.q_head < most && a.page_stride < most && a.head_stride < most && a.row_stride < most &&
           a.page_size % 8 == 0 && a.group <= 128 && a.num_pages > 0 && a.max_pages > 0 && a.q_token > 0 && a.q_head > 0 && a.page_stride > 0 &&
           a.head_stride > 0 && a.row_stride > 0;
}

int launch_paged_tc(xn_dtype dt, int head_dim, const PagedArgs &p, cudaStream_t st) {
    TcArgs a{};
    a.p = p;
    a.tile_tokens = 128 / p.group;
    a.box = 8;
    while (a.box < 128 && p.page_size % (2 * a.box) == 0) a.box *= 2;
    if (int rc = wait_ctx(&a.wait)) return rc;
    CUtensorMap mq, mk, mv;
    if (int rc = make_map_rows(&mq, p.q, head_dim, {(size_t)p.heads, (size_t)p.tokens}, {(size_t)p.q_head, (size_t)p.q_token},
                               {(unsigned)p.group, (unsigned)a.tile_tokens}))
        return rc;
    for (int i = 0; i < 2; ++i)
        if (int rc = make_map_rows(i ? &mv : &mk, i ? p.v : p.k, head_dim, {(size_t)p.page_size, (size_t)p.kv_heads, (size_t)p.num_pages},
                                   {(size_t)p.row_stride, (size_t)p.head_stride, (size_t)p.page_stride}, {(unsigned)a.box, 1, 1}))
            return rc;
    if (dt == XN_F16) return head_dim == 64 ? launch_tc<__half, 64>(a, mq, mk, mv, st) : launch_tc<__half, 128>(a, mq, mk, mv, st);
    return head_dim == 64 ? launch_tc<__nv_bfloat16, 64>(a, mq, mk, mv, st) : launch_tc<__nv_bfloat16, 128>(a, mq, mk, mv, st);
}

}  // namespace xn
