// What the kernels of attention over a paged cache share: the call's arguments, the geometry of a sequence, and the records of
// rows whose keys were shared out.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace xn {

// Sequence b has the query rows [starts[b], starts[b + 1]) (starts == null: row b alone) and context[b] keys, its own rows'
// keys the last of them; key j lies in row j % page_size of page table[b][j / page_size].  Row i of n sees the keys
// j <= i + context - n, of those the last `window` only (0: all).  Lengths and indexes come from device memory and are
// bounded where they are read: nothing they say can lead outside the tensors.  A page index outside the pool reads as a
// page of zeros.
struct PagedArgs {
    const void *q, *k, *v;
    void *out;
    const int *table, *context, *starts;
    long long q_token, q_head, out_token, out_head;   // strides in elements
    long long page_stride, head_stride, row_stride;   // of both pools
    long long table_stride;
    int tokens, batch, heads, kv_heads, group;
    int num_pages, page_size, page_shift, max_pages;  // page_shift: log2(page_size), or -1
    int window;  // 0, or fewer keys than a table holds
    float c;  // scale * log2(e)
    void *ws;
    int parts;  // CTAs that share the work
};

struct Sequence {
    int q0, n;    // first query row, number of them
    int ctx, off; // keys, and the last key that row 0 sees
};
__device__ __forceinline__ Sequence load_sequence(const PagedArgs &a, int b) {
    Sequence s;
    if (a.starts) {
        s.q0 = min(max(a.starts[b], 0), a.tokens);
        s.n = min(max(a.starts[b + 1], s.q0), a.tokens) - s.q0;
    } else {
        s.q0 = min(b, a.tokens);
        s.n = b < a.tokens ? 1 : 0;
    }
    const long long room = (long long)a.max_pages * a.page_size;
    s.ctx = (int)min((long long)max(a.context[b], 0), room);
    s.off = s.ctx - s.n;
    return s;
}

// The first key that a row sees whose last is `last`.  Windows go up to 2^31: last - window + 1 alone could leave 32 bits.
__device__ __forceinline__ int first_key(const PagedArgs &a, int last) { return a.window && last >= a.window ? last - a.window + 1 : 0; }

// A row's result over a part of its keys: the sum of p v (head_dim floats), the maximum m of its scaled scores and the sum l of
// p = 2^(score - m).  CTA c of `parts` writes the part of the item that began before it into record 0 and the part of the one that it
// begins and does not end into record 1, and leaves a note of both.
struct PartNote {
    int joined;                    // whether record 0 is written
    int last;                      // record 1 is: the item goes on in the CTAs behind this one, up to this one (0: it is not)
    int q0, rows, tile_row, head;  // the item's: first query row of its sequence, rows of the sequence, first row of the item, kv head
};
__host__ __device__ constexpr size_t part_record_floats(int rows, int hd) { return (size_t)rows * (hd + 2); }
__host__ __device__ constexpr size_t part_bytes(int parts, int rows, int hd) {
    return ((size_t)parts * sizeof(PartNote) + 255) / 256 * 256 + (size_t)parts * 2 * part_record_floats(rows, hd) * sizeof(float);
}
__host__ __device__ inline float *part_records(void *ws, int parts) {
    return reinterpret_cast<float *>(static_cast<char *>(ws) + ((size_t)parts * sizeof(PartNote) + 255) / 256 * 256);
}
// Units are dealt out evenly, in order: share g of `count` gets [begin(g), begin(g + 1)).  The 64-bit divisions that are not needed are
// left out: they would take longer than the rest of a short call's way to its first load.
struct Shares {
    unsigned long long total, each;
    unsigned rest, count;
    __device__ __forceinline__ Shares(unsigned long long units, unsigned shares) : total(units), count(shares) {
        if (units >> 32) {
            each = units / shares;
            rest = (unsigned)(units % shares);
        } else {
            each = (unsigned)units / shares;
            rest = (unsigned)units % shares;
        }
    }
    __device__ __forceinline__ unsigned long long begin(unsigned g) const { return each * g + rest * g / count; }  // below 2^16 shares
    // the share that a unit falls into
    __device__ __forceinline__ unsigned of(unsigned long long unit) const {
        unsigned lo = 0, hi = count - 1;
        while (lo < hi) {
            const unsigned mid = (lo + hi + 1) >> 1;
            if (begin(mid) <= unit) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
};
__device__ __forceinline__ void divide(unsigned long long x, unsigned long long by, unsigned long long &quotient, unsigned long long &rest) {
    if ((x | by) >> 32) {
        quotient = x / by;
        rest = x % by;
    } else {
        quotient = (unsigned)x / (unsigned)by;
        rest = (unsigned)x % (unsigned)by;
    }
}

template <typename T> constexpr xn_dtype FMT_OF = std::is_same<T, __half>::value ? XN_F16 : XN_BF16;
template <typename T> __device__ __forceinline__ unsigned pack2(float x, float y);
template <> __device__ __forceinline__ unsigned pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const unsigned *>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const unsigned *>(&h);
}
// Whether an infinity or NaN is among the elements seen: a sum of their products with 0 is NaN then, and 0 otherwise.
template <typename T> struct NotFinite {
    typedef std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162> Pair;
    unsigned sum[4] = {0, 0, 0, 0};
    __device__ __forceinline__ void see(const uint4 &x) {
        const unsigned v[4] = {x.x, x.y, x.z, x.w}, zero = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Pair r = __hfma2(*reinterpret_cast<const Pair *>(&v[i]), *reinterpret_cast<const Pair *>(&zero), *reinterpret_cast<const Pair *>(&sum[i]));
            sum[i] = *reinterpret_cast<const unsigned *>(&r);
        }
    }
    __device__ __forceinline__ bool any() const { return ((sum[0] | sum[1] | sum[2] | sum[3]) & 0x7fff7fffu) != 0; }
};
__device__ __forceinline__ float exp2_fast(float x) {  // relative error about 2^-22; 0 for -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// attention_paged_stream.cu: up to 16 rows of a key head at a time, any page size
int launch_paged_stream(xn_dtype dt, int head_dim, int rows, PagedArgs &a, cudaStream_t st);
size_t paged_stream_workspace(int head_dim);
// Records of `rows` rows, of which the first `used` of every 128 are rows of the item.
int launch_paged_merge(xn_dtype dt, int head_dim, int rows, int used, const PagedArgs &a, cudaStream_t st);
// attention_paged_tc.cu: 256 rows of a key head at a time on the tensor-memory MMAs; pages of a multiple of 8 rows
bool paged_tc_fits(const PagedArgs &a);
size_t paged_tc_workspace(int head_dim);
int launch_paged_tc(xn_dtype dt, int head_dim, const PagedArgs &a, cudaStream_t st);

}  // namespace xn
