// Entry points of attention over a paged cache: checks, and which kernel a call gets.
#include <float.h>
#include <math.h>

#include "paged.cuh"

using namespace xn;

extern "C" size_t xn_mm_attention_paged_workspace_bytes(size_t head_dim) {
    if (head_dim != 64 && head_dim != 128) return 0;
    const size_t a = paged_stream_workspace((int)head_dim), b = paged_tc_workspace((int)head_dim);
    return a > b ? a : b;
}

extern "C" int xn_mm_attention_paged(xn_dtype dtype, void *out, size_t out_token_stride, size_t out_head_stride, const void *q,
                                     size_t q_token_stride, size_t q_head_stride, size_t tokens, size_t heads, const void *k_pages,
                                     const void *v_pages, size_t page_stride, size_t head_stride, size_t row_stride, size_t num_pages,
                                     size_t page_size, size_t kv_heads, size_t head_dim, const int32_t *page_table, size_t table_stride,
                                     size_t max_pages, const int32_t *context, const int32_t *query_starts_or_null, size_t batch,
                                     size_t max_query, size_t window, float scale, void *workspace, size_t workspace_bytes,
                                     void *stream) {
    XN_API_RANGE("xn_mm_attention_paged");
    XN_REQUIRE(dtype == XN_F16 || dtype == XN_BF16, "attention_paged: 16-bit elements only, got dtype %d", (int)dtype);
    XN_REQUIRE(head_dim == 64 || head_dim == 128, "attention_paged: head_dim %zu is not supported (64 and 128 are)", head_dim);
    XN_REQUIRE(kv_heads > 0 ? heads % kv_heads == 0 : heads == 0, "attention_paged: %zu query heads do not share %zu key heads evenly",
               heads, kv_heads);
    XN_REQUIRE(scale >= 0.0f && scale <= 3.0e38f, "attention_paged: scale must be finite and not negative");
    XN_REQUIRE(page_size > 0 && page_size <= 0x40000000ull, "attention_paged: a page of %zu tokens", page_size);
    XN_REQUIRE(tokens <= 0x3fffffffull && heads <= 65536 && batch <= 0x3fffffffull && num_pages <= 0x7fffffffull &&
                   max_pages <= 0x7fffffffull && max_pages * page_size <= 0x7fffff00ull && tokens * (heads ? heads : 1) <= 0x7fffffffull,
               "attention_paged: sizes beyond 32-bit positions");
    if (tokens == 0 || heads == 0 || batch == 0) return XN_OK;
    XN_REQUIRE(query_starts_or_null || batch == tokens, "attention_paged: %zu rows for %zu sequences of one row each", tokens, batch);
    XN_REQUIRE(out && q && context && (max_pages == 0 || page_table) && (max_pages == 0 || num_pages == 0 || (k_pages && v_pages)),
               "attention_paged: null pointer");
    XN_REQUIRE(aligned(q, 16) && aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(out, 16) && q_token_stride % 8 == 0 &&
                   q_head_stride % 8 == 0 && out_token_stride % 8 == 0 && out_head_stride % 8 == 0 && page_stride % 8 == 0 &&
                   head_stride % 8 == 0 && row_stride % 8 == 0,
               "attention_paged: tensors must be 16-byte aligned, strides multiples of 8 elements");
    const size_t need = xn_mm_attention_paged_workspace_bytes(head_dim);
    if (!workspace || workspace_bytes < need)
        return fail(XN_ERR_WORKSPACE, "attention_paged: workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : 0);
    XN_REQUIRE(aligned(workspace, 256), "attention_paged: workspace must be 256-byte aligned");
    PagedArgs a{};
    a.q = q; a.k = k_pages; a.v = v_pages; a.out = out;
    a.table = page_table; a.context = context; a.starts = query_starts_or_null;
    a.q_token = (long long)q_token_stride; a.q_head = (long long)q_head_stride;
    a.out_token = (long long)out_token_stride; a.out_head = (long long)out_head_stride;
    a.page_stride = (long long)page_stride; a.head_stride = (long long)head_stride; a.row_stride = (long long)row_stride;
    a.table_stride = (long long)table_stride;
    a.tokens = (int)tokens; a.batch = (int)batch; a.heads = (int)heads; a.kv_heads = (int)kv_heads; a.group = (int)(heads / kv_heads);
    a.num_pages = (int)num_pages; a.page_size = (int)page_size; a.max_pages = (int)max_pages;
    a.page_shift = -1;
    if ((page_size & (page_size - 1)) == 0)
        for (a.page_shift = 0; (size_t)1 << a.page_shift < page_size; ++a.page_shift) {}
    a.window = window < max_pages * page_size ? (int)window : 0;  // one as wide as the table hides nothing
    a.c = fminf(fmaxf(scale * 1.4426950408889634f, 1e-37f), FLT_MAX);  // above zero, so that a masked score, -inf, stays -inf, and finite
    a.ws = workspace;
    if (!query_starts_or_null) max_query = 1;
    if (max_query > tokens || max_query == 0) max_query = tokens;
    // rows: query heads of one key head times the new tokens.  The streaming kernel reads the keys once for 16 of them and has its first
    // loads on their way sooner; the tensor-memory kernel reads them once for 256.  Measured at head_dim 128 (streaming / tensor
    // memory, us): 8 rows of 4 key heads, 4 x 30000 keys 30 / 35, 16 x 3000 18 / 25; 16 rows of 2, 4 x 30000 24 / 26, 16 x 3000
    // 20 / 21, 1 x 1000 13 / 16; 32 rows of 4, 4 x 30000 53 / 36, 16 x 3000 37 / 25, 1 x 1000 13 / 18.
    const size_t rows = max_query * (heads / kv_heads);
    // More rows take the streaming kernel too where they make few items of 16 rows and few keys are read for them, as far as the tensors'
    // sizes tell: its way to the first and from the last key is the shorter one.  Items and MB read (streaming / tensor memory, us), at
    // head_dim 128: 28 and 1.4 13 / 19, 148 and 20 14 / 20, 35 and 27 18 / 19, 192 and 53 25 / 18; at head_dim 64, where fewer of
    // them outweigh it: 14 and 4.7 15 / 17, 48 and 0.6 12 / 14, 64 and 2.7 14 / 13, 112 and 5.1 18 / 14, 56 and 59 24 / 21.
    const size_t room = max_pages * page_size, keys = window > 0 && window < room && window + max_query < room ? window + max_query : room;
    const double items = (double)batch * kv_heads * ((rows + 15) / 16), bytes = items * keys * head_dim * 4;
    const bool small = items <= (head_dim == 128 ? sm_count() : sm_count() / 3) && bytes <= 32e6;
    if (rows > 16 && !small && paged_tc_fits(a)) return launch_paged_tc(dtype, (int)head_dim, a, (cudaStream_t)stream);
    return launch_paged_stream(dtype, (int)head_dim, rows > 16 ? 16 : (int)rows, a, (cudaStream_t)stream);
}
