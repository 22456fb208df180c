// ops_abi.h -- the C entry points: argument checks, then launches on the caller's stream.
// A fragment of the ONE translation unit csrc/ops/ccsp_ops.hip (included there, inside extern "C"): not a standalone header.
// Nothing below allocates, throws or waits.

int32_t ccsp_ops_version(void) { return 1000 * CCSP_OPS_VERSION_MAJOR + CCSP_OPS_VERSION_MINOR; }
const char* ccsp_ops_last_error(void) { return g_err; }

int64_t ccsp_ops_route_workspace(int64_t n_assign, int32_t n_experts, int64_t n_tokens, int32_t list_tokens) {
    if (n_assign < 0 || n_assign > CCSP_OPS_MAX_ASSIGN || n_experts < 1 || n_experts > CCSP_OPS_MAX_EXPERTS || n_tokens < 0 || n_tokens > CCSP_OPS_MAX_ASSIGN) return -1;
    return 4 * (int64_t)route_workspace_ints(n_assign, n_experts, n_tokens, list_tokens != 0);
}

int ccsp_ops_route(const void* expert, const void* token, int32_t id_bits, int64_t n_assign, int32_t k, int32_t n_experts, int64_t n_tokens, int32_t* offsets, int32_t* rows, int32_t* assign,
                   int32_t* row_token, int32_t* place, int32_t* token_ptr, int32_t* token_assign, void* workspace, int64_t workspace_bytes, void* stream) {
    CCSP_OPS_CHECK(id_bits == 32 || id_bits == 64, "route: ids of 32 or 64 bits, not %d", id_bits);
    CCSP_OPS_CHECK(n_assign >= 0 && n_assign <= CCSP_OPS_MAX_ASSIGN, "route: %lld assignments out of range", (long long)n_assign);
    CCSP_OPS_CHECK(n_tokens >= 0 && n_tokens <= CCSP_OPS_MAX_ASSIGN, "route: %lld tokens out of range", (long long)n_tokens);
    CCSP_OPS_CHECK(n_experts >= 1 && n_experts <= CCSP_OPS_MAX_EXPERTS, "route: %d experts, supported are 1 to %d", n_experts, CCSP_OPS_MAX_EXPERTS);
    const bool list = token_ptr != nullptr;                      // (an empty list may have no address)
    CCSP_OPS_CHECK(list || (!token && k >= 1 && n_assign == n_tokens * k), "route: %lld assignments are not %lld tokens of %d each (list tokens need token_ptr)", (long long)n_assign, (long long)n_tokens, k);
    CCSP_OPS_CHECK(offsets && (n_assign == 0 || (expert && rows && assign && row_token && place)), "route: null argument");
    CCSP_OPS_CHECK(!list || n_assign == 0 || (token && token_assign), "route: list tokens need token, token_ptr and token_assign");
    CCSP_OPS_CHECK(workspace_bytes >= ccsp_ops_route_workspace(n_assign, n_experts, n_tokens, list) && (workspace || workspace_bytes == 0), "route: workspace of %lld bytes is too small",
                   (long long)workspace_bytes);
    const RouteIds r = {expert, token, id_bits == 64, (int)n_assign, k, n_experts, (int)n_tokens};
    const RouteOut o = {offsets, rows, assign, row_token, place, token_ptr, token_assign};
    return route(r, o, static_cast<int*>(workspace), (hipStream_t)stream);
}

static int check_rows(const char* who, int32_t type, int64_t n, int64_t width) {
    CCSP_OPS_CHECK(type_ok(type), "%s: element type %d", who, type);
    CCSP_OPS_CHECK(n >= 0 && n <= CCSP_OPS_MAX_ASSIGN && width >= 0 && width <= CCSP_OPS_MAX_WIDTH, "%s: %lld rows of width %lld out of range", who, (long long)n, (long long)width);
    return 0;
}

int ccsp_ops_rows_gather(int32_t type, int64_t n_rows, int64_t width, const void* src, int64_t src_stride, const int32_t* row_token, const int32_t* assign, const int32_t* place,
                         const int32_t* token_assign, void* dst, void* stream) {
    if (check_rows("rows_gather", type, n_rows, width)) return 1;
    if (n_rows == 0 || width == 0) return 0;
    CCSP_OPS_CHECK(row_token && assign && place && dst, "rows_gather: null argument");
    const long b = type_bytes(type) / 2;
    return rows_gather({row_token, assign, place, token_assign}, n_rows, (int)(width * b), src, src_stride * b, dst, width * b, (hipStream_t)stream);
}

int ccsp_ops_rows_combine(int32_t type, int64_t n_tokens, int64_t n_rows, int64_t width, int32_t k, const int32_t* token_ptr, const int32_t* token_assign, const int32_t* rows, const void* weight,
                          int32_t weight_type, const void* src, int64_t src_stride, void* dst, void* stream) {
    if (check_rows("rows_combine", type, n_tokens, width) || check_rows("rows_combine", type, n_rows, width)) return 1;
    CCSP_OPS_CHECK(token_ptr || n_rows == n_tokens * k, "rows_combine: %lld rows are not %lld tokens of %d each (list tokens need token_ptr)", (long long)n_rows, (long long)n_tokens, k);
    if (n_tokens == 0 || width == 0) return 0;
    CCSP_OPS_CHECK(dst && (n_rows == 0 || (rows && src)), "rows_combine: null argument");
    CCSP_OPS_CHECK(!token_ptr || n_rows == 0 || token_assign, "rows_combine: list tokens need token_assign");
    CCSP_OPS_CHECK(!weight || weight_type == CCSP_OPS_F32 || weight_type == type, "rows_combine: weights are 32 bits or of the rows' type");
    return dispatch_type(type, [&](auto t) {
        typedef decltype(t) T;
        return rows_combine<T>(n_tokens, n_rows, (int)width, k, token_ptr, token_assign, rows, weight, weight_type == CCSP_OPS_F32, (const T*)src, src_stride, (T*)dst, width, (hipStream_t)stream);
    });
}

int ccsp_ops_rows_back(int32_t type, int64_t n_rows, int64_t width, const int32_t* row_token, const int32_t* assign, const int32_t* place, const int32_t* token_assign, const void* weight, int32_t weight_type, const void* dy, int64_t dy_stride,
                       const void* src, int64_t src_stride, void* d_src, void* d_weight, void* stream) {
    if (check_rows("rows_back", type, n_rows, width)) return 1;
    if (n_rows == 0) return 0;
    CCSP_OPS_CHECK(assign && row_token && place && (width == 0 || (d_src || d_weight)), "rows_back: null argument");
    CCSP_OPS_CHECK(src || !d_weight || width == 0, "rows_back: null argument (the weights' gradient reads src)");
    CCSP_OPS_CHECK((!weight && !d_weight) || weight_type == CCSP_OPS_F32 || weight_type == type, "rows_back: weights are 32 bits or of the rows' type");
    return dispatch_type(type, [&](auto t) {
        typedef decltype(t) T;
        return rows_back<T>({row_token, assign, place, token_assign}, n_rows, (int)width, weight, weight_type == CCSP_OPS_F32, (const T*)dy, dy_stride, (const T*)src, src_stride, (T*)d_src, d_src ? width : 0, d_weight,
                            (hipStream_t)stream);
    });
}

static int check_linear(const char* who, int32_t type, int32_t n_experts, int64_t n_rows, int64_t inp, int64_t out, const int32_t* offsets) {
    CCSP_OPS_CHECK(type_ok(type), "%s: element type %d", who, type);
    CCSP_OPS_CHECK(n_experts >= 1 && n_experts <= CCSP_OPS_MAX_EXPERTS, "%s: %d experts, supported are 1 to %d", who, n_experts, CCSP_OPS_MAX_EXPERTS);
    CCSP_OPS_CHECK(n_rows >= 0 && n_rows <= CCSP_OPS_MAX_ASSIGN && inp >= 1 && inp <= CCSP_OPS_MAX_FEATURES && out >= 1 && out <= CCSP_OPS_MAX_FEATURES,
                   "%s: %lld rows, %lld -> %lld out of range", who, (long long)n_rows, (long long)inp, (long long)out);
    CCSP_OPS_CHECK(offsets, "%s: null argument", who);
    return 0;
}

int64_t ccsp_ops_linear_workspace(int32_t product, int32_t type, int32_t n_experts, int64_t n_rows, int64_t inp, int64_t out, const void* a, int64_t a_stride, const void* b, int64_t b_stride) {
    static const int32_t some = 0;
    if (product < CCSP_OPS_FORWARD || product > CCSP_OPS_BACK_WEIGHT || check_linear("linear_workspace", type, n_experts, n_rows, inp, out, &some)) return -1;
    int64_t bytes = 0;
    dispatch_type(type, [&](auto t) { bytes = product_workspace<decltype(t)>(product, n_experts, n_rows, inp, out, a, a_stride, b, b_stride); return 0; });
    return bytes;
}

int ccsp_ops_linear(int32_t type, int32_t n_experts, int64_t n_rows, int64_t inp, int64_t out, const int32_t* offsets, const void* x, int64_t x_stride, const void* weight, const void* bias,
                    int32_t activation, void* y, void* z, void* workspace, int64_t workspace_bytes, void* stream) {
    if (check_linear("linear", type, n_experts, n_rows, inp, out, offsets)) return 1;
    CCSP_OPS_CHECK(activation == CCSP_OPS_NONE || activation == CCSP_OPS_SILU, "linear: activation %d", activation);
    if (n_rows == 0) return 0;
    CCSP_OPS_CHECK(x && weight && y, "linear: null argument");
    ProdArgs p = {};
    p.bias = bias; p.c = y; p.ldc = out; p.z = z; p.offsets = offsets; p.E = n_experts; p.R = (int)n_rows; p.M = -1; p.N = (int)out; p.K = (int)inp; p.silu = activation == CCSP_OPS_SILU;
    p.seg_log2 = 31;
    return dispatch_type(type, [&](auto t) { return run_product<decltype(t), PROD_FORWARD>(p, inp, out, x, x_stride, weight, inp, workspace, workspace_bytes, (hipStream_t)stream); });
}

int ccsp_ops_linear_silu_back(int32_t type, int32_t n_experts, int64_t n_rows, int64_t out, const int32_t* offsets, const void* dy, int64_t dy_stride, const void* z, void* dz, void* stream) {
    if (check_linear("linear_silu_back", type, n_experts, n_rows, 1, out, offsets)) return 1;
    if (n_rows == 0) return 0;
    CCSP_OPS_CHECK(dy && z && dz, "linear_silu_back: null argument");
    return dispatch_type(type, [&](auto t) {
        typedef decltype(t) T;
        dispatch_vec<sizeof(T)>(out, [&](auto vc) {
            constexpr int V = decltype(vc)::value;
            const long n = cdiv(n_rows * cdiv(out, V), 256);
            hipLaunchKernelGGL((k_silu_back<T, V>), dim3((unsigned)(n < 8192 ? n : 8192)), dim3(256), 0, (hipStream_t)stream, offsets + n_experts, (int)out, (const T*)dy, (long)dy_stride, (const T*)z,
                               (T*)dz);
        });
        LAUNCHED();
        return 0;
    });
}

int ccsp_ops_linear_back_input(int32_t type, int32_t n_experts, int64_t n_rows, int64_t inp, int64_t out, const int32_t* offsets, const void* dz, int64_t dz_stride, const void* weight, void* dx,
                               void* workspace, int64_t workspace_bytes, void* stream) {
    if (check_linear("linear_back_input", type, n_experts, n_rows, inp, out, offsets)) return 1;
    if (n_rows == 0) return 0;
    CCSP_OPS_CHECK(dz && weight && dx, "linear_back_input: null argument");
    ProdArgs p = {};
    p.c = dx; p.ldc = inp; p.offsets = offsets; p.E = n_experts; p.R = (int)n_rows; p.M = -1; p.N = (int)inp; p.K = (int)out; p.seg_log2 = 31;
    return dispatch_type(type, [&](auto t) { return run_product<decltype(t), PROD_INPUT>(p, inp, out, dz, dz_stride, weight, inp, workspace, workspace_bytes, (hipStream_t)stream); });
}

int ccsp_ops_linear_back_weight(int32_t type, int32_t n_experts, int64_t n_rows, int64_t inp, int64_t out, const int32_t* offsets, const void* dz, int64_t dz_stride, const void* x, int64_t x_stride,
                                void* d_weight, void* d_bias, void* workspace, int64_t workspace_bytes, void* stream) {
    if (check_linear("linear_back_weight", type, n_experts, n_rows, inp, out, offsets)) return 1;
    CCSP_OPS_CHECK((n_rows == 0 || (dz && x)) && (d_weight || d_bias), "linear_back_weight: null argument");
    ProdArgs p = {};
    p.c = d_weight; p.ldc = inp; p.c_expert = inp * out; p.offsets = offsets; p.E = n_experts; p.R = (int)n_rows; p.M = (int)out; p.K = -1;
    p.sum = d_bias;                                              // (one kernel makes both; for the bias alone it goes over the first columns of x and writes no product)
    p.N = (int)(d_weight || inp < 64 ? inp : 64);
    return dispatch_type(type, [&](auto t) {
        typedef decltype(t) T;
        p.seg_log2 = seg_log2_for<T>(n_rows, n_experts, out, inp);
        return run_product<T, PROD_WEIGHT>(p, inp, out, dz, dz_stride, x, x_stride, workspace, workspace_bytes, (hipStream_t)stream);
    });
}

int64_t ccsp_ops_norm_workspace(int32_t n_tensors, const int64_t* sizes) {
    if (n_tensors < 0 || (n_tensors && !sizes)) return -1;
    int64_t b = 1;
    for (int32_t i = 0; i < n_tensors; ++i) if (sizes[i] < 0) return -1;
    const long chunk = norm_chunk_for(n_tensors, sizes);
    for (int32_t i = 0; i < n_tensors; ++i) b += cdiv(sizes[i], chunk);
    return 8 * b;
}

int ccsp_ops_clip_norm(int32_t n_tensors, const void* const* in, void* const* out, const int64_t* sizes, const int32_t* types, double max_norm, float* norm, float* scale, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    CCSP_OPS_CHECK(n_tensors >= 0 && norm && (n_tensors == 0 || (in && sizes && types)), "clip_norm: null argument");
    CCSP_OPS_CHECK(!out || scale, "clip_norm: clipping needs a place for the factor");
    CCSP_OPS_CHECK(!out || !(max_norm < 0.0), "clip_norm: max_norm %g is negative", max_norm);
    for (int32_t i = 0; i < n_tensors; ++i) {
        CCSP_OPS_CHECK(sizes[i] >= 0 && type_ok(types[i]), "clip_norm: tensor %d: size %lld, element type %d", i, (long long)sizes[i], types[i]);
        CCSP_OPS_CHECK(sizes[i] == 0 || (in[i] && (!out || out[i])), "clip_norm: tensor %d has no address", i);
    }
    CCSP_OPS_CHECK(workspace && workspace_bytes >= ccsp_ops_norm_workspace(n_tensors, sizes), "clip_norm: workspace of %lld bytes is too small", (long long)workspace_bytes);
    double* part = static_cast<double*>(workspace);
    hipStream_t s = (hipStream_t)stream;
    long total = 0;
    if (norm_tables(n_tensors, in, out, sizes, types, [&](const NormTable& t, int blocks, long before) {
            hipLaunchKernelGGL(k_norm_part, dim3((unsigned)blocks), dim3(256), 0, s, t, part + before);
            total = before + blocks;
            LAUNCHED();
            return 0;
        })) return 1;
    hipLaunchKernelGGL(k_norm_finish, dim3(1), dim3(1024), 0, s, (const double*)part, total, max_norm, norm, scale);
    LAUNCHED();
    if (!out) return 0;
    return norm_tables(n_tensors, in, out, sizes, types, [&](const NormTable& t, int blocks, long) {
        hipLaunchKernelGGL(k_norm_clip, dim3((unsigned)blocks), dim3(256), 0, s, t, blocks, (const float*)scale);
        LAUNCHED();
        return 0;
    });
}
