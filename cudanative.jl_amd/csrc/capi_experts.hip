// C ABI of the experts' operators and of the microscaled 4-bit matrices (declared in include/miwmma.h): checks of the
// arguments and dispatch.  Nothing here allocates or throws.
#include "../../include/miwmma.h"
#include "api_common.hpp"
#include "experts.hpp"

#include <algorithm>

namespace {

using miw::api_fail;

#define HIP_TRY(expr)                                                 \
    do {                                                              \
        hipError_t e_ = (expr);                                       \
        if (e_ != hipSuccess) return miw::api_hip_fail(e_, #expr);    \
    } while (0)
#define REQUIRE_INIT(what)                                                                                                   \
    do {                                                                                                                     \
        if (!miw::api_initialized())                                                                                         \
            return api_fail(MIW_ERR_NOT_INITIALIZED, "%s: miw_init has not been called (it selects the device and checks that it is a gfx950 part)", what); \
    } while (0)

bool half_type(int t) { return t == MIW_F16 || t == MIW_BF16; }
bool any_type(int t) { return half_type(t) || t == MIW_F32; }
long type_size(int t) { return t == MIW_F32 ? 4 : 2; }
bool aligned(const void *p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

constexpr int64_t EXTENT = 1 << 26;      // columns of a matrix, and lengths of sums
constexpr int64_t POSITIONS = 1 << 30;   // rows of a matrix
constexpr int64_t PITCH = 1ll << 30;     // elements or bytes from row to row
constexpr int64_t STRIDE = 1ll << 40;    // from group to group

// A pitch that is not given is the extent; *ld becomes the one that counts.
int check_pitch(const char *what, const char *name, int64_t *ld, int64_t extent)
{
    if (*ld == 0) *ld = extent;
    if (*ld < extent || *ld > PITCH)
        return api_fail(MIW_ERR_INVALID_VALUE, "%s: %s must be 0 or %lld .. %lld, got %lld", what, name, (long long)extent, (long long)PITCH, (long long)*ld);
    return 0;
}
int check_extent(const char *what, const char *name, int64_t v, int64_t low, int64_t high)
{
    if (v < low || v > high)
        return api_fail(MIW_ERR_INVALID_SHAPE, "%s: %s must be %lld .. %lld, got %lld", what, name, (long long)low, (long long)high, (long long)v);
    return 0;
}
int check_stride(const char *what, const char *name, int64_t *stride, int64_t dense)
{
    if (*stride == 0) *stride = dense;
    if (*stride < 0 || *stride > STRIDE) return api_fail(MIW_ERR_INVALID_VALUE, "%s: %s must be 0 .. %lld, got %lld", what, name, (long long)STRIDE, (long long)*stride);
    return 0;
}
int check_element(const char *what, const char *name, const void *p, long size)
{
    if (!p) return api_fail(MIW_ERR_NULL_POINTER, "%s: %s is null", what, name);
    if (!aligned(p, (uintptr_t)size)) return api_fail(MIW_ERR_MISALIGNED, "%s: %s is not aligned to %ld bytes", what, name, size);
    return 0;
}
#define CHECK(expr)                \
    do {                           \
        if (int rc_ = (expr)) return rc_; \
    } while (0)

int check_routing(const char *what, int dtype, int64_t tokens, int experts, int top)
{
    if (!any_type(dtype)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: unknown element type %d", what, dtype);
    CHECK(check_extent(what, "tokens", tokens, 0, POSITIONS));
    CHECK(check_extent(what, "experts", experts, 1, 1024));
    CHECK(check_extent(what, "top", top, 1, std::min(16, experts)));
    return check_extent(what, "tokens * top", tokens * top, 0, POSITIONS);
}

int check_epilogue(const char *what, int epilogue, int64_t n)
{
    if (epilogue != MIW_EPILOGUE_NONE && epilogue != MIW_EPILOGUE_GATED_SILU) return api_fail(MIW_ERR_INVALID_VALUE, "%s: unknown epilogue %d", what, epilogue);
    if (epilogue == MIW_EPILOGUE_GATED_SILU && n % 2) return api_fail(MIW_ERR_INVALID_SHAPE, "%s: the gated form needs an even n, got %lld", what, (long long)n);
    return 0;
}

int check_gated(const char *what, int dtype, int64_t rows, int64_t n)
{
    if (!half_type(dtype)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: unknown element type %d", what, dtype);
    CHECK(check_extent(what, "rows", rows, 0, POSITIONS));
    CHECK(check_extent(what, "n", n, 2, EXTENT));
    return check_epilogue(what, MIW_EPILOGUE_GATED_SILU, n);
}

// Codes and scales of rows x k values; *ldq, *lds become the pitches that count.
int check_mxfp4(const char *what, int64_t rows, int64_t k, int64_t *ldq, int64_t *lds, const void *codes, const void *scales)
{
    CHECK(check_pitch(what, "a pitch of codes", ldq, (k + 31) / 32 * 16));
    CHECK(check_pitch(what, "a pitch of scales", lds, rows + rows % 2));
    if (*ldq % 16 || *lds % 2) return api_fail(MIW_ERR_INVALID_VALUE, "%s: a pitch of codes is a multiple of 16 and one of scales even, got %lld and %lld", what, (long long)*ldq, (long long)*lds);
    CHECK(check_element(what, "a matrix' codes", codes, 16));
    return check_element(what, "a matrix' scales", scales, 16);
}

// Can results be stored four at a time (two in the gated form)?
bool stores_vectors(const void *D, int64_t ldd, int64_t sd, long size, bool gated)
{
    const long per = gated ? 2 : 4;
    return aligned(D, (uintptr_t)(per * size)) && ldd % per == 0 && sd % per == 0;
}

}  // namespace

extern "C" {

int miw_route_workspace(int64_t tokens, int experts, int top, size_t *bytes)
{
    if (!bytes) return api_fail(MIW_ERR_NULL_POINTER, "route_workspace: null output pointer");
    CHECK(check_routing("route_workspace", MIW_F32, tokens, experts, top));
    const int chunks = miw::route_most_chunks(tokens);
    *bytes = chunks == 1 ? 0 : (size_t)chunks * (size_t)experts * sizeof(int);
    return 0;
}

int miw_route(int dtype, int64_t tokens, int experts, int top, int64_t ld, int over_all, const void *logits, int *chosen,
              float *gates, int *offsets, int *rows, int *place, void *workspace, size_t workspace_bytes, void *stream)
{
    CHECK(check_routing("route", dtype, tokens, experts, top));
    CHECK(check_pitch("route", "ld", &ld, experts));
    CHECK(check_element("route", "offsets", offsets, 4));
    if (tokens) {
        CHECK(check_element("route", "logits", logits, type_size(dtype)));
        CHECK(check_element("route", "chosen", chosen, 4));
        CHECK(check_element("route", "gates", gates, 4));
        CHECK(check_element("route", "rows", rows, 4));
        CHECK(check_element("route", "place", place, 4));
    }
    size_t need = 0;
    CHECK(miw_route_workspace(tokens, experts, top, &need));
    if (need) {
        CHECK(check_element("route", "workspace", workspace, 16));
        if (workspace_bytes < need) return api_fail(MIW_ERR_INVALID_VALUE, "route: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
    }
    REQUIRE_INIT("route");
    miw::route_params p{};
    p.logits = logits;
    p.chosen = chosen;
    p.gates = gates;
    p.offsets = offsets;
    p.rows = rows;
    p.place = place;
    p.counts = (int *)workspace;
    p.tokens = (int)tokens;
    p.experts = experts;
    p.top = top;
    p.over_all = over_all != 0;
    p.ld = ld;
    HIP_TRY(miw::launch_route(p, dtype, (hipStream_t)stream));
    return 0;
}

int miw_route_grad(int dtype, int64_t tokens, int experts, int top, int64_t ld, int64_t ldd, int over_all, const void *logits,
                   const int *chosen, const float *gates, const float *dgates, void *dlogits, void *stream)
{
    CHECK(check_routing("route_grad", dtype, tokens, experts, top));
    CHECK(check_pitch("route_grad", "ld", &ld, experts));
    CHECK(check_pitch("route_grad", "ldd", &ldd, experts));
    if (!tokens) return 0;
    CHECK(check_element("route_grad", "logits", logits, type_size(dtype)));
    CHECK(check_element("route_grad", "chosen", chosen, 4));
    CHECK(check_element("route_grad", "gates", gates, 4));
    CHECK(check_element("route_grad", "dgates", dgates, 4));
    CHECK(check_element("route_grad", "dlogits", dlogits, type_size(dtype)));
    REQUIRE_INIT("route_grad");
    const miw::route_grad_params p{logits, chosen, gates, dgates, dlogits, (int)tokens, experts, top, over_all != 0, ld, ldd};
    HIP_TRY(miw::launch_route_grad(p, dtype, (hipStream_t)stream));
    return 0;
}

int miw_grouped_gemm(int dtype, int d_type, int w_layout, int epilogue, int64_t rows, int groups, int64_t n, int64_t k,
                     int64_t lda, int64_t ldw, int64_t stride_w, int64_t ldd, int64_t a_rows, const void *A, const void *W,
                     void *D, const int *offsets, const int *gather, void *stream)
{
    const char *what = "grouped_gemm";
    if (!half_type(dtype) || (d_type != dtype && d_type != MIW_F32)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: element types %d and %d", what, dtype, d_type);
    if (w_layout != MIW_ROW_MAJOR && w_layout != MIW_COL_MAJOR) return api_fail(MIW_ERR_INVALID_LAYOUT, "%s: unknown layout %d", what, w_layout);
    CHECK(check_extent(what, "rows", rows, 0, POSITIONS));
    CHECK(check_extent(what, "groups", groups, 1, 65536));
    CHECK(check_extent(what, "n", n, 1, EXTENT));
    CHECK(check_extent(what, "k", k, 1, EXTENT));
    CHECK(check_epilogue(what, epilogue, n));
    const bool k_major = w_layout == MIW_COL_MAJOR, gated = epilogue == MIW_EPILOGUE_GATED_SILU;
    CHECK(check_pitch(what, "lda", &lda, k));
    CHECK(check_pitch(what, "ldw", &ldw, k_major ? k : n));
    CHECK(check_pitch(what, "ldd", &ldd, gated ? n / 2 : n));
    CHECK(check_stride(what, "stride_w", &stride_w, ldw * (k_major ? n : k)));
    if (a_rows == 0 && !gather) a_rows = rows;
    CHECK(check_extent(what, "a_rows", a_rows, gather ? (rows ? 1 : 0) : rows, POSITIONS));
    if (rows == 0) return 0;
    CHECK(check_element(what, "A", A, 2));
    CHECK(check_element(what, "W", W, 2));
    CHECK(check_element(what, "D", D, type_size(d_type)));
    CHECK(check_element(what, "offsets", offsets, 4));
    if (gather) CHECK(check_element(what, "gather", gather, 4));
    REQUIRE_INIT(what);
    miw::grouped_params p{};
    p.X = (const char *)W;
    p.Y = (const char *)A;
    p.offsets = offsets;
    p.gather = gather;
    p.D = D;
    p.groups = groups;
    p.rows = (int)rows;
    p.source_rows = (int)a_rows;
    p.I = (int)n;
    p.K = (int)k;
    p.ldx = ldw * 2;
    p.ldy = lda * 2;
    p.ldd = ldd;
    p.sx = stride_w * 2;
    p.x_k_major = k_major;
    p.gated = gated;
    p.vector = aligned(A, 16) && aligned(W, 16) && lda % 8 == 0 && ldw % 8 == 0 && stride_w % 8 == 0 && k % 8 == 0 && (k_major || n % 8 == 0);
    p.d_vector = stores_vectors(D, ldd, 0, type_size(d_type), gated);
    HIP_TRY(miw::launch_grouped(p, dtype, d_type, false, miw::api_cu_count(), (hipStream_t)stream));
    return 0;
}

int miw_grouped_wgrad(int dtype, int d_type, int accumulate, int64_t rows, int groups, int64_t m, int64_t n, int64_t lda,
                      int64_t ldb, int64_t ldd, int64_t stride_d, int64_t b_rows, const void *A, const void *B, void *D,
                      const int *offsets, const int *gather, void *stream)
{
    const char *what = "grouped_wgrad";
    if (!half_type(dtype) || (d_type != dtype && d_type != MIW_F32)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: element types %d and %d", what, dtype, d_type);
    CHECK(check_extent(what, "rows", rows, 0, POSITIONS));
    CHECK(check_extent(what, "groups", groups, 1, 65536));
    CHECK(check_extent(what, "m", m, 1, EXTENT));
    CHECK(check_extent(what, "n", n, 1, EXTENT));
    CHECK(check_pitch(what, "lda", &lda, m));
    CHECK(check_pitch(what, "ldb", &ldb, n));
    CHECK(check_pitch(what, "ldd", &ldd, n));
    CHECK(check_stride(what, "stride_d", &stride_d, ldd * m));
    if (groups > 1 && stride_d < ldd * (m - 1) + n) return api_fail(MIW_ERR_INVALID_VALUE, "%s: results of neighbouring groups overlap", what);
    if (b_rows == 0 && !gather) b_rows = rows;
    CHECK(check_extent(what, "b_rows", b_rows, gather ? (rows ? 1 : 0) : rows, POSITIONS));
    if (rows) {
        CHECK(check_element(what, "A", A, 2));
        CHECK(check_element(what, "B", B, 2));
        if (gather) CHECK(check_element(what, "gather", gather, 4));
    }
    CHECK(check_element(what, "D", D, type_size(d_type)));
    CHECK(check_element(what, "offsets", offsets, 4));
    REQUIRE_INIT(what);
    miw::grouped_params p{};
    p.X = (const char *)B;
    p.Y = (const char *)A;
    p.offsets = offsets;
    p.gather = gather;
    p.D = D;
    p.groups = groups;
    p.rows = (int)rows;
    p.source_rows = (int)b_rows;
    p.I = (int)n;
    p.J = (int)m;
    p.ldx = ldb * 2;
    p.ldy = lda * 2;
    p.ldd = ldd;
    p.sd = stride_d;
    p.accumulate = accumulate != 0;
    p.vector = aligned(A, 16) && aligned(B, 16) && lda % 8 == 0 && ldb % 8 == 0 && m % 8 == 0 && n % 8 == 0;
    p.d_vector = stores_vectors(D, ldd, stride_d, type_size(d_type), false);
    HIP_TRY(miw::launch_grouped(p, dtype, d_type, true, miw::api_cu_count(), (hipStream_t)stream));
    return 0;
}

int miw_combine(int dtype, int64_t tokens, int top, int64_t n, int64_t rows, int64_t ldh, int64_t ldy, const void *H,
                const float *gates, const int *place, void *Y, void *stream)
{
    const char *what = "combine";
    if (!half_type(dtype)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: unknown element type %d", what, dtype);
    CHECK(check_extent(what, "tokens", tokens, 0, (1 << 24) - 1));
    CHECK(check_extent(what, "top", top, 1, 1 << 16));
    CHECK(check_extent(what, "n", n, 1, EXTENT));
    CHECK(check_extent(what, "rows", rows, 0, POSITIONS));
    CHECK(check_pitch(what, "ldh", &ldh, n));
    CHECK(check_pitch(what, "ldy", &ldy, n));
    if (!tokens) return 0;
    if (rows) CHECK(check_element(what, "H", H, 2));
    if (gates) CHECK(check_element(what, "gates", gates, 4));
    CHECK(check_element(what, "place", place, 4));
    CHECK(check_element(what, "Y", Y, 2));
    REQUIRE_INIT(what);
    miw::combine_params p{};
    p.H = H;
    p.gates = gates;
    p.place = place;
    p.out = Y;
    p.tokens = (int)tokens;
    p.top = top;
    p.rows = (int)rows;
    p.n = n;
    p.ldh = ldh;
    p.ldy = ldy;
    p.vector = aligned(H, 16) && aligned(Y, 16) && n % 8 == 0 && ldh % 8 == 0 && ldy % 8 == 0;
    HIP_TRY(miw::launch_combine(p, dtype, (hipStream_t)stream));
    return 0;
}

int miw_combine_grad(int dtype, int64_t tokens, int top, int64_t n, int64_t rows, int64_t ldy, int64_t ldh, int64_t lddh,
                     const void *dY, const void *H, const float *gates, const int *place, void *dH, float *dgates, void *stream)
{
    const char *what = "combine_grad";
    if (!half_type(dtype)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: unknown element type %d", what, dtype);
    CHECK(check_extent(what, "tokens", tokens, 0, (1 << 24) - 1));
    CHECK(check_extent(what, "top", top, 1, 1 << 16));
    CHECK(check_extent(what, "n", n, 1, EXTENT));
    CHECK(check_extent(what, "rows", rows, 0, POSITIONS));
    CHECK(check_pitch(what, "ldy", &ldy, n));
    CHECK(check_pitch(what, "ldh", &ldh, n));
    CHECK(check_pitch(what, "lddh", &lddh, n));
    if (!tokens) return 0;
    CHECK(check_element(what, "dY", dY, 2));
    if (gates) CHECK(check_element(what, "gates", gates, 4));
    CHECK(check_element(what, "place", place, 4));
    if (rows) CHECK(check_element(what, "dH", dH, 2));
    if (dgates) {
        CHECK(check_element(what, "dgates", dgates, 4));
        if (rows) CHECK(check_element(what, "H", H, 2));
    }
    REQUIRE_INIT(what);
    miw::combine_params p{};
    p.H = H;
    p.dY = dY;
    p.gates = gates;
    p.place = place;
    p.out = dH;
    p.dgates = dgates;
    p.tokens = (int)tokens;
    p.top = top;
    p.rows = (int)rows;
    p.n = n;
    p.ldh = ldh;
    p.ldy = ldy;
    p.lddh = lddh;
    p.vector = aligned(dY, 16) && aligned(dH, 16) && (!dgates || aligned(H, 16)) && n % 8 == 0 && ldh % 8 == 0 && ldy % 8 == 0 && lddh % 8 == 0;
    HIP_TRY(miw::launch_combine_grad(p, dtype, (hipStream_t)stream));
    return 0;
}

int miw_gated_silu(int dtype, int64_t rows, int64_t n, int64_t ldz, int64_t lda, const void *Z, void *A, void *stream)
{
    const char *what = "gated_silu";
    CHECK(check_gated(what, dtype, rows, n));
    CHECK(check_pitch(what, "ldz", &ldz, n));
    CHECK(check_pitch(what, "lda", &lda, n / 2));
    if (!rows) return 0;
    CHECK(check_element(what, "Z", Z, 2));
    CHECK(check_element(what, "A", A, 2));
    REQUIRE_INIT(what);
    miw::gated_params p{};
    p.Z = Z;
    p.out = A;
    p.rows = rows;
    p.n = n;
    p.ldz = ldz;
    p.ldo = lda;
    p.vector = aligned(Z, 16) && aligned(A, 8) && n % 8 == 0 && ldz % 8 == 0 && lda % 4 == 0;
    HIP_TRY(miw::launch_gated_silu(p, dtype, (hipStream_t)stream));
    return 0;
}

int miw_gated_silu_grad(int dtype, int64_t rows, int64_t n, int64_t ldz, int64_t ldda, int64_t lddz, const void *Z, const void *dA,
                        void *dZ, void *stream)
{
    const char *what = "gated_silu_grad";
    CHECK(check_gated(what, dtype, rows, n));
    CHECK(check_pitch(what, "ldz", &ldz, n));
    CHECK(check_pitch(what, "ldda", &ldda, n / 2));
    CHECK(check_pitch(what, "lddz", &lddz, n));
    if (!rows) return 0;
    CHECK(check_element(what, "Z", Z, 2));
    CHECK(check_element(what, "dA", dA, 2));
    CHECK(check_element(what, "dZ", dZ, 2));
    if (dZ == Z && lddz != ldz)
        return api_fail(MIW_ERR_INVALID_VALUE, "%s: dZ in Z's place needs Z's pitch, got %lld and %lld", what, (long long)lddz, (long long)ldz);
    REQUIRE_INIT(what);
    miw::gated_params p{};
    p.Z = Z;
    p.dA = dA;
    p.out = dZ;
    p.rows = rows;
    p.n = n;
    p.ldz = ldz;
    p.ldda = ldda;
    p.ldo = lddz;
    p.vector = aligned(Z, 16) && aligned(dA, 8) && aligned(dZ, 16) && n % 8 == 0 && ldz % 8 == 0 && ldda % 4 == 0 && lddz % 8 == 0;
    HIP_TRY(miw::launch_gated_silu(p, dtype, (hipStream_t)stream));
    return 0;
}

int miw_mxfp4_quantize(int dtype, int64_t rows, int64_t k, int64_t ld, int64_t ldq, int64_t lds, const void *X, void *codes,
                       void *scales, void *stream)
{
    const char *what = "mxfp4_quantize";
    if (!any_type(dtype)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: unknown element type %d", what, dtype);
    CHECK(check_extent(what, "rows", rows, 0, POSITIONS));
    CHECK(check_extent(what, "k", k, 1, EXTENT));
    CHECK(check_pitch(what, "ld", &ld, k));
    if (!rows) return 0;
    CHECK(check_mxfp4(what, rows, k, &ldq, &lds, codes, scales));
    CHECK(check_element(what, "X", X, type_size(dtype)));
    REQUIRE_INIT(what);
    miw::mxfp4_convert_params p{};
    p.in = X;
    p.codes = (uint8_t *)codes;
    p.scales = (uint8_t *)scales;
    p.rows = rows;
    p.k = k;
    p.ld = ld;
    p.ldq = ldq;
    p.lds = lds;
    p.vector = aligned(X, 16) && ld * type_size(dtype) % 16 == 0;
    HIP_TRY(miw::launch_mxfp4_quantize(p, dtype, (hipStream_t)stream));
    return 0;
}

int miw_mxfp4_dequantize(int dtype, int64_t rows, int64_t k, int64_t ldq, int64_t lds, int64_t ld, const void *codes,
                         const void *scales, void *X, void *stream)
{
    const char *what = "mxfp4_dequantize";
    if (!any_type(dtype)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: unknown element type %d", what, dtype);
    CHECK(check_extent(what, "rows", rows, 0, POSITIONS));
    CHECK(check_extent(what, "k", k, 1, EXTENT));
    CHECK(check_pitch(what, "ld", &ld, k));
    if (!rows) return 0;
    CHECK(check_mxfp4(what, rows, k, &ldq, &lds, codes, scales));
    CHECK(check_element(what, "X", X, type_size(dtype)));
    REQUIRE_INIT(what);
    miw::mxfp4_convert_params p{};
    p.out = X;
    p.codes = (uint8_t *)codes;
    p.scales = (uint8_t *)scales;
    p.rows = rows;
    p.k = k;
    p.ld = ld;
    p.ldq = ldq;
    p.lds = lds;
    p.vector = aligned(X, 16) && ld * type_size(dtype) % 16 == 0;
    HIP_TRY(miw::launch_mxfp4_dequantize(p, dtype, (hipStream_t)stream));
    return 0;
}

}  // extern "C"

namespace {

int mxfp4_product(const char *what, int d_type, int epilogue, int64_t rows, int groups, int64_t n, int64_t k, int64_t lda, int64_t lds_a,
                  int64_t ldw, int64_t lds_w, int64_t stride_w, int64_t stride_ws, int64_t ldd, int64_t a_rows, const void *A,
                  const void *A_scales, const void *W, const void *W_scales, void *D, const int *offsets, const int *gather, void *stream)
{
    if (!any_type(d_type)) return api_fail(MIW_ERR_INVALID_TYPE, "%s: unknown element type %d", what, d_type);
    CHECK(check_extent(what, "rows", rows, 0, POSITIONS));
    CHECK(check_extent(what, "groups", groups, 1, 65536));
    CHECK(check_extent(what, "n", n, 1, EXTENT));
    CHECK(check_extent(what, "k", k, 1, EXTENT));
    CHECK(check_epilogue(what, epilogue, n));
    const bool gated = epilogue == MIW_EPILOGUE_GATED_SILU;
    CHECK(check_pitch(what, "ldd", &ldd, gated ? n / 2 : n));
    if (a_rows == 0 && !gather) a_rows = rows;
    CHECK(check_extent(what, "a_rows", a_rows, gather ? (rows ? 1 : 0) : rows, POSITIONS));
    if (rows == 0) return 0;
    CHECK(check_mxfp4(what, a_rows, k, &lda, &lds_a, A, A_scales));
    CHECK(check_mxfp4(what, n, k, &ldw, &lds_w, W, W_scales));
    CHECK(check_stride(what, "stride_w", &stride_w, n * ldw));
    CHECK(check_stride(what, "stride_ws", &stride_ws, (k + 255) / 256 * lds_w * 8));
    if (stride_w % 16 || stride_ws % 16) return api_fail(MIW_ERR_MISALIGNED, "%s: strides from group to group are multiples of 16 bytes", what);
    CHECK(check_element(what, "D", D, type_size(d_type)));
    if (gather) CHECK(check_element(what, "gather", gather, 4));
    REQUIRE_INIT(what);
    miw::grouped_params p{};
    p.X = (const char *)W;
    p.Y = (const char *)A;
    p.xs = (const uint8_t *)W_scales;
    p.ys = (const uint8_t *)A_scales;
    p.offsets = offsets;
    p.gather = gather;
    p.D = D;
    p.groups = groups;
    p.rows = (int)rows;
    p.source_rows = (int)a_rows;
    p.I = (int)n;
    p.K = (int)k;
    p.ldx = ldw;
    p.ldy = lda;
    p.ldd = ldd;
    p.sx = stride_w;
    p.sxs = stride_ws;
    p.lxs = lds_w;
    p.lys = lds_a;
    p.x_k_major = 1;
    p.gated = gated;
    p.vector = 1;
    p.d_vector = stores_vectors(D, ldd, 0, type_size(d_type), gated);
    HIP_TRY(miw::launch_grouped_mxfp4(p, d_type, miw::api_cu_count(), (hipStream_t)stream));
    return 0;
}

}  // namespace

extern "C" {

int miw_mxfp4_gemm(int d_type, int epilogue, int64_t m, int64_t n, int64_t k, int64_t lda, int64_t lds_a, int64_t ldb,
                   int64_t lds_b, int64_t ldd, const void *A, const void *A_scales, const void *B, const void *B_scales, void *D,
                   void *stream)
{
    return mxfp4_product("mxfp4_gemm", d_type, epilogue, m, 1, n, k, lda, lds_a, ldb, lds_b, 0, 0, ldd, m, A, A_scales, B, B_scales, D, nullptr, nullptr, stream);
}

int miw_mxfp4_grouped_gemm(int d_type, int epilogue, int64_t rows, int groups, int64_t n, int64_t k, int64_t lda, int64_t lds_a,
                           int64_t ldw, int64_t lds_w, int64_t stride_w, int64_t stride_ws, int64_t ldd, int64_t a_rows,
                           const void *A, const void *A_scales, const void *W, const void *W_scales, void *D, const int *offsets,
                           const int *gather, void *stream)
{
    if (!offsets) return api_fail(MIW_ERR_NULL_POINTER, "mxfp4_grouped_gemm: offsets is null");
    CHECK(check_element("mxfp4_grouped_gemm", "offsets", offsets, 4));
    return mxfp4_product("mxfp4_grouped_gemm", d_type, epilogue, rows, groups, n, k, lda, lds_a, ldw, lds_w, stride_w, stride_ws, ldd, a_rows, A, A_scales,
                         W, W_scales, D, offsets, gather, stream);
}

}  // extern "C"
