// gated_ffn.cu -- the gated feed-forward block and its gradient.
//
// Forward: g = x wg^T, u = x wu^T, y = act(g) * u. Backward, from dy and the kept g and u:
// du = dy * act(g), dg = dy * u * act'(g), dx = dg wg + du wu, dwg = dg^T x, dwu = du^T x.
// Sums are held in fp32; dg and du are rounded to the operands' 16-bit type before the products,
// as any 16-bit matrix product's operand is. Where the terms of a sum are independent that makes a gradient's
// error sqrt 2 times its own rounding's; where they cancel, more; and an fp16 dg or du past 65504 is infinite.
// Products of what the rounding leaves off, added on, would take as long again as the products themselves.
//
// The products run on the tensor cores (gated_tc.cuh). TMA needs 16-byte rows: an operand whose
// address or row stride is not is first copied to scratch with a stride that is.
#include "gated_few.cuh"
#include "gated_small.cuh"
#include "gated_tc.cuh"

#include <initializer_list>

namespace xspmm_b200 {
namespace {

using namespace gated;

int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }

// Eight elements from anywhere in a matrix (bytes [begin, end)): the two aligned 16-byte words that hold
// them, shifted together; words that reach outside, and the `valid` < 8 at a row's end, element by element,
// with zeros after them.
template <typename T>
__device__ __forceinline__ uint4 load_shifted(const T* src, int64_t valid, uintptr_t begin, uintptr_t end) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(src), low = at & ~uintptr_t(15);
    const int shift = (int)(at & 15);
    uint32_t out[4];
    if (valid >= 8 && low >= begin && low + (shift ? 32 : 16) <= end) {
        const uint4 v0 = __ldg(reinterpret_cast<const uint4*>(low));
        const uint4 v1 = shift ? __ldg(reinterpret_cast<const uint4*>(low) + 1) : v0;
        uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
        if (shift & 8)
#pragma unroll
            for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
        if (shift & 4)
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __funnelshift_r(w[i], w[i + 1], (shift & 2) * 8);
    } else {
        const uint16_t* e = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = 2 * i < valid ? e[2 * i] : 0u;
            const uint32_t hi = 2 * i + 1 < valid ? e[2 * i + 1] : 0u;
            out[i] = lo | hi << 16;
        }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// dg and du with row stride ldp = round8(F), 8 elements a thread. WIDE: F and the rows of dy, gate and up
// allow 16-byte loads; otherwise the words are shifted together, which costs less than element by element
// (gradient of 2107 rows, 48 -> 4311: 59 us, 67 so).
template <typename T, Activation ACT, bool WIDE>
__global__ void __launch_bounds__(256)
gated_slopes_kernel(int64_t rows, int64_t F, const T* __restrict__ dy, int64_t lddy,
                    const T* __restrict__ gate, const T* __restrict__ up, T* __restrict__ dg,
                    T* __restrict__ du, int64_t ldp) {
    const int64_t per = ldp / 8;
    auto load = [&](const T* p, int64_t ld, int64_t r, int64_t c) {
        if constexpr (WIDE) return *reinterpret_cast<const uint4*>(p + r * ld + c);
        else return load_shifted(p + r * ld + c, F - c, reinterpret_cast<uintptr_t>(p),
                                 reinterpret_cast<uintptr_t>(p + (rows - 1) * ld + F));
    };
    cudaGridDependencySynchronize();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per;
         i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per, c = (i - r * per) * 8;
        const uint4 d = load(dy, lddy, r, c), g = load(gate, F, r, c), u = load(up, F, r, c);
        const uint32_t dw[4] = {d.x, d.y, d.z, d.w}, gw[4] = {g.x, g.y, g.z, g.w}, uw[4] = {u.x, u.y, u.z, u.w};
        uint32_t a[4], b[4];
        slope_words<ACT, T>(a, b, dw, gw, uw);
        *reinterpret_cast<uint4*>(dg + r * ldp + c) = make_uint4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<uint4*>(du + r * ldp + c) = make_uint4(b[0], b[1], b[2], b[3]);
    }
}

// Copies of up to three matrices to row strides that TMA can take, in one launch.
template <typename T>
struct Restride {
    struct {
        const T* src;
        T* dst;
        int64_t rows, cols, ld, ldp;
    } m[3];
};
// A warp per row, 8 elements a lane. The row's padding becomes zeros.
template <typename T>
__global__ void __launch_bounds__(256) restride_kernel(const __grid_constant__ Restride<T> a) {
    const auto& m = a.m[blockIdx.y];
    cudaGridDependencySynchronize();
    const uintptr_t begin = reinterpret_cast<uintptr_t>(m.src);
    const uintptr_t end = reinterpret_cast<uintptr_t>(m.src + (m.rows - 1) * m.ld + m.cols);
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < m.rows; r += (int64_t)gridDim.x * 8)
        for (int64_t c = (threadIdx.x & 31) * 8; c < m.cols; c += 256)
            *reinterpret_cast<uint4*>(m.dst + r * m.ldp + c) =
                load_shifted(m.src + r * m.ld + c, m.cols - c, begin, end);
}

// Matrices as TMA can read them: the caller's, or copies in scratch.
template <typename T>
struct Operands {
    struct Rows {
        const T* p;
        int64_t ld, rows, cols;
    };
    Rows m[3];
    DevBuf<T> copy[3];
    Operands(Handle& h, std::initializer_list<Rows> list) {
        Restride<T> job = {};
        int n = 0, jobs = 0;
        int64_t most = 0;
        for (Rows r : list) {
            if (r.rows <= 1) r.ld = round8(r.cols);  // the stride of a single row is never taken
            if (!tma_ok(r.p, r.ld)) {
                const int64_t ldp = round8(r.cols);
                copy[n] = DevBuf<T>((size_t)(r.rows * ldp), h.stream);
                job.m[jobs++] = {r.p, copy[n].get(), r.rows, r.cols, r.ld, ldp};
                most = std::max(most, r.rows);
                r.p = copy[n].get();
                r.ld = ldp;
            }
            m[n++] = r;
        }
        if (jobs == 0) return;
        const dim3 grid((unsigned)std::min(ceil_div(most, 8), (int64_t)sm_count(h.device) * 8), (unsigned)jobs);
        launch_dependent(h.stream, restride_kernel<T>, grid, 256, 0, 1, job);
        after_launch(h, "gated_restride");
    }
    CUtensorMap map(int i, int box_rows) const {
        return make_map_2d(m[i].p, (uint64_t)m[i].cols, (uint64_t)m[i].rows, (uint64_t)m[i].ld * 2, 64,
                           (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
    }
};

template <typename T>
CUtensorMap map_of(const T* p, int64_t ld, int64_t rows, int64_t cols, int box_rows) {
    return make_map_2d(p, (uint64_t)cols, (uint64_t)rows, (uint64_t)ld * 2, 64, (uint32_t)box_rows,
                       CU_TENSOR_MAP_SWIZZLE_128B);
}

// Picks a product's tile width, and how many slices the tiles are cut into that do not fill a wave of the
// GPU's SMs. The model, in clocks: a 64-deep slice of a tile costs an SM the slower of its MMAs (2 per
// accumulator column, at least 64 columns' worth), of shared memory written and read at 128 bytes a
// clock, and of its loads at about 56 bytes a clock (measured: 2048 tokens of 4096 x 11008 forward take
// 275 us with the loads left out and 299 with them); a tile adds a fill and drain. A split costs a
// second kernel and its partials' trip through L2.
template <Product P, int CG>
void choose_tiles(Handle& h, TileArgs& t) {
    const int slots = sm_count(h.device) / CG;
    const int unit = P == Product::Forward ? 8 * CG : 16 * CG;  // MMA N: a multiple of 16, in a pair of 32
    const int widest = P == Product::Forward ? 128 : 256;
    const double a_bytes = P == Product::Dw ? A_BYTES : 128.0 * (double)std::min<int64_t>(t.M, TM);
    double least = -1.0;
    for (int bn = unit; bn <= widest; bn += unit) {
        // Dx and Dw load whole 64-column chunks: other widths only where the output is narrower
        if (P != Product::Forward && bn % (32 * CG) != 0 && bn < t.N) continue;
        const int acc = acc_columns<P, CG>(bn);
        const double b_bytes = P == Product::Forward ? 128.0 * acc / CG : (double)((acc / CG + 63) / 64 * CHUNK);
        const double step = std::max({2.0 * std::max(acc, 64), 2.0 * (A_BYTES + b_bytes) / 128.0, (a_bytes + b_bytes) / 56.0});
        const double ends = 1500.0 + 6.0 * acc;
        const int64_t nt = ceil_div(t.N, bn), tiles = t.mt * nt;
        const int64_t whole = tiles / slots * slots, rest = tiles - whole;
        const double full = (double)(tiles / slots) * (t.ksteps * step + ends);
        const int64_t most = rest > 0 ? std::max<int64_t>(1, std::min<int64_t>(slots / rest, t.ksteps / 4)) : 1;
        for (int64_t sp = 1; sp <= most; ++sp) {
            double cost = full;
            if (rest > 0) cost += (double)ceil_div(t.ksteps, sp) * step + ends;
            if (sp > 1) cost += 6000.0 + (double)(rest * sp) * TM * CG * acc * 8.0 / 3000.0;
            if (least < 0.0 || cost < least) {
                least = cost;
                t.bn = bn;
                t.nt = (int)nt;
                t.splits = (int)sp;
                t.whole = (int)(sp > 1 ? whole : tiles);
            }
        }
        if (bn >= t.N) break;
    }
}

template <typename T>
void zero_rows(Handle& h, T* p, int64_t ld, int64_t rows, int64_t cols) {
    if (p && rows > 0 && cols > 0)
        XS_CHECK_CUDA(cudaMemset2DAsync(p, ld * sizeof(T), 0, cols * sizeof(T), rows, h.stream));
}

template <typename T>
void check_sizes(const GatedArgs<T>& a) {
    const int64_t most = (int64_t(1) << 31) - 512;  // TMA coordinates are 32 bits
    XS_REQUIRE(a.rows < most && a.K < most && a.F < most, XSPMM_STATUS_UNSUPPORTED,
               "a dimension of the gated feed-forward block passes 2^31");
}

}  // namespace

template <typename T>
void gated_ffn(Handle& h, const GatedArgs<T>& a, T* y, int64_t ldy, T* gate, T* up) {
    if (a.rows == 0 || a.F == 0) return;
    check_sizes(a);
    if (a.K == 0) {  // sums of no terms
        zero_rows(h, y, ldy, a.rows, a.F);
        zero_rows(h, gate, a.F, a.rows, a.F);
        zero_rows(h, up, a.F, a.rows, a.F);
        return;
    }
    if (a.rows <= 16) {
        few_rows(h, a, y, ldy, gate, up);
        return;
    }
    const Operands<T> in(h, {{a.x, a.ldx, a.rows, a.K}, {a.wg, a.ldwg, a.F, a.K}, {a.wu, a.ldwu, a.F, a.K}});
    TileArgs t = {};
    t.M = a.rows;
    t.N = a.F;
    const int cg = a.rows > TM ? 2 : 1;
    t.mt = (int)ceil_div(a.rows, TM * cg);
    t.ksteps = t.kseg = (int)ceil_div(a.K, TK);
    t.cols_first = a.rows > 2 * a.F;  // the operand of the inner index is read again and should fit L2
    if (cg == 2) choose_tiles<Product::Forward, 2>(h, t);
    else choose_tiles<Product::Forward, 1>(h, t);
    t.a[0] = in.map(0, TM);
    t.b[0] = in.map(1, t.bn);
    t.b[1] = in.map(2, t.bn);
    t.act = a.act;
    set_output(t, 0, y, ldy);
    set_output(t, 1, gate, a.F);
    set_output(t, 2, up, a.F);
    if (cg == 2) launch_product<T, Product::Forward, 2>(h, t);
    else launch_product<T, Product::Forward, 1>(h, t);
}

template <typename T>
void gated_ffn_backward(Handle& h, const GatedArgs<T>& a, const T* dy, int64_t lddy, const T* gate,
                        const T* up, T* dx, int64_t lddx, T* dwg, T* dwu) {
    check_sizes(a);
    const int sms = sm_count(h.device);
    if (a.rows == 0 || a.F == 0 || a.K == 0) {
        zero_rows(h, dx, lddx, a.rows, a.K);
        zero_rows(h, dwg, a.K, a.F, a.K);
        zero_rows(h, dwu, a.K, a.F, a.K);
        return;
    }
    if (!dx && !dwg) return;
    if (small_grad_ok(a, dy, lddy, gate, up, dx, lddx, dwg)) {
        small_grad(h, a, dy, lddy, gate, up, dx, lddx, dwg, dwu);
        return;
    }
    const int64_t ldp = round8(a.F);
    DevBuf<T> d((size_t)(2 * a.rows * ldp), h.stream);
    T *dg = d.get(), *du = d.get() + a.rows * ldp;
    {
        const bool wide = a.F % 8 == 0 && lddy % 8 == 0 && aligned_to(dy, 16) && aligned_to(gate, 16) &&
                          aligned_to(up, 16);
        const unsigned grid = (unsigned)std::min(ceil_div(a.rows * (ldp / 8), 256), (int64_t)sms * 8);
        with_activation(a.act, [&](auto act) {
            constexpr Activation A = decltype(act)::value;
            auto kern = wide ? gated_slopes_kernel<T, A, true> : gated_slopes_kernel<T, A, false>;
            launch_dependent(h.stream, kern, grid, 256, 0, 1, a.rows, a.F, dy, lddy, gate, up, dg, du, ldp);
        });
        after_launch(h, "gated_slopes");
    }
    if (dx) {
        const Operands<T> in(h, {{a.wg, a.ldwg, a.F, a.K}, {a.wu, a.ldwu, a.F, a.K}});
        TileArgs t = {};
        t.M = a.rows;
        t.N = a.K;
        const int cg = a.rows > TM ? 2 : 1;
        t.mt = (int)ceil_div(a.rows, TM * cg);
        t.kseg = (int)ceil_div(a.F, TK);
        t.ksteps = 2 * t.kseg;
        t.cols_first = a.rows > a.K;
        if (cg == 2) choose_tiles<Product::Dx, 2>(h, t);
        else choose_tiles<Product::Dx, 1>(h, t);
        t.a[0] = map_of<T>(dg, ldp, a.rows, a.F, TM);
        t.a[1] = map_of<T>(du, ldp, a.rows, a.F, TM);
        t.b[0] = in.map(0, TK);
        t.b[1] = in.map(1, TK);
        set_output(t, 0, dx, lddx);
        if (cg == 2) launch_product<T, Product::Dx, 2>(h, t);
        else launch_product<T, Product::Dx, 1>(h, t);
    }
    if (dwg) {
        const Operands<T> in(h, {{a.x, a.ldx, a.rows, a.K}});
        TileArgs t = {};
        t.M = a.F;
        t.N = a.K;
        t.mt = (int)ceil_div(a.F, TM);
        t.kseg = t.ksteps = (int)ceil_div(a.rows, TK);
        t.cols_first = 2 * a.F > a.K;
        choose_tiles<Product::Dw, 2>(h, t);
        t.a[0] = map_of<T>(dg, ldp, a.rows, a.F, TK);
        t.a[1] = map_of<T>(du, ldp, a.rows, a.F, TK);
        t.b[0] = in.map(0, TK);
        set_output(t, 0, dwg, a.K);
        set_output(t, 1, dwu, a.K);
        launch_product<T, Product::Dw, 2>(h, t);
    }
}

#define XS_INST_FFN(T)                                                                            \
    template void gated_ffn<T>(Handle&, const GatedArgs<T>&, T*, int64_t, T*, T*);                \
    template void gated_ffn_backward<T>(Handle&, const GatedArgs<T>&, const T*, int64_t, const T*, \
                                        const T*, T*, int64_t, T*, T*);
XS_INST_FFN(__half)
XS_INST_FFN(__nv_bfloat16)

}  // namespace xspmm_b200
