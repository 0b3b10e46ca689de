// qtts_kv4.hip — serving many sequences over a paged cache held in 4 bits:
//
//   k_kv4_tables       block tables, positions and slots of a step
//   k_qk_norm_rope     norms and rotation of q and k, k and v into the cache
//   k_kv4_gather       the values held at given slots
//   k_kv4_attn         attention over the pages, tiles of 16 columns: decode
//   k_kv4_attn_rows    the same, tiles of 128 columns: prompts
//   k_kv4_attn_join    partial results of tiles that were split
//
// Times are kernel times (rocprofv3) or, where they compare variants, of calls
// back to back.  On this card a large copy moves 4.74 TB/s and a large bf16
// matrix product reaches 1229 TFLOP/s.
//
// The layout of a page's block is in qtts_kv4.h.  A value is (code - 8) *
// scale with a scale of 8 significant bits, so it has at most 11 and is exact
// in f16: the matrix cores multiply what the cache stands for, not a rounding
// of it.

#include "qtts_kv4.h"
#include "../../include/qtts.h"
#include "qtts_devutil.h"
#include "qtts_mfma.h"

#include <algorithm>

namespace qtts {

// ---------------------------------------------------------------------------
// rows of f32, f16 or bf16
// ---------------------------------------------------------------------------

// four elements; vec: the address allows one load of them
template <class T>
__device__ __forceinline__ f32x4 load4(const T *p, bool vec)
{
    typedef T V __attribute__((ext_vector_type(4)));
    V v;
    if (vec) {
        v = *(const V *)p;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = p[i];
    }
    return __builtin_convertvector(v, f32x4);
}

template <class T>
__device__ __forceinline__ void store4(T *p, f32x4 x, bool vec)
{
    typedef T V __attribute__((ext_vector_type(4)));
    const V v = __builtin_convertvector(x, V);
    if (vec) {
        *(V *)p = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = v[i];
    }
}

// ---------------------------------------------------------------------------
// k_kv4_tables
// ---------------------------------------------------------------------------

// Every workgroup sums all sequences' rows and pages into LDS (8 bytes a
// sequence, from cache after the first) and then writes its own part of the
// rows and of the table: one launch, no workgroup waits for another.  All
// come to the same verdict on whether the step fits.  The entries that are
// read (a sequence's last partial page) are never the ones that are written.
// 8 sequences take 5.4 us, 64 with 515 rows 7.1: three waits for memory and four
// barriers one after the other, hardly any bytes.
__global__ void __launch_bounds__(1024)
k_kv4_tables(Kv4Tables a)
{
    __shared__ int32_t rs[KV4_MAX_SEQS + 1], ps[KV4_MAX_SEQS + 1];
    __shared__ int64_t wave_rows[16], wave_pages[16];
    __shared__ int32_t bad;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    constexpr int PER = KV4_MAX_SEQS / 1024;
    if (t == 0) bad = 0;
    __syncthreads();
    // thread t sums sequences PER t .. PER t + PER - 1
    int32_t n[PER], pg[PER];
    int64_t rows = 0, pages = 0;
    int worst = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int b = t * PER + i;
        n[i] = pg[i] = 0;
        if (b >= a.n_seqs) continue;
        const int64_t c = a.cached[b], f = a.fresh[b];
        if (c < 0 || f < 0) {
            worst = QTTS_ERR_INVALID;
            continue;
        }
        const int64_t total = (c + f + KV4_PAGE - 1) / KV4_PAGE;
        if (total > a.max_pages || f > a.n_rows) {
            worst = worst ? worst : QTTS_ERR_CAPACITY;
            continue;
        }
        n[i] = (int32_t)f;
        pg[i] = (int32_t)(total - (c + KV4_PAGE - 1) / KV4_PAGE);
        rows += n[i];
        pages += pg[i];
    }
    int64_t r = rows, p = pages;     // inclusive sums over the wave, then over the waves
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t r2 = __shfl_up(r, d), p2 = __shfl_up(p, d);
        if (lane >= d) r += r2, p += p2;
    }
    if (lane == 63) wave_rows[wave] = r, wave_pages[wave] = p;
    // one verdict for all: a negative length before a lack of room
    if (worst) atomicMin(&bad, worst == QTTS_ERR_INVALID ? -2 : -1);
    __syncthreads();
    int64_t all_rows = 0, all_pages = 0;
    r -= rows;
    p -= pages;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        if (w < wave) r += wave_rows[w], p += wave_pages[w];
        all_rows += wave_rows[w];
        all_pages += wave_pages[w];
    }
    const int status = bad == -2 ? QTTS_ERR_INVALID
                       : bad == -1 || all_rows > a.n_rows || all_pages > a.n_free ? QTTS_ERR_CAPACITY : QTTS_OK;
    const bool ok = status == QTTS_OK;
    if (!ok) all_rows = all_pages = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int b = t * PER + i;
        if (b < a.n_seqs) rs[b] = ok ? (int32_t)r : 0, ps[b] = ok ? (int32_t)p : 0;
        r += n[i];
        p += pg[i];
    }
    if (t == 0) rs[a.n_seqs] = (int32_t)all_rows, ps[a.n_seqs] = (int32_t)all_pages;
    __syncthreads();

    const int64_t first = (int64_t)blockIdx.x * 1024 + t, step = (int64_t)gridDim.x * 1024;
    for (int64_t b = first; b <= a.n_seqs; b += step) {
        a.row_start[b] = rs[b];
        if (b < a.n_seqs) a.lengths[b] = ok ? a.cached[b] + a.fresh[b] : 0;
    }
    if (first == 0) {
        a.status[0] = status;
        a.status[1] = (int32_t)all_pages;
    }
    // the last sequence whose sum is at most x: it holds element x
    const auto owner = [&](const int32_t *sum, int32_t x) {
        int lo = 0, hi = a.n_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sum[mid] <= x) lo = mid; else hi = mid;
        }
        return lo;
    };
    for (int64_t row = first; row < a.n_rows; row += step) {
        int32_t pos = -1;
        int64_t slot = -1;
        if (row < all_rows) {
            const int b = owner(rs, (int32_t)row);
            const int32_t c = a.cached[b], old = (c + KV4_PAGE - 1) / KV4_PAGE;
            pos = c + (int32_t)row - rs[b];
            const int32_t col = pos / KV4_PAGE;
            const int32_t page = col < old ? a.table[b * a.table_stride + col] : a.free_pages[ps[b] + col - old];
            slot = page < 0 ? -1 : (int64_t)page * KV4_PAGE + pos % KV4_PAGE;
        }
        a.positions[row] = pos;
        a.slots[row] = slot;
    }
    for (int64_t i = first; i < all_pages; i += step) {
        const int b = owner(ps, (int32_t)i);
        const int32_t old = (a.cached[b] + KV4_PAGE - 1) / KV4_PAGE;
        a.table[b * a.table_stride + old + i - ps[b]] = a.free_pages[i];
    }
}

hipError_t enqueue_kv4_tables(const Kv4Tables &a, hipStream_t s)
{
    const int64_t items = std::max<int64_t>(a.n_rows, a.n_seqs + 1);
    const int grid = (int)std::min<int64_t>((items + 1023) / 1024, 256);
    hipLaunchKernelGGL(k_kv4_tables, dim3(grid), dim3(1024), 0, s, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// k_qk_norm_rope
// ---------------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ double dpp_mov64(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// sums over L = 8 or 16 neighbouring lanes, the same in each
template <int L>
__device__ __forceinline__ float lanes_sum(float v)
{
    v += dpp_mov<0xB1>(v);
    v += dpp_mov<0x4E>(v);
    v += dpp_mov<0x141>(v);
    if constexpr (L == 16) v += dpp_mov<0x140>(v);
    return v;
}
template <int L>
__device__ __forceinline__ double lanes_sum(double v)
{
    v += dpp_mov64<0xB1>(v);
    v += dpp_mov64<0x4E>(v);
    v += dpp_mov64<0x141>(v);
    if constexpr (L == 16) v += dpp_mov64<0x140>(v);
    return v;
}

// 1 / sqrt(x): within an ulp in f32; in f64 from the instruction's 2^-28 or so by
// two steps of Newton's (each squares the error).
__device__ __forceinline__ float inv_sqrt(float x) { return __builtin_amdgcn_rsqf(x); }
__device__ __forceinline__ double inv_sqrt(double x)
{
    double r = __builtin_amdgcn_rsq(x);
    const double h = 0.5 * x;
    r = fma(r, fma(-h * r, r, 0.5), r);
    return fma(r, fma(-h * r, r, 0.5), r);
}

// One lane's part of a head: columns 4j .. 4j+3 and, D / 2 further, the ones
// they are rotated with.
template <class F>
struct Head {
    F a[4], b[4];
};

// The norm over the head's lanes and the rotation.  F float for rows that
// leave in their own type, double for keys that are quantised: a code is
// decided where a value lies between two borders, and sums in another order
// must not move it.
template <class F, int L>
__device__ __forceinline__ void norm_rope(Head<F> &x, bool norm, f32x4 ga, f32x4 gb, float eps, bool rope, f32x4 c, f32x4 s)
{
    if (norm) {
        F ss = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) ss = fma(x.a[i], x.a[i], fma(x.b[i], x.b[i], ss));
        ss = lanes_sum<L>(ss);
        const F r = inv_sqrt(ss * F(1.0 / (8 * L)) + (F)eps);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x.a[i] = x.a[i] * r * (F)ga[i];
            x.b[i] = x.b[i] * r * (F)gb[i];
        }
    }
    if (!rope) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const F a = x.a[i], b = x.b[i];
        x.a[i] = a * (F)c[i] - b * (F)s[i];
        x.b[i] = b * (F)c[i] + a * (F)s[i];
    }
}

// Codes and scale of 32 values, four in each of eight neighbouring lanes: the
// step is -1/8 of the value of largest magnitude, rounded to f16 and then to
// 8 significant bits; the nearest step's number, halves to even, plus 8.
//
// In f32 where that decides as f64 does: rounding to f32 keeps the order of
// values, so only two extremes that it makes equal have to be looked at again,
// and the quotient (at most 16, off by 2^-22 of it from x, the reciprocal and the
// product) only next to a half.  In f64 throughout, the kernel took 22.3 us for 4001
// rows of 16 heads instead of 17.2.
template <class F>
__device__ __forceinline__ uint32_t quantise(const F (&x)[4], uint16_t &scale)
{
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (float)x[i];
    float hi = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), lo = fminf(fminf(v[0], v[1]), fminf(v[2], v[3]));
    hi = fmaxf(hi, dpp_mov<0xB1>(hi)), lo = fminf(lo, dpp_mov<0xB1>(lo));
    hi = fmaxf(hi, dpp_mov<0x4E>(hi)), lo = fminf(lo, dpp_mov<0x4E>(lo));
    hi = fmaxf(hi, dpp_mov<0x141>(hi)), lo = fminf(lo, dpp_mov<0x141>(lo));
    // beyond the format's range a value's quotient goes past the last code, where it ends
    hi = fminf(hi, 65280.0f), lo = fmaxf(lo, -65280.0f);
    bool plus = hi >= -lo;
    if constexpr (std::is_same<F, double>::value)
        if (__any(hi == -lo && hi != 0.0f)) {
            double h = fmax(fmax(x[0], x[1]), fmax(x[2], x[3])), l = fmin(fmin(x[0], x[1]), fmin(x[2], x[3]));
            h = fmax(h, dpp_mov64<0xB1>(h)), l = fmin(l, dpp_mov64<0xB1>(l));
            h = fmax(h, dpp_mov64<0x4E>(h)), l = fmin(l, dpp_mov64<0x4E>(l));
            h = fmax(h, dpp_mov64<0x141>(h)), l = fmin(l, dpp_mov64<0x141>(l));
            plus = fmin(h, 65280.0) >= -fmax(l, -65280.0);
        }
    const _Float16 d16 = (_Float16)((plus ? hi : lo) * -0.125f);
    scale = (uint16_t)((__builtin_bit_cast(uint16_t, d16) + 4) & 0xFFF8);
    const float d = (float)__builtin_bit_cast(_Float16, scale);
    const float inv = d != 0.0f ? __builtin_amdgcn_rcpf(d) : 0.0f;
    float code[4], far = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float q = v[i] * inv, r = __builtin_rintf(q);
        far = fmaxf(far, fabsf(q - r));
        code[i] = __builtin_amdgcn_fmed3f(r + 8.0f, 0.0f, 15.0f);
    }
    if (far > 0.49999f) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // on which side of the half next to it x / d lies: h d has 13 bits, so the
            // difference has the right sign and is zero only at a tie
            const float q = v[i] * inv, r = __builtin_rintf(q), h = q < r ? r - 0.5f : r + 0.5f;
            const F e = fma((F)-h, (F)d, x[i]);
            const uint32_t up = __builtin_bit_cast(uint32_t, (float)e) ^ __builtin_bit_cast(uint32_t, d);    // its sign: e / d's
            const float near = h + __builtin_copysignf(0.5f, __builtin_bit_cast(float, up)), even = __builtin_rintf(h);
            const float n = e == 0 ? even : near;
            code[i] = __builtin_amdgcn_fmed3f(n + 8.0f, 0.0f, 15.0f);
        }
    }
    return (uint32_t)fmaf(4096.0f, code[3], fmaf(256.0f, code[2], fmaf(16.0f, code[1], code[0])));
}

// D / 8 lanes take one row's query heads of one kv head, that kv head's key
// and, with a cache, its value: the angles are loaded once for all of them.
// 4001 rows of 16 and 8 heads of 128, bf16, stored: 54 MB in 17.2 us, 3.1 TB/s; the
// 700 vector instructions of a wave (four keys in 64 bits, 16 groups quantised)
// take 12 us of the SIMDs' time, and all waves fit the card at once, so that they
// load first and compute then (13.7 us without the quantisation).  64 rows 5.3 us, one 4.5: the way of one wave.
// FAST: a wave's heads are of one row (the kv heads are a multiple of those
// that a wave holds), whose addresses are then scalar, and four elements move at
// once everywhere.
template <class T, int D, bool STORE, bool FAST>
__global__ void __launch_bounds__(256)
k_qk_norm_rope(QkNormRope a)
{
    constexpr int L = D / 8, HEADS = 64 / L;
    const int lane = threadIdx.x & 63, j = lane % L;
    const int first = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * HEADS;
    int row, hk;
    if constexpr (FAST) {
        row = __builtin_amdgcn_readfirstlane(first / a.kv_heads);
        hk = first - row * a.kv_heads + lane / L;
    } else {
        row = (first + lane / L) / a.kv_heads;
        hk = (first + lane / L) % a.kv_heads;
    }
    if (row >= a.rows) return;
    const bool vec = FAST || a.vec;
    const uint32_t at = hk * D + 4 * j, up = at + D / 2;     // a lane's columns of k and v
    const int32_t pos = a.positions ? a.positions[row] : 0;

    // the loads that wait for nothing first
    const T *kp = (const T *)a.k + row * a.k_stride;
    const f32x4 ka = load4(kp + at, vec), kb = load4(kp + up, vec);
    f32x4 va{}, vb{};
    int64_t slot = 0;
    if constexpr (STORE) {
        const T *vp = (const T *)a.v + row * a.v_stride;
        va = load4(vp + at, vec), vb = load4(vp + up, vec);
        slot = a.slots[row];
    }
    const T *qp = (const T *)a.q + row * a.q_stride;
    const uint32_t qat = hk * a.group * D + 4 * j;
    f32x4 qa = load4(qp + qat, vec), qb = load4(qp + (qat + D / 2), vec);
    if (pos < 0) return;
    f32x4 c{}, s{};
    if (a.positions) {
        if (pos < a.max_pos) {
            c = load4(a.cos + (int64_t)pos * (D / 2) + 4 * j, vec);
            s = load4(a.sin + (int64_t)pos * (D / 2) + 4 * j, vec);
        } else {
            c = s = __builtin_nanf("");
        }
    }

    f32x4 ga{}, gb{};
    if (a.q_norm) ga = load4((const _Float16 *)a.q_norm + 4 * j, vec), gb = load4((const _Float16 *)a.q_norm + D / 2 + 4 * j, vec);
    T *qo = (T *)a.q_out + row * a.q_out_stride;
    for (int g = 0; g < a.group; g++) {
        Head<float> x;
#pragma unroll
        for (int i = 0; i < 4; i++) x.a[i] = qa[i], x.b[i] = qb[i];
        const uint32_t here = qat + g * D;
        if (g + 1 < a.group) qa = load4(qp + (here + D), vec), qb = load4(qp + (here + D + D / 2), vec);
        norm_rope<float, L>(x, a.q_norm, ga, gb, a.eps, a.positions, c, s);
        store4(qo + here, f32x4{x.a[0], x.a[1], x.a[2], x.a[3]}, vec);
        store4(qo + (here + D / 2), f32x4{x.b[0], x.b[1], x.b[2], x.b[3]}, vec);
    }

    if (a.k_norm) ga = load4((const _Float16 *)a.k_norm + 4 * j, vec), gb = load4((const _Float16 *)a.k_norm + D / 2 + 4 * j, vec);
    using F = typename std::conditional<STORE, double, float>::type;
    Head<F> x;
#pragma unroll
    for (int i = 0; i < 4; i++) x.a[i] = ka[i], x.b[i] = kb[i];
    norm_rope<F, L>(x, a.k_norm, ga, gb, a.eps, a.positions, c, s);
    if (a.k_out) {
        T *ko = (T *)a.k_out + row * a.k_out_stride;
        store4(ko + at, f32x4{(float)x.a[0], (float)x.a[1], (float)x.a[2], (float)x.a[3]}, vec);
        store4(ko + up, f32x4{(float)x.b[0], (float)x.b[1], (float)x.b[2], (float)x.b[3]}, vec);
    }
    if constexpr (STORE) {
        bool nan = false;
        float y[4], z[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            nan |= x.a[i] != x.a[i] || x.b[i] != x.b[i] || va[i] != va[i] || vb[i] != vb[i];
            y[i] = va[i], z[i] = vb[i];
        }
        // any lane of the head
        const uint64_t lanes = ((1ull << L) - 1) << (lane / L * L);
        nan = (__ballot(nan) & lanes) != 0;
        uint16_t s0, s1, s2, s3;
        const uint32_t k0 = quantise(x.a, s0), k1 = quantise(x.b, s1);
        const uint32_t v0 = quantise(y, s2), v1 = quantise(z, s3);
        if (slot < 0 || slot >= a.cache.n_pages * KV4_PAGE) return;
        uint8_t *page = a.cache.base + slot / KV4_PAGE * a.cache.stride;
        const int p = (int)(slot % KV4_PAGE);
        const uint32_t blk = hk * kv4_block(D);
        *(uint16_t *)(page + (blk + kv4_k_at(D, p) + 2 * j)) = (uint16_t)k0;
        *(uint16_t *)(page + (blk + kv4_k_at(D, p) + D / 4 + 2 * j)) = (uint16_t)k1;
        *(uint16_t *)(page + (blk + kv4_v_at(D, p, j))) = (uint16_t)v0;
        *(uint16_t *)(page + (blk + kv4_v_at(D, p, j + D / 8))) = (uint16_t)v1;
        if (j % 8 == 0) {
            *(uint16_t *)(page + (blk + kv4_ks_at(D, p, j / 8))) = nan ? 0x7E00 : s0;
            *(uint16_t *)(page + (blk + kv4_ks_at(D, p, j / 8 + D / 64))) = nan ? 0x7E00 : s1;
            *(uint16_t *)(page + (blk + kv4_vs_at(D, p, j / 8))) = nan ? 0 : s2;
            *(uint16_t *)(page + (blk + kv4_vs_at(D, p, j / 8 + D / 64))) = nan ? 0 : s3;
        }
    }
}

template <class T, int D, bool FAST>
static void launch_qk_as(const QkNormRope &a, bool store, hipStream_t s)
{
    const int64_t heads = (int64_t)a.rows * a.kv_heads, per = 256 / (D / 8);
    const dim3 grid((unsigned)((heads + per - 1) / per));
    if (store)
        hipLaunchKernelGGL((k_qk_norm_rope<T, D, true, FAST>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((k_qk_norm_rope<T, D, false, FAST>), grid, dim3(256), 0, s, a);
}

template <class T, int D>
static hipError_t launch_qk(const QkNormRope &a, bool store, hipStream_t s)
{
    if (a.vec && a.kv_heads % (512 / D) == 0)
        launch_qk_as<T, D, true>(a, store, s);
    else
        launch_qk_as<T, D, false>(a, store, s);
    return hipGetLastError();
}

// F<T, D>::go for an element type and head width that the caller has checked
#define KV4_TYPED(dtype, D, call)                                            \
    do {                                                                     \
        if ((D) == 64) {                                                     \
            if ((dtype) == QTTS_F32) { using T = float; constexpr int HD = 64; return call; }      \
            if ((dtype) == QTTS_F16) { using T = _Float16; constexpr int HD = 64; return call; }   \
            using T = __bf16; constexpr int HD = 64; return call;            \
        }                                                                    \
        if ((dtype) == QTTS_F32) { using T = float; constexpr int HD = 128; return call; }         \
        if ((dtype) == QTTS_F16) { using T = _Float16; constexpr int HD = 128; return call; }      \
        using T = __bf16; constexpr int HD = 128; return call;               \
    } while (0)

hipError_t enqueue_qk_norm_rope(const QkNormRope &a, int dtype, int D, bool store, hipStream_t s)
{
    KV4_TYPED(dtype, D, (launch_qk<T, HD>(a, store, s)));
}

// ---------------------------------------------------------------------------
// k_kv4_gather
// ---------------------------------------------------------------------------

// Bound by the rows it writes: 4001 slots of 8 heads of 128 in f16, 37 MB, 7.0 us.
template <class T, int D>
__global__ void __launch_bounds__(256)
k_kv4_gather(Kv4Pages c, const int64_t *slots, int n, T *K, T *V)
{
    constexpr int L = D / 4;                     // lanes of a head, four columns each
    const int u = threadIdx.x % L;
    const int64_t item = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (item >= (int64_t)n * c.heads) return;
    const int i = (int)(item / c.heads), h = (int)(item % c.heads), g = u / 8;
    const int64_t slot = slots[i];
    uint32_t kc = 0x8888, vc = 0x8888;
    float ks = 0.0f, vs = 0.0f;
    if (slot >= 0 && slot < c.n_pages * KV4_PAGE) {
        const uint8_t *blk = c.base + slot / KV4_PAGE * c.stride + (int64_t)h * kv4_block(D);
        const int p = (int)(slot % KV4_PAGE);
        kc = *(const uint16_t *)(blk + kv4_k_at(D, p) + 2 * u);
        vc = *(const uint16_t *)(blk + kv4_v_at(D, p, u));
        ks = h2f(*(const uint16_t *)(blk + kv4_ks_at(D, p, g)));
        vs = h2f(*(const uint16_t *)(blk + kv4_vs_at(D, p, g)));
    }
    f32x4 k, v;
#pragma unroll
    for (int b = 0; b < 4; b++) {
        k[b] = (float)((int)(kc >> (4 * b) & 15) - 8) * ks;
        v[b] = (float)((int)(vc >> (4 * b) & 15) - 8) * vs;
    }
    const int64_t at = item * D + 4 * u;
    if (K) store4(K + at, k, true);
    if (V) store4(V + at, v, true);
}

template <class T, int D>
static hipError_t launch_gather(const Kv4Pages &c, const int64_t *slots, int n, void *K, void *V, hipStream_t s)
{
    const int64_t items = (int64_t)n * c.heads, per = 256 / (D / 4);
    hipLaunchKernelGGL((k_kv4_gather<T, D>), dim3((unsigned)((items + per - 1) / per)), dim3(256), 0, s, c, slots, n,
                       (T *)K, (T *)V);
    return hipGetLastError();
}

hipError_t enqueue_kv4_gather(const Kv4Pages &c, int D, const int64_t *slots, int n, int dtype, void *K, void *V, hipStream_t s)
{
    KV4_TYPED(dtype, D, (launch_gather<T, HD>(c, slots, n, K, V, s)));
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

__device__ __forceinline__ float max_xor32(float v)
{
    const unsigned u = __builtin_bit_cast(unsigned, v);
    unsigned w;
    asm volatile("" : "=v"(w) : "0"(u));
    const auto r = __builtin_amdgcn_permlane32_swap(u, w, false, false);
    unsigned a = r[0], b = r[1];
    asm volatile("" : "+v"(a), "+v"(b));
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

__device__ __forceinline__ float max_xor16(float v)
{
    const unsigned u = __builtin_bit_cast(unsigned, v);
    unsigned w;
    asm volatile("" : "=v"(w) : "0"(u));
    const auto r = __builtin_amdgcn_permlane16_swap(u, w, false, false);
    unsigned a = r[0], b = r[1];
    asm volatile("" : "+v"(a), "+v"(b));
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

__device__ __forceinline__ float add_xor16(float v)
{
    const unsigned u = __builtin_bit_cast(unsigned, v);
    unsigned w;
    asm volatile("" : "=v"(w) : "0"(u));
    const auto r = __builtin_amdgcn_permlane16_swap(u, w, false, false);
    return swap_pair_sum(r[0], r[1]);
}

__device__ __forceinline__ h16x2 as_h2(uint32_t u) { return __builtin_bit_cast(h16x2, u); }
__device__ __forceinline__ uint32_t as_u(h16x2 h) { return __builtin_bit_cast(uint32_t, h); }

// Masks and exponents of unpack8 where one v_and_or_b32 can take both: a
// VALU instruction reads one scalar register and no literal beside it, so the
// masks are kept in scalar registers and the exponent in a vector register
// (as constants they cost an and and an or: 128 instructions more, of 520 a page).
struct Unpack {
    uint32_t low = 0x000F000Fu, high = 0x00F000F0u, one = 0x64006400u;
    __device__ __forceinline__ Unpack() { asm volatile("" : "+s"(low), "+s"(high), "+v"(one)); }
};

// Eight codes (four bits at 0, 4, 8 and 12 of each half of w) times scales, as
// f16 pairs: out[n] = (code n of the low half, code n of the high half).  A
// code under 0x6400 is the f16 1024 + code, four bits further up 1024 + 16
// code; the subtraction, the factor 1/16 and the product with a scale of 8
// significant bits are all exact.
__device__ __forceinline__ void unpack8(const Unpack &u, uint32_t w, const h16x2 scale, uint32_t (&out)[4])
{
    const h16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const h16x2 m0 = {(_Float16)-1032.0f, (_Float16)-1032.0f}, m1 = {(_Float16)-72.0f, (_Float16)-72.0f};
    const uint32_t w8 = w >> 8;
    const h16x2 c0 = as_h2((w & u.low) | u.one) + m0;
    const h16x2 c1 = __builtin_elementwise_fma(as_h2((w & u.high) | u.one), sixteenth, m1);
    const h16x2 c2 = as_h2((w8 & u.low) | u.one) + m0;
    const h16x2 c3 = __builtin_elementwise_fma(as_h2((w8 & u.high) | u.one), sixteenth, m1);
    out[0] = as_u(c0 * scale);
    out[1] = as_u(c1 * scale);
    out[2] = as_u(c2 * scale);
    out[3] = as_u(c3 * scale);
}

__device__ __forceinline__ half8 as_half8(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __builtin_bit_cast(half8, u32x4{a, b, c, d});
}

// What a tile of W columns is: its sequence's rows r0 .. r0 + n - 1 at the end
// of `len` positions, its first column cb of n * group.
struct AttnTile {
    int b, r0, n, len, cb, ncols;
};

// Sums over lanes 0 .. l of the wave, in each lane l.
__device__ __forceinline__ int wave_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8: sums over rows of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast 15: the row before, to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast 31: the first half, to the second
    return v;
}

// Workgroups a round: about as many as the card has CUs.
constexpr int ROUND = 256;

// Tiles in descending order of their pages, `all` of them of which the card
// takes `round` at once: the place that number i has among them.  Where there
// are no more than two rounds, a CU gets a second tile while it still has its
// first, the smaller ones beside the larger: the first round begins with those
// that are to share a CU, and the second goes upwards.
__device__ __forceinline__ int tile_place(int i, int all, int round)
{
    if (all <= round || all > 2 * round) return i;
    const int shared = all - round;
    return i >= round ? all - 1 - (i - round) : i < shared ? round - shared + i : i - shared;
}

// The tile with number ti, found by the whole wave: first its block of 64
// sequences (each round, 64 lanes look at 64 evenly spaced ones), then the
// sequence by a sum over the block's.  One load of latency for 64 sequences,
// two for 4096.  False where no tile has this number, and for row sums that
// are none.
//
// Where there are more workgroups than CUs, a block's tiles are numbered by
// the pages that they see, the most first: a lane counts its sequence's tiles
// of p pages or more (a sequence's later tiles see more), and p is found by
// bisection, in 1 us.  64 sequences of 1365 to 4096 positions in no order take
// 37 us, numbered in the order of the sequences 46 (of 667 to 2000 24 / 27, 256 of
// 1365 to 4096 158 / 162); four prompts of 500 to 1000 rows on 667 to 2000 60 / 69.
// Not for tiles of fewer pages (256 sequences of up to 500 positions 35 / 33) and
// not where they are cut into parts of less than 64 pages, which are even already
// (48 sequences of up to 4096 40 / 38).
__device__ __forceinline__ bool find_tile(const Kv4Attn &a, int ti, int W, AttnTile &t)
{
    const int lane = threadIdx.x & 63;
    const auto start = [&](int b) { return min(max(a.row_start[b], 0), a.rows); };
    int lo = 0, cnt = (a.n_seqs + 63) / 64;
    while (cnt > 1) {
        const int step = (cnt + 63) / 64, i = lane * step;
        const bool in = i < cnt && kv4_first_tile(start(64 * (lo + i)), a.group, 64 * (lo + i), W) <= ti;
        const uint64_t m = __ballot(in);
        const int last = m ? 63 - __clzll(m) : 0;
        lo += last * step;
        cnt = min(step, cnt - last * step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo) * 64;
    // what a lane's sequence is comes with the same wait as its rows
    const int b = min(lo + lane, a.n_seqs), r0 = a.row_start[b], r1 = a.row_start[min(b + 1, a.n_seqs)];
    const int len = a.lengths[min(b, a.n_seqs - 1)];
    const int s0 = min(max(r0, 0), a.rows), s1 = min(max(r1, 0), a.rows), n = max(s1 - s0, 0);
    const int tiles = (n * a.group + W - 1) / W;
    int rel = ti - (int)kv4_first_tile(__builtin_amdgcn_readlane(s0, 0), a.group, lo, W);
    int end = wave_scan(tiles), first = end - tiles, skip = 0;
    const int all = __builtin_amdgcn_readlane(end, 63);
    if (rel < 0 || rel >= all) return false;
    const int seen = min(max(len, 0), INT32_MAX - KV4_PAGE);
    // more pages than any tile sees: a length rounded to f32 is off by a page at most
    const int bound = min((int)wave_max_dpp(n ? (float)seen : 0.0f) / KV4_PAGE + 4, a.max_pages + 1);
    if (all * a.cache.heads > ROUND && a.chunk >= 64 && bound > (W == KV4_W ? 20 : 8)) {
        rel = tile_place(rel, all, max(ROUND / a.cache.heads, 1));
        // tiles of p + 1 pages or more: those of the rows that see position 64 p
        const auto count = [&](int p) {
            const int at = p * KV4_PAGE, row = max(at - (seen - n), 0);
            return at >= seen ? 0 : tiles - (int)((uint32_t)(row * a.group) / (uint32_t)W);
        };
        int p = 0, more = bound;
        while (more - p > 1) {
            const int mid = (p + more) / 2;
            if (__builtin_amdgcn_readlane(wave_scan(count(mid - 1)), 63) > rel) p = mid; else more = mid;
        }
        // those of p pages: of each sequence the tiles before the `skip` last
        skip = more > a.max_pages ? 0 : count(more - 1);
        rel -= __builtin_amdgcn_readlane(wave_scan(skip), 63);
        const int here = (p ? count(p - 1) : tiles) - skip;
        end = wave_scan(here), first = end - here;
    }
    const uint64_t m = __ballot(rel >= first && rel < end);
    if (!m) return false;
    const int at = __ffsll((unsigned long long)m) - 1;
    t.b = lo + at;
    t.r0 = __builtin_amdgcn_readlane(r0, at);
    const int last = __builtin_amdgcn_readlane(r1, at);
    t.len = __builtin_amdgcn_readlane(len, at);
    if (t.r0 < 0 || last > a.rows || last <= t.r0 || t.len < 0 || t.len > INT32_MAX - KV4_PAGE) return false;
    t.n = last - t.r0;
    t.ncols = t.n * a.group;
    // from the last of a sequence's tiles to its first
    const int j = __builtin_amdgcn_readlane(tiles - 1 - skip, at) - (rel - __builtin_amdgcn_readlane(first, at));
    t.cb = j * W;
    return t.cb < t.ncols;
}

// The last position that a column sees is len - n + row; minpos and maxpos are
// the first and last column's, and pages pg0 .. pg0 + pages - 1 hold all that
// the tile's columns see (as far as the table has columns).
__device__ __forceinline__ void tile_pages(const Kv4Attn &a, const AttnTile &t, int W, int &minpos, int &maxpos, int &pg0,
                                           int &pages)
{
    minpos = t.len - t.n + t.cb / a.group;
    maxpos = t.len - t.n + min(t.cb + W - 1, t.ncols - 1) / a.group;
    const int lo = a.window ? max(0, minpos - a.window + 1) : 0;
    pg0 = lo / KV4_PAGE;
    pages = maxpos < lo ? 0 : max(min(maxpos / KV4_PAGE + 1, a.max_pages) - pg0, 0);
}

// Workgroups that share a tile of so many pages: `chunk` pages each, the last
// of `splits` what is left.  The sequence's own length says how many, so that
// a long one among short ones is not one workgroup's work.
__device__ __forceinline__ int tile_parts(int pages, int chunk, int splits)
{
    return max(1, min((pages + chunk - 1) / chunk, splits));
}

// Whether a position sees any key of a page.
__device__ __forceinline__ bool sees(int pos, int window, int page)
{
    const int first = page * KV4_PAGE;
    return pos >= first && (!window || pos - window < first + KV4_PAGE - 1);
}

// One page's block as a wave holds it: lane l = (r, kg) = (l % 16, l / 16) has
// of K rows 4r + t (t = 0..3) the D / 4 columns from kg D / 4, of V positions
// 16 kg .. 16 kg + 15 of the D / 16 columns from r D / 16, and their scales.
template <int D>
struct PageK {
    uint32_t k[4][D / 32], s[2];
};
template <int D>
struct PageV {
    uint32_t v[4][D / 32], s[8];
};

// Where a lane's parts lie in a block, apart from what is the same for all
// lanes: 32 bits beside a scalar address, one register each.
template <int D>
struct LaneAt {
    uint32_t k, ks, v, vs;
    __device__ __forceinline__ LaneAt(int r, int kg)
    {
        k = kv4_k_at(D, 4 * r) + kg * (D / 8);
        ks = kv4_ks_at(D, 4 * r, kg * (D / 4) / 32);
        v = kv4_v_at(D, 16 * kg, r * (D / 64));
        vs = kv4_vs_at(D, 16 * kg, r * (D / 16) / 32);
    }
};

template <int D>
__device__ __forceinline__ void load_words(uint32_t *out, const uint8_t *p)
{
    if constexpr (D == 128) {
        const u32x4 w = *(const u32x4 *)p;
        out[0] = w.x, out[1] = w.y, out[2] = w.z, out[3] = w.w;
    } else {
        const uint2 w = *(const uint2 *)p;
        out[0] = w.x, out[1] = w.y;
    }
}

template <int D>
__device__ __forceinline__ void load_page(PageK<D> &g, const uint8_t *blk, const LaneAt<D> &at)
{
#pragma unroll
    for (int t = 0; t < 4; t++) load_words<D>(g.k[t], blk + t * (kv4_k_at(D, 1) - kv4_k_at(D, 0)) + at.k);
    const uint2 s = *(const uint2 *)(blk + at.ks);
    g.s[0] = s.x, g.s[1] = s.y;
}

template <int D>
__device__ __forceinline__ void load_page(PageV<D> &g, const uint8_t *blk, const LaneAt<D> &at)
{
#pragma unroll
    for (int q = 0; q < 4; q++) load_words<D>(g.v[q], blk + q * (kv4_v_at(D, 4, 0) - kv4_v_at(D, 0, 0)) + at.v);
    const u32x4 *s = (const u32x4 *)(blk + at.vs);
    const u32x4 s0 = s[0], s1 = s[1];
    g.s[0] = s0.x, g.s[1] = s0.y, g.s[2] = s0.z, g.s[3] = s0.w;
    g.s[4] = s1.x, g.s[5] = s1.y, g.s[6] = s1.z, g.s[7] = s1.w;
}

// A column's query as the second operand of K q: its D / 4 values from kg D /
// 4, eight to a step in the order in which unpack8 leaves K's.  Values are
// first scaled by the power of two that puts the row's largest near 2^14
// (undone in `unit`): a bf16 or f32 row of any range fits f16; f32 keeps 22
// bits in two parts.
template <class T, int D>
struct Query {
    static constexpr int PARTS = std::is_same<T, float>::value ? 2 : 1;
    half8 f[PARTS][D / 32];
};

template <class T, int D>
__device__ __forceinline__ float load_query(Query<T, D> &q, const T *p, bool valid, bool vec)
{
    f32x4 x[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; i++) x[i] = valid ? load4(p + 4 * i, vec) : f32x4{0, 0, 0, 0};
    float unit = 1.0f;
    if constexpr (!std::is_same<T, _Float16>::value) {
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(x[i][e]));
        mx = max_xor32(max_xor16(mx));
        const int sh = range_shift(mx);
        const float up = ldexpf(1.0f, sh);
        unit = ldexpf(1.0f, -sh);
#pragma unroll
        for (int i = 0; i < D / 16; i++) x[i] *= up;
    }
#pragma unroll
    for (int j = 0; j < D / 32; j++) {
        const f32x4 lo = x[2 * j], hi = x[2 * j + 1];
        uint32_t h[4], l[4];
#pragma unroll
        for (int n = 0; n < 4; n++) split_f16_pair<true>(lo[n], hi[n], h[n], l[n]);
        q.f[0][j] = as_half8(h[0], h[1], h[2], h[3]);
        if constexpr (Query<T, D>::PARTS == 2) q.f[1][j] = as_half8(l[0], l[1], l[2], l[3]);
    }
    return unit;
}

// Column cc of a tile: its query, its position (-1: there is no such column)
// and the factor from products to log2 units.
template <class T, int D>
__device__ __forceinline__ float load_column(Query<T, D> &q, const Kv4Attn &a, const AttnTile &t, int hk, int cc, int kg, int &pos)
{
    const int row = cc / a.group;
    const bool valid = cc < t.ncols;
    pos = valid ? t.len - t.n + row : -1;
    const T *qp = (const T *)a.q + (t.r0 + row) * a.q_stride + (hk * a.group + cc % a.group) * D + kg * (D / 4);
    float unit = load_query<T, D>(q, qp, valid, a.vec) * (a.scale * 1.44269504088896341f);
    if (a.scale < 0.0f) {            // the running maximum is taken before the factor
        unit = -unit;
#pragma unroll
        for (int i = 0; i < Query<T, D>::PARTS; i++)
#pragma unroll
            for (int j = 0; j < D / 32; j++) q.f[i][j] = -q.f[i][j];
    }
    return fmaxf(unit, 1.2e-38f);    // 0 * -inf would be NaN
}

// Running state of 16 columns in a wave: lane (m, kg) holds column m's reference
// (in units of log2), its own share of the sum, and rows D/16 (4 kg + e) + i of
// the output as o[i][e].  The reference is a score that was the largest when
// it was taken.  A probability is kept times 2^TOP over the reference's, where
// f16 holds the small ones too, and the reference moves (sum and output are
// scaled) only when one would pass 2^15: most pages neither exchange maxima
// between lanes nor touch the output.  16-bit rows, whose probabilities are
// rounded to f16's 11 bits anyway, leave more room for that than f32 rows.
// Sums and outputs carry the factor until they are divided.
template <int D>
struct Running {
    float m = -INFINITY, l = 0.0f;
    f32x4 o[D / 16] = {};
};
template <class T>
constexpr float TOP = std::is_same<T, float>::value ? 14.0f : 9.0f;

// Scores of one page's 64 keys: lane (m, kg) gets column m's of keys 16 kg + 4 i
// + t as x[t][i].
template <class T, int D>
__device__ __forceinline__ void page_scores(f32x4 (&x)[4], const Unpack &un, const PageK<D> &g, const Query<T, D> &q)
{
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint32_t sc = g.s[t / 2];
        const uint32_t both = t % 2 ? (sc >> 16) | (sc & 0xFFFF0000u) : (sc & 0xFFFFu) | (sc << 16);
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            uint32_t a[4];
            unpack8(un, g.k[t][j], as_h2(both), a);
            const half8 k8 = as_half8(a[0], a[1], a[2], a[3]);
            if constexpr (Query<T, D>::PARTS == 2) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, q.f[1][j], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, q.f[0][j], acc, 0, 0, 0);
        }
        x[t] = acc;
    }
}

// Keys that a column does not see.
__device__ __forceinline__ void mask_scores(f32x4 (&x)[4], int key0, int pos, int window, int kg)
{
    const int first = key0 + 16 * kg;
    const int low = window ? pos - window : -1;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int key = first + 4 * i + t;
            if (key > pos || key <= low) x[t][i] = -INFINITY;
        }
}

// Scales of the values at positions first, first + 1, .. (two to a word), zero
// past the sequence's end: what is there may be anything, and 0 * NaN is not 0.
template <int N>
__device__ __forceinline__ void mask_values(uint32_t (&scales)[N], int first, int len)
{
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int left = len - (first + 2 * i);
        scales[i] = left <= 0 ? 0u : left == 1 ? scales[i] & 0xFFFFu : scales[i];
    }
}

// The running softmax over a page's scores, NC sets of 16 columns: probabilities
// of keys 16 kg + 4 i + t at 4 i + t, in f16 pairs, of two parts for f32 rows.
template <class T, int D, int NC>
__device__ __forceinline__ void page_softmax(Running<D> (&s)[NC], f32x4 (&x)[NC][4], const float (&unit)[NC],
                                             half8 (&p8)[NC][Query<T, D>::PARTS][2])
{
    float off[NC], top[NC];
    bool move = false;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        off[c] = s[c].m == -INFINITY ? 0.0f : TOP<T> - s[c].m;
        top[c] = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[c][t][i] = fmaf(x[c][t][i], unit[c], off[c]);      // the exponent
                top[c] = fmaxf(top[c], x[c][t][i]);
            }
        move |= top[c] > (s[c].m == -INFINITY ? -INFINITY : 15.0f);
    }
    if (__any(move)) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const float m = fmaxf(s[c].m, max_xor32(max_xor16(top[c])) - off[c]);
            const float f = m > s[c].m ? __builtin_amdgcn_exp2f(s[c].m - m) : 1.0f;   // exp2(-inf) = 0 at the first page
            const float by = m == -INFINITY ? 0.0f : TOP<T> - m - off[c];
            s[c].l *= f;
            s[c].m = m;
#pragma unroll
            for (int i = 0; i < D / 16; i++) s[c].o[i] *= f;
#pragma unroll
            for (int t = 0; t < 4; t++) x[c][t] += by;
        }
    }
#pragma unroll
    for (int c = 0; c < NC; c++) {
        float p[16], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            p[i] = __builtin_amdgcn_exp2f(x[c][i % 4][i / 4]);
            sum += p[i];
        }
        s[c].l += sum;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float p0 = p[8 * u + 2 * n], p1 = p[8 * u + 2 * n + 1];
                if constexpr (Query<T, D>::PARTS == 2)
                    split_f16_pair<true>(p0, p1, ph[n], pl[n]);
                else
                    ph[n] = as_u(h16x2{(_Float16)p0, (_Float16)p1});
            }
            p8[c][0][u] = as_half8(ph[0], ph[1], ph[2], ph[3]);
            if constexpr (Query<T, D>::PARTS == 2) p8[c][1][u] = as_half8(pl[0], pl[1], pl[2], pl[3]);
        }
    }
}

// o += V p over 32 keys, the small part first.
template <int PARTS>
__device__ __forceinline__ void add_values(f32x4 &o, half8 v8, const half8 (&p8)[PARTS][2], int u)
{
    if constexpr (PARTS == 2) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, p8[1][u], o, 0, 0, 0);
    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, p8[0][u], o, 0, 0, 0);
}

// P V on the lanes that hold the scores: nothing goes from lane to lane but
// the maximum.
template <class T, int D>
__device__ __forceinline__ void page_values(Running<D> (&s)[1], const Unpack &un, f32x4 (&x)[1][4], const PageV<D> &g,
                                            const float (&unit)[1])
{
    half8 p8[1][Query<T, D>::PARTS][2];
    page_softmax<T, D, 1>(s, x, unit, p8);
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int c = 0; c < D / 64; c++) {       // units of four columns
            uint32_t a[4][4];
#pragma unroll
            for (int h = 0; h < 4; h++) unpack8(un, g.v[2 * u + h / 2][2 * c + h % 2], as_h2(g.s[4 * u + h]), a[h]);
#pragma unroll
            for (int n = 0; n < 4; n++) add_values(s[0].o[4 * c + n], as_half8(a[0][n], a[1][n], a[2][n], a[3][n]), p8[0], u);
        }
}

// Attention of 16 columns of one kv head over a share of the tile's pages, the
// waves taking them in turn and joining through LDS.  64 sequences of 1365 to
// 4096 positions, 8 kv heads of 128: 200 MB in 45 us, 4.4 TB/s, nine tenths of a
// copy; a page costs a wave about 520 vector instructions (four fifths of them
// unpack codes) and 32 products, nearly as long for a SIMD as its bytes take to come.  One sequence of 300 positions 8.6 us: tile, query, table entry and
// page are waited for one after the other.
//
// Eight waves where there are no more workgroups than CUs: half the pages one
// after the other.  28 sequences of 3000 positions 22 us, with four waves in three
// parts 29; where there are more, two workgroups of four waves share a CU
// better (64 of 1365 to 4096 positions 36 us, eight waves 46).  f32 queries of 128
// need 185 registers: two waves a SIMD without spills, not three with 28 (64
// sequences of 4096, f32, 40 us and 60).
template <class T, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, WAVES == 8 || (std::is_same<T, float>::value && D == 128) ? 2 : 3)
k_kv4_attn(Kv4Attn a)
{
    constexpr int W = KV4_W, LD = D + 4;
    __shared__ float so[WAVES][W][LD], sm[WAVES][W], sl[WAVES][W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, kg = lane >> 4;
    const int ti = blockIdx.x / a.cache.heads, hk = blockIdx.x % a.cache.heads, sp = blockIdx.y;
    AttnTile t;
    if (!find_tile(a, ti, W, t)) return;
    int minpos, maxpos, pg0, pages;
    tile_pages(a, t, W, minpos, maxpos, pg0, pages);
    const int parts = tile_parts(pages, a.chunk, a.splits);
    if (sp >= parts) return;
    const int pb = pg0 + sp * a.chunk, pe = sp == parts - 1 ? pg0 + pages : pb + a.chunk;

    Query<T, D> q;
    int pos;
    const float unit[1] = {load_column<T, D>(q, a, t, hk, t.cb + r, kg, pos)};
    Running<D> run[1];
    bool poisoned = pos >= (int64_t)a.max_pages * KV4_PAGE;   // sees a page that the table has no column for
    const int32_t *table = a.table + (int64_t)t.b * a.table_stride;
    const Unpack un;
    const LaneAt<D> at(r, kg);
    const int n = (pe - pb - wave + WAVES - 1) / WAVES;      // this wave's pages: pb + wave + WAVES i
    int ids = 0;                                 // of 64 of them, one a lane
    const uint8_t *blk = nullptr;
    int held = 0;                                // positions whose values count
    const auto find = [&](int i) {
        const int page = pb + wave + WAVES * i;
        if ((i & 63) == 0) ids = page + WAVES * lane < pe ? table[page + WAVES * lane] : -1;
        int id = __builtin_amdgcn_readlane(ids, i & 63);
        held = t.len;
        if (id < 0 || id >= a.cache.n_pages) {   // what sees this page is NaN, and for the others its values are zero
            id = held = 0;
            poisoned |= sees(pos, a.window, page);
        }
        blk = a.cache.base + id * a.cache.stride + (int64_t)hk * kv4_block(D);
    };
    // V is on its way while K is multiplied, the next page's K while V is
    PageK<D> gk;
    if (n > 0) {
        find(0);
        load_page(gk, blk, at);
    }
    for (int i = 0; i < n; i++) {
        PageV<D> gv;
        load_page(gv, blk, at);
        const int key0 = (pb + wave + WAVES * i) * KV4_PAGE, count = held;
        f32x4 x[1][4];
        __builtin_amdgcn_sched_barrier(0);
        page_scores<T, D>(x[0], un, gk, q);
        __builtin_amdgcn_sched_barrier(0);
        if (i + 1 < n) {
            find(i + 1);
            load_page(gk, blk, at);
        }
        if (key0 + KV4_PAGE - 1 > minpos || (a.window && key0 <= maxpos - a.window)) mask_scores(x[0], key0, pos, a.window, kg);
        if (key0 + KV4_PAGE > count) mask_values(gv.s, key0 + 16 * kg, count);
        page_values<T, D>(run, un, x, gv, unit);
    }
    Running<D> &s = run[0];
    s.l = add_xor32(add_xor16(s.l));
    if (poisoned) s.l = __builtin_nanf("");
    if (kg == 0) sm[wave][r] = s.m, sl[wave][r] = s.l;
    __syncthreads();
    const auto largest = [&](int c) {
        float m = sm[0][c];
#pragma unroll
        for (int w = 1; w < WAVES; w++) m = fmaxf(m, sm[w][c]);
        return m;
    };
    const float M = largest(r);
    const float f = s.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s.m - M);
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
        for (int i = 0; i < D / 16; i += 4)
            *(f32x4 *)&so[wave][r][D / 16 * (4 * kg + e) + i] =
                f32x4{s.o[i][e], s.o[i + 1][e], s.o[i + 2][e], s.o[i + 3][e]} * f;
    __syncthreads();
    const int64_t pi = ((int64_t)ti * a.cache.heads + hk) * a.splits + sp;
    for (int e = threadIdx.x; e < W * D / 4; e += 64 * WAVES) {
        const int c = e / (D / 4), d = e % (D / 4) * 4, col = t.cb + c;
        if (col >= t.ncols) break;
        f32x4 o = {0, 0, 0, 0};
        float l = 0.0f;
        const float Mc = largest(c);
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            o += *(const f32x4 *)&so[w][c][d];
            l += sm[w][c] == -INFINITY ? 0.0f * sl[w][c] : sl[w][c] * __builtin_amdgcn_exp2f(sm[w][c] - Mc);
        }
        if (parts > 1) {
            if (d == 0) a.part[pi * 2 * W + c] = Mc, a.part[(pi * 2 + 1) * W + c] = l;
            *(f32x4 *)(a.part + a.part_rows + (pi * W + c) * D + d) = o;
        } else {
            // a column that saw nothing has l = 0
            store4((T *)a.out + (t.r0 + col / a.group) * a.out_stride + (hk * a.group + col % a.group) * D + d,
                   l == 0.0f ? f32x4{0, 0, 0, 0} : o / l, a.vec);
        }
    }
}

// A page of a prompt's tile as a thread loads it, each code of it unpacked once
// for four waves.  Each takes one K tile (rows 4r + share) and of V, with D = 128,
// eight positions (16 kg + 8 (share / 2) ..) of half the columns, which are whole
// 16 bytes of four fragments (as halves of eight, their writes met in LDS banks: one
// prompt of 4000 positions 108 us, now 106); with D = 64 four positions of all
// columns, halves of four fragments.
template <int D>
struct PageShare {
    uint32_t k[D / 32], v[D / 32], vs[D / 32];
    uint16_t ks;
    int held;                        // positions whose values count
};

constexpr int DS_STAYS = 0x47F;      // sched_barrier: all but LDS instructions may pass

// Attention of 128 columns of one kv head, two sets of 16 a wave: the prompt
// path.  A page is unpacked to f16 once for four waves and laid in LDS in the
// order in which the matrix instructions read it (1 KiB a fragment, each lane
// its 16 bytes), one page ahead of the products; two sets a wave halve the LDS
// reads of a product.  Matrix and other vector instructions of a SIMD hardly
// overlap here (48 of 4.4 cycles and four of 16.6 take their sum, from one wave or
// from two), so a page costs what its 425 vector instructions and 64 products a
// wave add up to, 3000 cycles, and a fifth more for waits.  Four prompts of 500
// to 1000 rows, 29.6 GFLOP: 59 us, 500 TFLOP/s; the longest tile's 32 pages, one
// after the other, are 50 of them.
//
// HALVES 2, for no more tiles than CUs: eight waves, the second four taking every
// other page, joined at the end.  The longest tile's way is half as long, and
// each SIMD has two waves to take turns.  2048 positions, sequences of 64 rows, in
// us with four waves / eight: 16 sequences (128 tiles) 65 / 51, 32 70 / 59, 64 104 /
// 114, and four prompts of 500 to 1000 rows (376 tiles) 79 / 84 (61 with the
// tiles in order): there two workgroups of four share a CU.
template <class T, int D, int HALVES>
__global__ void __launch_bounds__(256 * HALVES, 2)
k_kv4_attn_rows(Kv4Attn a)
{
    constexpr int W = KV4_WIDE, NC = 2, KF = D / 8, VF = D / 8;  // fragments of a page: 4 x D/32 and 2 x D/16
    constexpr int PARTS = Query<T, D>::PARTS, LD = D + 4;
    static_assert(W == 4 * NC * 16, "four waves' columns");
    // pages while they are multiplied: [half][buffer][K, then V fragments]; then the second half's result
    __shared__ union {
        u32x4 page[HALVES][2][KF + VF][64];
        struct { float o[HALVES == 2 ? W : 1][LD], m[W], l[W]; } half;
    } lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, kg = lane >> 4, share = wave & 3, half = HALVES == 2 ? wave >> 2 : 0;
    const int ti = blockIdx.x / a.cache.heads, hk = blockIdx.x % a.cache.heads, sp = blockIdx.y;
    AttnTile t;
    if (!find_tile(a, ti, W, t)) return;
    int minpos, maxpos, pg0, pages;
    tile_pages(a, t, W, minpos, maxpos, pg0, pages);
    const int parts = tile_parts(pages, a.chunk, a.splits);
    if (sp >= parts) return;
    const int pb = pg0 + sp * a.chunk, pe = sp == parts - 1 ? pg0 + pages : pb + a.chunk;

    Query<T, D> q[NC];
    int pos[NC], low[NC], high[NC];  // low, high: the first and last position of 16 columns
    float unit[NC];
    Running<D> s[NC];
    bool poisoned[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int first = t.cb + (share * NC + c) * 16;
        unit[c] = load_column<T, D>(q[c], a, t, hk, first + r, kg, pos[c]);
        low[c] = t.len - t.n + first / a.group;
        high[c] = first < t.ncols ? t.len - t.n + min(first + 15, t.ncols - 1) / a.group : -1;
        poisoned[c] = pos[c] >= (int64_t)a.max_pages * KV4_PAGE;
    }
    const int32_t *table = a.table + (int64_t)t.b * a.table_stride;
    const Unpack un;
    const LaneAt<D> at(r, kg);
    int ids = 0;                     // of 64 pages, one a lane
    const auto fetch = [&](PageShare<D> &g, int it) {
        const int page = pb + HALVES * it + half;
        if ((it & 63) == 0) ids = page + HALVES * lane < pe ? table[page + HALVES * lane] : -1;
        int id = __builtin_amdgcn_readlane(ids, it & 63);
        g.held = t.len;
        if (id < 0 || id >= a.cache.n_pages) {   // what sees this page is NaN, and for the others its values are zero
            id = 0;
            g.held = 0;
#pragma unroll
            for (int c = 0; c < NC; c++) poisoned[c] |= page < pe && sees(pos[c], a.window, page);
        }
        const uint8_t *blk = a.cache.base + id * a.cache.stride + (int64_t)hk * kv4_block(D);
        load_words<D>(g.k, blk + share * (kv4_k_at(D, 1) - kv4_k_at(D, 0)) + at.k);
        g.ks = *(const uint16_t *)(blk + share * 2 + at.ks);
        constexpr int block = kv4_v_at(D, 4, 0) - kv4_v_at(D, 0, 0);
        if constexpr (D == 128) {
            const uint8_t *v = blk + share / 2 * 2 * block + share % 2 * 8 + at.v;
            load_words<64>(g.v, v);
            load_words<64>(g.v + 2, v + block);
            load_words<128>(g.vs, blk + share / 2 * 16 + at.vs);
        } else {
            load_words<D>(g.v, blk + share * block + at.v);
            load_words<64>(g.vs, blk + share * 8 + at.vs);
        }
    };
    const auto stage = [&](PageShare<D> &g, int it) {
        const int key0 = (pb + HALVES * it + half) * KV4_PAGE;
        u32x4 (*const to)[64] = lds.page[half][it & 1];
        const h16x2 ks = as_h2((uint32_t)g.ks | (uint32_t)g.ks << 16);
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
            uint32_t k[4];
            unpack8(un, g.k[j], ks, k);
            to[share * (D / 32) + j][lane] = u32x4{k[0], k[1], k[2], k[3]};
        }
        const int first = key0 + 16 * kg + (D == 128 ? 8 * (share / 2) : 4 * share);
        if (key0 + KV4_PAGE > g.held) mask_values(g.vs, first, g.held);
        uint32_t v[D / 32][4];
#pragma unroll
        for (int h = 0; h < D / 32; h++) unpack8(un, g.v[h], as_h2(g.vs[h]), v[h]);
        u32x4 (*const tv)[64] = to + KF + share / 2 * (D / 16);
#pragma unroll
        for (int n = 0; n < 4; n++)
            if constexpr (D == 128)
                tv[4 * (share % 2) + n][lane] = u32x4{v[0][n], v[1][n], v[2][n], v[3][n]};
            else
                *((uint2 *)&tv[n][lane] + share % 2) = make_uint2(v[0][n], v[1][n]);
    };

    // a page too many for the second half is fetched as none and masked for every column
    const int rounds = (pe - pb + HALVES - 1) / HALVES;
    PageShare<D> g;
    if (rounds > 0) {
        fetch(g, 0);
        stage(g, 0);
    }
    __syncthreads();
    for (int it = 0; it < rounds; it++) {
        const int key0 = (pb + HALVES * it + half) * KV4_PAGE;
        const u32x4 (*const lk)[64] = lds.page[half][it & 1], (*const lv)[64] = lk + KF;
        if (it + 1 < rounds) fetch(g, it + 1);
        // fragments are read from LDS in pairs, two pairs ahead of the products; the
        // reads stay where they are written (otherwise each is waited for by itself)
        f32x4 x[NC][4];
        half8 f[3][2];
        const auto read = [&](half8 (&to)[2], const u32x4 (*from)[64], int n) {
            to[0] = __builtin_bit_cast(half8, from[2 * n][lane]);
            to[1] = __builtin_bit_cast(half8, from[2 * n + 1][lane]);
        };
        read(f[0], lk, 0);
        read(f[1], lk, 1);
#pragma unroll
        for (int n = 0; n < KF / 2; n++) {
            if (n < KF / 2 - 2) read(f[(n + 2) % 3], lk, n + 2);
            __builtin_amdgcn_sched_barrier(DS_STAYS);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k = (2 * n + h) / (D / 32), j = (2 * n + h) % (D / 32);    // K tile and step
#pragma unroll
                for (int part = PARTS - 1; part >= 0; part--)
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        x[c][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            f[n % 3][h], q[c].f[part][j], j == 0 && part == PARTS - 1 ? f32x4{0, 0, 0, 0} : x[c][k], 0, 0, 0);
            }
        }
        read(f[0], lv, 0);
        read(f[1], lv, 1);
        half8 p8[NC][PARTS][2];
#pragma unroll
        for (int c = 0; c < NC; c++) {
            if (key0 + KV4_PAGE - 1 > low[c] || (a.window && key0 <= high[c] - a.window) || key0 >= pe * KV4_PAGE)
                mask_scores(x[c], key0, key0 < pe * KV4_PAGE ? pos[c] : -1, a.window, kg);
        }
        // the next page is laid down in the buffer that was read before the last
        // barrier: early, so that this round's barrier does not wait for the writes (at
        // the end 1% more), but with f32 rows' scores, not their probabilities beside
        // it (33 registers spilled: 12% more)
        if (PARTS == 2 && it + 1 < rounds) stage(g, it + 1);
        page_softmax<T, D, NC>(s, x, unit, p8);
        if (PARTS == 1 && it + 1 < rounds) stage(g, it + 1);
#pragma unroll
        for (int n = 0; n < VF / 2; n++) {
            if (n < VF / 2 - 2) read(f[(n + 2) % 3], lv, n + 2);
            __builtin_amdgcn_sched_barrier(DS_STAYS);
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < NC; c++)
                    add_values(s[c].o[(2 * n + h) % (D / 16)], f[n % 3][h], p8[c], (2 * n + h) / (D / 16));
        }
        __syncthreads();
    }
    float l[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        l[c] = add_xor32(add_xor16(s[c].l));
        if (poisoned[c]) l[c] = __builtin_nanf("");
        if (half) {                  // the pages are read: their place takes this half's result
            const int cw = (share * NC + c) * 16 + r;
            if (kg == 0) lds.half.m[cw] = s[c].m, lds.half.l[cw] = l[c];
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int i = 0; i < D / 16; i += 4)
                    *(f32x4 *)&lds.half.o[cw][D / 4 * kg + D / 16 * e + i] =
                        f32x4{s[c].o[i][e], s[c].o[i + 1][e], s[c].o[i + 2][e], s[c].o[i + 3][e]};
        }
    }
    if constexpr (HALVES == 2) __syncthreads();
    if (half) return;
    const int64_t pi = ((int64_t)ti * a.cache.heads + hk) * a.splits + sp;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int cw = (share * NC + c) * 16 + r, col = t.cb + cw;
        if (col >= t.ncols) continue;
        float M = s[c].m, f1 = 1.0f, f2 = 0.0f, sum = l[c];
        if constexpr (HALVES == 2) {
            const float m2 = lds.half.m[cw];
            M = fmaxf(s[c].m, m2);
            f1 = s[c].m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s[c].m - M);
            f2 = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m2 - M);
            sum = l[c] * f1 + lds.half.l[cw] * f2;
        }
        const float by = parts > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;   // a column that saw nothing has o = 0
        if (parts > 1 && kg == 0) a.part[pi * 2 * W + cw] = M, a.part[(pi * 2 + 1) * W + cw] = sum;
        float *part = a.part + a.part_rows + (pi * W + cw) * D + D / 4 * kg;
        T *out = (T *)a.out + (t.r0 + col / a.group) * a.out_stride + (hk * a.group + col % a.group) * D + D / 4 * kg;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int i = 0; i < D / 16; i += 4) {
                f32x4 o = f32x4{s[c].o[i][e], s[c].o[i + 1][e], s[c].o[i + 2][e], s[c].o[i + 3][e]} * (f1 * by);
                if constexpr (HALVES == 2) o += *(const f32x4 *)&lds.half.o[cw][D / 4 * kg + D / 16 * e + i] * (f2 * by);
                if (parts > 1)
                    *(f32x4 *)(part + D / 16 * e + i) = o;
                else
                    store4(out + D / 16 * e + i, o, a.vec);
            }
    }
}

// The parts of a tile's columns joined, one column at a time: weights 2^(m - M),
// then the rows' weighted sum, 256 / (D / 4) of them at once.  32 parts of 16
// columns 3.7 us, all of it the way from launch to store.
template <class T, int D, int W>
__global__ void __launch_bounds__(256)
k_kv4_attn_join(Kv4Attn a)
{
    constexpr int L = D / 4, ROWS = 256 / L;
    __shared__ float w[64];
    __shared__ f32x4 so[ROWS][L];
    const int ti = blockIdx.x / a.cache.heads, hk = blockIdx.x % a.cache.heads, lane = threadIdx.x & 63;
    AttnTile t;
    if (!find_tile(a, ti, W, t)) return;
    int minpos, maxpos, pg0, pages;
    tile_pages(a, t, W, minpos, maxpos, pg0, pages);
    const int parts = tile_parts(pages, a.chunk, a.splits);
    if (parts == 1) return;
    const int64_t p0 = ((int64_t)ti * a.cache.heads + hk) * a.splits;
    const int i = threadIdx.x % L, g = threadIdx.x / L;
    for (int c = blockIdx.y; c < min(W, t.ncols - t.cb); c += gridDim.y) {
        const int col = t.cb + c;
        float m = -INFINITY, l = 0.0f;
        if (lane < parts) m = a.part[(p0 + lane) * 2 * W + c], l = a.part[((p0 + lane) * 2 + 1) * W + c];
        const float M = wave_max_dpp(m);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
        const float sum = wave_sum_dpp(l * f);
        __syncthreads();             // the column before is read
        if (threadIdx.x < 64) w[lane] = f;
        __syncthreads();
        f32x4 o = {0, 0, 0, 0};
        for (int s = g; s < parts; s += ROWS)
            o += *(const f32x4 *)(a.part + a.part_rows + ((p0 + s) * W + c) * D + 4 * i) * w[s];
        so[g][i] = o;
        __syncthreads();
        if (g) continue;
#pragma unroll
        for (int k = 1; k < ROWS; k++) o += so[k][i];
        store4((T *)a.out + (t.r0 + col / a.group) * a.out_stride + (hk * a.group + col % a.group) * D + 4 * i,
               sum == 0.0f ? f32x4{0, 0, 0, 0} : o / sum, a.vec);
    }
}

// Tiles there can be: the number after the last sequence's last.
static int64_t attn_tiles(int64_t rows, int n_seqs, int group, int W) { return kv4_first_tile(rows, group, n_seqs, W); }

// How a call is cut: columns of a tile, pages of a workgroup, the most
// workgroups of a tile.
//
// The wide tiles unpack a page once for 128 columns, but cost the same for a
// few and take a page longer (1.9 us, 16 columns 0.9): they pay where three tiles
// of 16 columns (f32: four) do not hold a sequence's and there are enough to fill
// the card.  16 columns / wide, in us, 8 kv heads of two:
//   64 sequences of 400, 24, 28, 64 rows each  30 / 29, 35 / 29, 62 / 37
//     of 1000, f32, 32, 40, 64 rows            66 / 72, 80 / 74, 124 / 82
//   32 of 2048, 28, 40, 128 rows               49 / 49, 59 / 51, 168 / 93
//     f32, 32, 40, 128 rows                    60 / 72, 73 / 72, 216 / 140
//   8 of 2048, 64, 128, 256 rows               28 / 49, 48 / 51, 85 / 53
//     f32, 128, 256 rows                       59 / 73, 109 / 77
//
// Splitting a tile's pages costs a second kernel (5 us, and its launch), and
// pays where workgroups are few and the way is long: 16 sequences of 16000
// positions in 1024 parts 45 us, in 256 81.  Whole stay
// - up to 24 pages, and the more the more workgroups of eight waves there are:
//   whole / split, one sequence of 1500 13 / 15, of 2000 15 / 15, 16 of 2500 19 / 20, of
//   3000 21 / 20, 28 of 3000 22 / 29, of 4000 27 / 34;
// - up to 16 pages of more workgroups than CUs, of four waves, and up to 64 where
//   those fill the card twice (64 of 1365 to 4096 45, in two 61);
// - up to 128 on wide tiles (16 of 2048, 64 rows each, 51, in two 72).
// Longer ones are split there too, for the sake of the shorter ones beside them.
Kv4Cut kv4_attn_cut(bool f32, int64_t rows, int n_seqs, int group, int kv_heads, int64_t max_len, int window)
{
    Kv4Cut c{};
    const int64_t cols = n_seqs ? rows * group / n_seqs : 0;     // of an average sequence
    const bool wide = f32 ? cols > 64 && rows * group * kv_heads > 20480 : cols > 48 && rows * group * kv_heads > 16384;
    c.width = wide ? KV4_WIDE : KV4_W;
    const int64_t items = std::max<int64_t>(attn_tiles(rows, n_seqs, group, c.width) * kv_heads, 1);
    int64_t pages = (std::min<int64_t>(max_len, INT32_MAX) + KV4_PAGE - 1) / KV4_PAGE;    // lengths have 32 bits
    if (window) pages = std::min<int64_t>(pages, ((int64_t)window + c.width - 2) / KV4_PAGE + 2);
    int64_t per = 128;
    if (!wide) {
        const int64_t whole = items <= ROUND ? 24 + (items - 8) / 6 : 16;
        per = items >= 512 ? 64 : pages <= whole ? whole : std::max<int64_t>((items * pages / 1024 + 3) / 4 * 4, 8);
    }
    per = std::max<int64_t>(per, (pages + 63) / 64);
    c.chunk = (int)std::min<int64_t>(per, INT32_MAX / KV4_PAGE);
    c.splits = (int)std::max<int64_t>(1, (pages + per - 1) / per);
    c.parts = c.splits > 1 && rows && n_seqs ? items * c.splits : 0;
    return c;
}

// The kv heads of a tile are neighbours in the grid: workgroups go round the
// XCDs one by one, and so each XCD gets as much of a long sequence as of a
// short one (64 sequences of 1365 to 4096 positions in the order given: 53 us, with
// the tiles as neighbours 59).
template <class T, int D>
static hipError_t launch_attn(const Kv4Attn &a, int width, hipStream_t s)
{
    const unsigned tiles = (unsigned)attn_tiles(a.rows, a.n_seqs, a.group, width);
    const bool wide = width == KV4_WIDE;
    const dim3 grid(tiles * a.cache.heads, a.splits);
    // about how many tiles there are: sequences of the average length
    const int64_t cols = ((int64_t)a.rows * a.group + a.n_seqs - 1) / a.n_seqs;
    if (wide && (cols + width - 1) / width * a.n_seqs * a.cache.heads * a.splits <= 256)
        hipLaunchKernelGGL((k_kv4_attn_rows<T, D, 2>), grid, dim3(512), 0, s, a);
    else if (wide)
        hipLaunchKernelGGL((k_kv4_attn_rows<T, D, 1>), grid, dim3(256), 0, s, a);
    else if ((int64_t)grid.x * grid.y <= ROUND)
        hipLaunchKernelGGL((k_kv4_attn<T, D, 8>), grid, dim3(512), 0, s, a);
    else
        hipLaunchKernelGGL((k_kv4_attn<T, D, 4>), grid, dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    // a workgroup a column of an average sequence's tile
    const dim3 join(tiles * a.cache.heads, (unsigned)std::min<int64_t>(width, cols));
    if (wide)
        hipLaunchKernelGGL((k_kv4_attn_join<T, D, KV4_WIDE>), join, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((k_kv4_attn_join<T, D, KV4_W>), join, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t enqueue_kv4_attn(const Kv4Attn &a, int dtype, int D, int width, hipStream_t s)
{
    KV4_TYPED(dtype, D, (launch_attn<T, HD>(a, width, s)));
}

}  // namespace qtts
