// What the paged key/value operators (mocha_kv.h) share: the arguments as the kernels see
// them, the ranges of visible keys, the split of the attention's work over CTAs with the
// join of its parts, and the host-side checks.
//
// The split.  An attention call is a list of units (a sequence's block of query rows with
// the heads of one kv head) and a unit is a list of key tiles.  The tiles of all units, in
// order, are dealt to the CTAs in equal contiguous shares, so that ragged lengths, causal
// blocks and one long sequence load every SM alike.  Lengths are on the device, so each
// CTA finds its share itself.  A unit inside one share is finished there; one that is cut
// leaves an unnormalised part (maximum, sum, output) per share, and the join kernel adds
// the parts in the order of the shares: the result does not depend on timing.  A CTA
// leaves at most two parts, one of a unit that it continues and one of a unit that it
// begins, so the workspace does not grow with the batch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>
#include <type_traits>
#include <utility>

#include "mb_async.cuh"
#include "mb_common.cuh"
#include "mocha_kv.h"

namespace kv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxGroup = 64;  // query heads per kv head

// n / d for n < 2^31, by a multiplication (round-up method of Granlund and Montgomery).
struct FastDiv {
    uint32_t d, mul, s1, s2;
};

inline FastDiv fast_div(uint32_t d)
{
    int l = 0;
    while ((1ull << l) < d) l++;
    return FastDiv{d, (uint32_t)((((1ull << l) - d) << 32) / d + 1), (uint32_t)(l < 1 ? l : 1), (uint32_t)(l > 1 ? l - 1 : 0)};
}

MB_DEV uint32_t div(FastDiv f, uint32_t n)
{
    const uint32_t t = __umulhi(f.mul, n);
    return (t + ((n - t) >> f.s1)) >> f.s2;
}

// A unit that is cut, left for the join by the CTA in which it begins: parts lie in that
// CTA's slot 1 and in slot 0 of the CTAs up to c_end.  Row r of the unit is token
// row0 + r / ng, head head0 + r % ng.
struct Meta {
    int row0, head0, ng;
    int seq, pos0;  // sequence, and position of token row0
};

struct Args {
    const char *k, *v;
    long long ps, hs, ts;  // elements
    int pages, kv_heads, d;
    FastDiv page;
    const int *table;
    long long table_stride;
    int max_len;  // positions that a table row can hold
    const int *kv_len;
    int *status;
    int seqs;
    int heads, group, window;
    FastDiv group_div;
    float scale, cap;
    const int *prefix;
    const float *slopes;
    const char *q;
    char *out;
    long long q_row, q_head, o_row, o_head;  // elements
    float *lse;
    const int *q_start;  // prefill
    int rows;
    int wait_polls;  // of a wait in the prompt kernel before it gives up
    int drop;  // tests: CTA b never copies the values of its key tile b % drop, so that waits run out
    int2 *note;   // [CTAs] c_end, or -1 where no unit is cut, and rows of the unit; -1 - rows from a CTA that gave up
    Meta *meta;   // [CTAs]
    float *part;  // [CTAs][2][part rows][2 + padded dim]: outputs of all rows, then (m, l) of all rows
};

MB_DEV int seq_len(const Args &a, int s) { return min(max(__ldg(a.kv_len + s), 0), a.max_len); }
MB_DEV int seq_prefix(const Args &a, int s, int len) { return a.prefix ? min(max(__ldg(a.prefix + s), 0), len) : 0; }

// Tiles of T keys that queries at positions [pa, pb] of a sequence see: those of the
// prefix, [0, pre_t), and those from lo_t on.  At least one tile, so that rows that see
// nothing are written too.
template <int T>
struct Tiles {
    int pre_t, lo_t, n;
    MB_DEV void set(const Args &a, int len, int pre, int pa, int pb)
    {
        const int hi = min(pb + 1, len), lo = a.window ? max(pa - a.window + 1, 0) : 0;
        pre_t = (pre + T - 1) / T;
        lo_t = max(lo / T, pre_t);
        n = max(pre_t + max((max(hi, 0) + T - 1) / T - lo_t, 0), 1);
    }
    MB_DEV int key(int i) const { return (i < pre_t ? i : i - pre_t + lo_t) * T; }
};

MB_DEV bool visible(int j, int p, int len, int pre, int window)
{
    return j < len && ((j <= p && (window == 0 || p - j < window)) || j < pre);
}

// Page of position j, or -1 for an id outside the pool.
MB_DEV int page_of(const Args &a, int seq, int j)
{
    const int id = __ldg(a.table + (long long)seq * a.table_stride + div(a.page, (uint32_t)j));
    if ((unsigned)id < (unsigned)a.pages) return id;
    if (a.status) atomicMax(a.status, 1);
    return -1;
}

// Score in units of log2 from the plain product.
MB_DEV float score2(const Args &a, float dot, float slope, int p, int j)
{
    float z = dot * a.scale;
    if (a.cap > 0.f) z = a.cap * tanhf(z / a.cap);
    if (a.slopes) z -= slope * (float)abs(p - j);
    return z * kLog2e;
}

// 2^x by the hardware's exponential (2 ulp and subnormal results as zero, far below what
// rounding a weight to 16 bits costs).
MB_DEV float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// tanh x = x P(x^2) within 0.6, P of least largest relative error on [0, 0.36] (2^-23.4), so
// that scores far below their cap keep their places; 1 - 2 / (1 + exp 2x) elsewhere.
constexpr float kTanhPart = 0.6f;
constexpr float kTanh0 = 0.9999999403953552f, kTanh1 = -0.33332309126853943f, kTanh2 = 0.13310173153877258f,
                kTanh3 = -0.05210148170590401f, kTanh4 = 0.015475427731871605f;
MB_DEV float tanh_small(float x)
{
    const float t = x * x;
    return x * fmaf(fmaf(fmaf(fmaf(kTanh4, t, kTanh3), t, kTanh2), t, kTanh1), t, kTanh0);
}
MB_DEV float tanh_large(float x) { return 1.f - __fdividef(2.f, 1.f + ex2(x * (2.f * kLog2e))); }
MB_DEV float tanh_of(float x) { return fabsf(x) <= kTanhPart ? tanh_small(x) : tanh_large(x); }

// Weights are rounded to the cache's 16-bit type for the product with the values.  The prompt
// kernel rounds them once: with the rest of each in a second product the outputs' error falls
// by a sixth (1024 tokens) to a quarter (8192), to that of their own rounding, and the call takes
// 6 % (1024 tokens), 13 % (short pieces after long texts), 20 % (every option) and 36 % (8192)
// longer.  The single-token kernel has the second product: there it costs 1 to 2 % (wide groups:
// kv_decode.cu).
//
// They are taken 2^kLift above the value that they are relative to, and pass it by 2^8 before it
// is renewed: fp16's then reach from 2^15, half its range, down to its last bit, 2^-24, so that
// one is lost only 2^-32 below the largest, and 131071 of those are 2^-15 of the sum (fp32 sums
// lose as much).  bf16 has fp32's range.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;

template <typename T>
MB_DEV float to_f32(T x)
{
    return (float)x;
}
template <typename T>
MB_DEV T from_f32(float x)
{
    return (T)x;
}

// Zero if four values are finite, NaN else.
MB_DEV float load_zero4(const float *p)
{
    const float4 x = *reinterpret_cast<const float4 *>(p);
    return fmaf(x.x, 0.f, fmaf(x.y, 0.f, fmaf(x.z, 0.f, x.w * 0.f)));
}
template <typename T>
MB_DEV float load_zero4(const T *p)
{
    const uint2 r = *reinterpret_cast<const uint2 *>(p);
    const T *x = reinterpret_cast<const T *>(&r);
    return fmaf(to_f32(x[0]), 0.f, fmaf(to_f32(x[1]), 0.f, fmaf(to_f32(x[2]), 0.f, to_f32(x[3]) * 0.f)));
}

// Two roundings in one instruction.
template <typename T>
MB_DEV uint32_t pack2(float x, float y)
{
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

MB_DEV void store4(float *p, float4 x) { *reinterpret_cast<float4 *>(p) = x; }
MB_DEV void store4(__half *p, float4 x)
{
    __half2 h[2] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w)};
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(h);
}
MB_DEV void store4(__nv_bfloat16 *p, float4 x)
{
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(h);
}

// Whether a value that is not finite lies at a key which a prompt's row at position p does not
// see, in the tiles of T keys of its unit, whose rows stand at [pa, pb]: only then can it have
// reached the row's output (0 * inf).  By a warp, a key per lane; keys the row sees are not read.
template <typename T, int TILE>
__device__ __forceinline__ bool unseen_values(const Args &a, int seq, int p, int head, int pa, int pb)
{
    const int lane = threadIdx.x & 31, len = seq_len(a, seq), pre = seq_prefix(a, seq, len);
    const int kvh = div(a.group_div, head), lo = a.window ? max(p - a.window + 1, 0) : 0;
    Tiles<TILE> t;
    t.set(a, len, pre, pa, min(pb + 1, len) - 1);
    const int end = min(t.n * TILE + (t.lo_t - t.pre_t) * TILE, len);
    bool bad = false;
    // past the prefix, before the window, after the row
#pragma unroll 1
    for (int part = 0; part < 3 && !bad; part++) {
        const int j0 = part == 0 ? pre : part == 1 ? t.lo_t * TILE : max(p + 1, t.lo_t * TILE);
        const int j1 = part == 0 ? min(t.pre_t * TILE, len) : part == 1 ? min(lo, end) : end;
#pragma unroll 1
        for (int jb = j0; jb < j1 && !bad; jb += 32) {
            const int j = jb + lane;
            float worst = 0.f;
            if (j < j1 && !visible(j, p, len, pre, a.window)) {
                const int id = __ldg(a.table + (long long)seq * a.table_stride + div(a.page, j));
                if ((unsigned)id < (unsigned)a.pages) {
                    const T *v = reinterpret_cast<const T *>(a.v) + id * a.ps + kvh * a.hs + (long long)(j - div(a.page, j) * a.page.d) * a.ts;
#pragma unroll 4
                    for (int i = 0; i < a.d; i += 4) worst += load_zero4(v + i);
                }
            }
            bad = __any_sync(0xffffffffu, !(worst == 0.f));
        }
    }
    return bad;
}

// One row of a prompt's attention by a warp, reading only the keys that the row sees, where
// unseen_values says so.  Rare, so written for size.  The row's lse is right without it: masked
// scores are replaced, not multiplied.
template <typename T>
__device__ __forceinline__ void lone_row(const Args &a, int seq, int p, int head, int row)
{
    const int lane = threadIdx.x & 31, d = a.d, per = d / 32;
    const int len = seq_len(a, seq), pre = seq_prefix(a, seq, len);
    const int kvh = div(a.group_div, head);
    const T *q = reinterpret_cast<const T *>(a.q) + row * a.q_row + head * a.q_head;
    const float slope = a.slopes ? a.slopes[head] : 0.f;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int hi = min(p + 1, len), lo = max(a.window ? max(p - a.window + 1, 0) : 0, pre);
    bool known = false;  // every value of the row is NaN, whatever else it sees
#pragma unroll 1
    for (int part = 0; part < 2; part++) {
        const int j0 = part ? lo : 0, j1 = part ? hi : pre;
#pragma unroll 1
        for (int jb = j0; jb < j1 && !known; jb += 32) {
            const int j = jb + lane;
            float z = -INFINITY;
            long long at = -1;
            if (j < j1) {
                const int id = page_of(a, seq, j);
                float dot = 0.f;
                if (id >= 0) {
                    at = id * a.ps + kvh * a.hs + (long long)(j - div(a.page, j) * a.page.d) * a.ts;
                    const T *kr = reinterpret_cast<const T *>(a.k) + at;
#pragma unroll 1
                    for (int i = 0; i < d; i++) dot = fmaf(to_f32(q[i]), to_f32(kr[i]), dot);
                }
                z = score2(a, dot, slope, p, j);
            }
            const float mn = fmaxf(m, mb::warp_max(z)), ms = mn == -INFINITY ? 0.f : mn;
            const float f = exp2f(m - ms), e = j < j1 ? exp2f(z - ms) : 0.f;
            m = mn;
            l = l * f + mb::warp_sum(e);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] *= f;
#pragma unroll 1
            for (int t = 0; t < min(32, j1 - jb); t++) {
                const float w = __shfl_sync(0xffffffffu, e, t);
                const long long vt = __shfl_sync(0xffffffffu, at, t);
                if (vt >= 0)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (i < per) acc[i] = fmaf(w, to_f32(reinterpret_cast<const T *>(a.v)[vt + lane + 32 * i]), acc[i]);
            }
            bool nan = true;
#pragma unroll
            for (int i = 0; i < 4; i++) nan &= i >= per || isnan(acc[i]);
            known = isnan(l) || (l > 0.f && __all_sync(0xffffffffu, nan));
        }
    }
    T *o = reinterpret_cast<T *>(a.out) + row * a.o_row + head * a.o_head;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < per) o[lane + 32 * i] = from_f32<T>(l == 0.f ? 0.f : acc[i] / l);
}

// A row of a CTA that gave up: not a number, so that nobody takes it for a result.  By a warp.
template <typename T>
MB_DEV void lost_row(const Args &a, long long row, int head)
{
    const int lane = threadIdx.x & 31;
    const float x = __int_as_float(0x7fffffff);
    if (lane * 4 < a.d) store4(reinterpret_cast<T *>(a.out) + row * a.o_row + head * a.o_head + lane * 4, make_float4(x, x, x, x));
    if (a.lse && lane == 0) a.lse[row * a.heads + head] = x;
}

// ---- asynchronous copies ----------------------------------------------------------------

MB_DEV void cp_async16(uint32_t dst, const void *src, bool ok)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
MB_DEV void cp_async16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
MB_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
MB_DEV void cp_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---- join of the parts of cut units --------------------------------------------------
// The rows of all cut units are dealt to the blocks: a warp takes a row whose parts are
// few, a block one whose parts are many (more than kJoinSerial), lanes the dims.  Bound by
// the parts' bytes: each is read once.
// Two large blocks an SM: every block reads all notes, and more would queue for their lines.
// kJoinSerial: with 4 the short fp32 pieces take 36.8 us for 30.6, with 64 the pieces after long
// texts 48.2 for 40.8 and the long sequences' single tokens 40.4 for 36.8.
constexpr int kJoinWarps = 16, kJoinSerial = 16, kJoinMetas = 2 * mb::kSMs, kJoinBlocks = 2 * mb::kSMs;

struct Joined {
    float m, l;
    float4 acc;
    MB_DEV void add(float pm, float pl, float4 v, float ms)
    {
        const float f = exp2f(pm - ms);
        l = fmaf(pl, f, l);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
    }
    MB_DEV void rescale(float mn, float ms)
    {
        const float f = exp2f(m - ms);
        l *= f;
        acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
        m = mn;
    }
};

template <typename T, bool PREFILL>
__global__ void __launch_bounds__(32 * kJoinWarps, 2) k_join(const __grid_constant__ Args a, int metas, int part_rows, int dp)
{
    __shared__ Joined s_part[kJoinWarps][32];
    __shared__ int s_items[kJoinMetas], s_warp[kJoinWarps], s_total;
    __shared__ int2 s_note[kJoinMetas];
    __shared__ bool s_gave_up[kJoinMetas];
    mb::as::griddep_launch();
    mb::as::griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // items (a block's work) before each unit's end, in the order of the CTAs
    static_assert(kJoinMetas <= 32 * kJoinWarps, "a thread per note");
    int n = 0;
    if (tid < metas) {
        int2 note = __ldcg(a.note + tid);
        s_gave_up[tid] = note.y < 0;
        if (note.y < 0) note.y = -1 - note.y;
        s_note[tid] = note;
        if (note.x >= 0) n = note.x - tid < kJoinSerial ? (note.y + kJoinWarps - 1) / kJoinWarps : note.y;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    for (int w = 0; w < warp; w++) incl += s_warp[w];
    if (tid < metas) s_items[tid] = incl;
    if (tid == 32 * kJoinWarps - 1) s_total = incl;
    __syncthreads();
    const int total = s_total;
    const size_t slot = (size_t)part_rows * (dp + 2);
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        int c = 0;  // the first unit that ends after `item`
        for (int step = 256; step; step >>= 1)
            if (c + step <= metas && s_items[c + step - 1] <= item) c += step;
        const int2 note = s_note[c];
        const Meta mt = a.meta[c];
        const int first = c ? s_items[c - 1] : 0, c_end = note.x;
        const bool serial = c_end - c < kJoinSerial;
        const int r = serial ? (item - first) * kJoinWarps + warp : item - first;
        const bool there = r < note.y;
        if (PREFILL) {
            bool lost = false;
            for (int b = c + lane; b <= c_end; b += 32) lost |= s_gave_up[b];
            if (__any_sync(0xffffffffu, lost)) {  // a part is missing
                if (there && (serial || warp == 0)) lost_row<T>(a, mt.row0 + r / mt.ng, mt.head0 + r % mt.ng);
                continue;
            }
        }
        Joined x{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
        constexpr int U = 4;  // parts in flight per warp
        if (there)
            for (int b = c + (serial ? 0 : warp * U); b <= c_end; b += serial ? U : kJoinWarps * U) {
                float pm[U], pl[U];
                float4 pv[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    pm[u] = -INFINITY;
                    pl[u] = 0.f;
                    pv[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (b + u <= c_end) {
                        const float *pp = a.part + ((size_t)(b + u) * 2 + (b + u == c ? 1 : 0)) * slot;
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(pp + (size_t)part_rows * dp) + r);
                        pm[u] = ml.x;
                        pl[u] = ml.y;
                        if (lane * 4 < a.d) pv[u] = __ldcg(reinterpret_cast<const float4 *>(pp + (size_t)r * dp) + lane);
                    }
                }
                float mn = x.m;
#pragma unroll
                for (int u = 0; u < U; u++) mn = fmaxf(mn, pm[u]);
                const float ms = mn == -INFINITY ? 0.f : mn;
                x.rescale(mn, ms);
#pragma unroll
                for (int u = 0; u < U; u++) x.add(pm[u], pl[u], pv[u], ms);
            }
        if (!serial) {
            s_part[warp][lane] = x;
            __syncthreads();
            if (warp == 0) {
                float mn = x.m;
#pragma unroll
                for (int w = 1; w < kJoinWarps; w++) mn = fmaxf(mn, s_part[w][0].m);
                const float ms = mn == -INFINITY ? 0.f : mn;
                x.rescale(mn, ms);
#pragma unroll
                for (int w = 1; w < kJoinWarps; w++) x.add(s_part[w][lane].m, s_part[w][lane].l, s_part[w][lane].acc, ms);
            }
            __syncthreads();
        }
        if (there && (serial || warp == 0)) {
            const float inv = 1.f / x.l;
            const int t = r / mt.ng, head = mt.head0 + r - t * mt.ng;
            const long long row = mt.row0 + t;
            x.acc = x.l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                               : make_float4(x.acc.x * inv, x.acc.y * inv, x.acc.z * inv, x.acc.w * inv);
            if (lane * 4 < a.d) store4(reinterpret_cast<T *>(a.out) + row * a.o_row + head * a.o_head + lane * 4, x.acc);
            if (a.lse && lane == 0)
                a.lse[row * a.heads + head] = x.l == 0.f ? -INFINITY : ((x.m == -INFINITY ? 0.f : x.m) + log2f(x.l)) * kLn2;
            if (PREFILL) {
                const bool bad = !(isfinite(x.acc.x) && isfinite(x.acc.y) && isfinite(x.acc.z) && isfinite(x.acc.w));
                if (__any_sync(0xffffffffu, bad && lane * 4 < a.d) &&
                    unseen_values<T, sizeof(T) == 4 ? 64 : 128>(a, mt.seq, mt.pos0 + t, head, mt.pos0, mt.pos0 + note.y / mt.ng - 1)) {
                    __syncwarp();
                    lone_row<T>(a, mt.seq, mt.pos0 + t, head, (int)row);
                }
            }
        }
    }
}

// n / d by 32-bit arithmetic where both fit, as they nearly always do.
MB_DEV long long div64(long long n, long long d)
{
    if (((n | d) >> 32) == 0) return (uint32_t)n / (uint32_t)d;
    return n / d;
}

// ---- host ------------------------------------------------------------------------------

inline int fail(const char *who, const char *what)
{
    fprintf(stderr, "%s: %s\n", who, what);
    return 1;
}

// Makes `device` current for a call and puts the caller's back.  What a device is does not
// change, so it is asked once (two threads that ask at once find the same).
class DeviceGuard {
  public:
    int enter(const char *who, int device)
    {
        static std::atomic<unsigned long long> known{0};
        if (cudaGetDevice(&old_) != cudaSuccess) return (void)cudaGetLastError(), fail(who, "no CUDA device");
        const unsigned long long bit = device >= 0 && device < 64 ? 1ull << device : 0;
        if (!(known.load(std::memory_order_relaxed) & bit)) {
            int count = 0, major = 0;
            if (cudaGetDeviceCount(&count) != cudaSuccess) return (void)cudaGetLastError(), fail(who, "no CUDA device");
            if (device < 0 || device >= count) return fail(who, "device out of range");
            if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) != cudaSuccess || major != 10)
                return fail(who, "requires a compute capability 10.x (B200) device");
            known.fetch_or(bit, std::memory_order_relaxed);
        }
        if (device != old_) {
            if (cudaSetDevice(device) != cudaSuccess) return (void)cudaGetLastError(), fail(who, "cudaSetDevice failed");
            changed_ = true;
        }
        device_ = device;
        return 0;
    }
    int device() const { return device_; }
    ~DeviceGuard()
    {
        if (changed_) cudaSetDevice(old_);
    }

  private:
    int old_ = 0, device_ = 0;
    bool changed_ = false;
};

inline int type_bytes(int type) { return type == MOCHA_KV_F32 ? 4 : type == MOCHA_KV_F16 || type == MOCHA_KV_BF16 ? 2 : 0; }

inline bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

inline int check_pages(const char *who, const mocha_kv_pages *p)
{
    if (!p) return fail(who, "null pages");
    const int b = type_bytes(p->type);
    if (!b) return fail(who, "type must be MOCHA_KV_F32, MOCHA_KV_F16 or MOCHA_KV_BF16");
    if (p->pages < 1 || p->kv_heads < 1) return fail(who, "pages and kv_heads must be positive");
    if (p->page_size < 8 || p->page_size % 8 || p->page_size > 65536)
        return fail(who, "page_size must be a multiple of 8 up to 65536");
    if (p->head_dim < 32 || p->head_dim % 32 || p->head_dim > 128)
        return fail(who, "head_dim must be 32, 64, 96 or 128");
    if (p->page_stride < 0 || p->head_stride < 0 || p->token_stride < p->head_dim)
        return fail(who, "strides must not be negative and token_stride at least head_dim");
    // the byte strides must stay below 2^40, where the tiled copies can address them
    const long long most = (1ll << 40) / b - 1;
    if (p->page_stride > most || p->head_stride > most || p->token_stride > most) return fail(who, "stride too large");
    if (p->page_stride * b % 16 || p->head_stride * b % 16 || p->token_stride * b % 16)
        return fail(who, "page, head and token strides must be multiples of 16 bytes");
    if (!p->k || !p->v || !aligned(p->k) || !aligned(p->v)) return fail(who, "k and v must be 16-byte aligned pointers");
    return 0;
}

inline int check_seqs(const char *who, const mocha_kv_seqs *s)
{
    if (!s) return fail(who, "null seqs");
    if (s->seqs < 0) return fail(who, "seqs must not be negative");
    if (s->table_width < 1 || s->table_stride < s->table_width) return fail(who, "table_width must be positive and table_stride at least that");
    if (s->seqs && !s->table) return fail(who, "null table");
    return 0;
}

inline int check_rows(const char *who, const char *name, const mocha_kv_rows *r, int bytes, int dim, int rows)
{
    const long long most = (1ll << 40) / bytes - 1;
    if (!r || (rows && !r->data)) return fprintf(stderr, "%s: null %s\n", who, name), 1;
    if (!aligned(r->data) || r->row_stride < 0 || r->head_stride < dim || r->row_stride > most || r->head_stride > most ||
        r->row_stride * bytes % 16 || r->head_stride * bytes % 16) {
        fprintf(stderr, "%s: %s must be 16-byte aligned with strides that are multiples of 16 bytes and a head stride of at least head_dim\n", who, name);
        return 1;
    }
    return 0;
}

inline int check_scores(const char *who, const mocha_kv_pages *p, const mocha_kv_scores *s)
{
    if (!s) return fail(who, "null scores");
    if (s->heads < 1 || s->heads % p->kv_heads || s->heads / p->kv_heads > kMaxGroup)
        return fail(who, "heads must be a multiple of kv_heads, at most 64 times as many");
    // within these bounds no scale / cap or multiple of it leaves the range of fp32
    constexpr float kMost = 0x1p40f;
    if (!(fabsf(s->scale) <= kMost)) return fail(who, "scale must be finite, 2^40 at most");
    if (s->cap != 0.f && !(s->cap >= 1.f / kMost && s->cap <= kMost)) return fail(who, "cap must be 0 or from 2^-40 to 2^40");
    if (s->window < 0) return fail(who, "window must not be negative");
    return 0;
}

// Positions and rows, so that no sum or difference of two, a window or a tile overflows.
constexpr int kMostPositions = 1 << 30;

inline int max_len(const mocha_kv_pages *p, const mocha_kv_seqs *s)
{
    const long long n = (long long)s->table_width * p->page_size;
    return n > kMostPositions ? kMostPositions : (int)n;
}

inline Args make_args(const mocha_kv_pages *p, const mocha_kv_seqs *s, const mocha_kv_scores *z, const mocha_kv_rows *q,
                      const mocha_kv_rows *out, float *lse)
{
    Args a{};
    a.k = (const char *)p->k;
    a.v = (const char *)p->v;
    a.ps = p->page_stride;
    a.hs = p->head_stride;
    a.ts = p->token_stride;
    a.pages = p->pages;
    a.kv_heads = p->kv_heads;
    a.d = p->head_dim;
    a.page = fast_div(p->page_size);
    a.table = s->table;
    a.table_stride = s->table_stride;
    a.max_len = max_len(p, s);
    a.kv_len = s->kv_len;
    a.status = s->status;
    a.seqs = s->seqs;
    a.heads = z->heads;
    a.group = z->heads / p->kv_heads;
    a.group_div = fast_div(a.group);
    a.window = z->window < a.max_len ? z->window : 0;  // a window that holds every position is none
    a.scale = z->scale;
    a.cap = z->cap;
    a.prefix = z->prefix;
    a.slopes = z->slopes;
    a.q = (const char *)q->data;
    a.q_row = q->row_stride;
    a.q_head = q->head_stride;
    a.out = (char *)out->data;
    a.o_row = out->row_stride;
    a.o_head = out->head_stride;
    a.lse = lse;
    return a;
}

// Launch on the current device with an error message.  The kernel may start while the one
// before it in the stream ends, and waits for it itself before it reads or writes anything.
template <typename... K, typename... A>
int launch(const char *who, void (*kernel)(K...), dim3 grid, int threads, size_t smem, cudaStream_t s, A &&...args)
{
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
    if (e != cudaSuccess) return (void)cudaGetLastError(), fail(who, cudaGetErrorString(e));
    return 0;
}

// More than 48 KB of shared memory for a kernel, asked for once per kernel and device:
// `allowed` is the kernel's own.
template <typename... K>
int allow_smem(const char *who, void (*kernel)(K...), size_t smem, int device, std::atomic<unsigned long long> &allowed)
{
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (allowed.load(std::memory_order_relaxed) & bit) return 0;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (void)cudaGetLastError(), fail(who, cudaGetErrorString(e));
    allowed.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

// Workspace of one call: the CTAs' notes of cut units, then their parts.
inline size_t meta_bytes(int ctas) { return ((size_t)ctas * (sizeof(int2) + sizeof(Meta)) + 255) / 256 * 256; }
inline void lay_out(Args &a, void *space, int ctas)
{
    a.note = static_cast<int2 *>(space);
    a.meta = reinterpret_cast<Meta *>(a.note + ctas);
    a.part = reinterpret_cast<float *>(static_cast<char *>(space) + meta_bytes(ctas));
}
inline size_t part_bytes(int ctas, int rows, int dp) { return (size_t)ctas * 2 * rows * (dp + 2) * sizeof(float); }
inline int padded_dim(int d) { return d <= 64 ? 64 : 128; }

}  // namespace kv
