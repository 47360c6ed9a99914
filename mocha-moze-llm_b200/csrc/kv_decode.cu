// mocha_kv_decode: attention of one new token per sequence over a paged cache (mocha_kv.h).
//
// Each cached value is used by heads / kv heads queries only (4 flops per element and
// head), so the kernel is bound by reading the visible keys and values once.  A unit is a
// sequence and one kv head with up to 8 NG of its query heads; its key tiles of 64 are
// shared out over the CTAs (kv_common.cuh).  The four warps of a CTA take 16 keys each of
// every tile and run on their own: each keeps a ring of tiles in flight in its own part of
// shared memory (16-byte asynchronous copies, which also fill the rows of keys that are
// not visible with zeros, so nothing of them can reach a sum), an online softmax and an
// output in registers; they meet when a unit ends.
//
// 16-bit types: scores are K q^T and outputs V^T p^T by m16n8k16 products, so the eight
// (or 16, 32) heads of the group are the narrow side and no lane computes on padding when
// a group has 8 heads.  The weights are rounded to the cache's type for the second
// product; their sum is taken before that, in fp32.  fp32: the same tiles on the FMA
// units, a lane holding half a key's products with 8 heads.
#include "kv_common.cuh"

namespace {

using namespace kv;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kKeys = 16;              // keys of a warp's tile
constexpr int kTile = kKeys * kWarps;  // keys of a CTA's tile

// CTAs of an SM, and the stages of a warp's ring (keys then values): 192 KB of rings per
// SM.  Two CTAs overlap one's unit ends with the other's tiles; wide groups (registers) and
// fp32 rows of 128 (three stages at least) leave room for one.
template <typename T, int DP, int NG>
struct Ring {
    static constexpr int kHalf = kKeys * DP * (int)sizeof(T), kStage = 2 * kHalf;
    static constexpr int kCtas = NG > 1 || (sizeof(T) == 4 && DP == 128) ? 1 : 2;
    static constexpr int kStages = 192 * 1024 / kCtas / kWarps / kStage;
};

template <typename T, int DP, int NG>
struct Smem {
    static constexpr int kPad = DP + 4;  // floats of a head's row in the merge buffers
    static constexpr int kQ = 8 * NG * DP * (int)sizeof(T);
    static constexpr int kRing = kWarps * Ring<T, DP, NG>::kStages * Ring<T, DP, NG>::kStage;
    static constexpr int kMerge = 3 * 8 * kPad * 4;
    static constexpr int kStat = 2 * kWarps * 8 * NG * 2 * 4;  // two buffers of (m, l)
    static constexpr int kW = sizeof(T) == 4 ? kWarps * 8 * kKeys * 4 : 0;
    static constexpr int kTotal = kRing + 2 * kQ + kMerge + kStat + kW;
};

struct Work {
    Args a;
    int hgroups, unit_heads;  // units per kv head, and query heads of a unit (the last may have fewer)
    int min_tiles;            // of a share
};

// A walk along a CTA's tiles.
struct Walk {
    int seq, hh, i;
    int len, pre;
    Tiles<kTile> t;
    MB_DEV void load(const Args &a)
    {
        len = pre = 0;
        if (seq < a.seqs) {
            len = seq_len(a, seq);
            pre = seq_prefix(a, seq, len);
        }
        t.set(a, len, pre, len - 1, len - 1);
    }
    MB_DEV void next(const Args &a, int hh_n)
    {
        if (++i < t.n) return;
        i = 0;
        if (++hh < hh_n) return;
        hh = 0;
        seq++;
        load(a);
    }
};

MB_DEV void cp_async16(uint32_t dst, const void *src, bool ok)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
MB_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
MB_DEV void cp_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

MB_DEV void ldsm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
MB_DEV void ldsm4_t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
MB_DEV uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <typename T>
MB_DEV void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

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

// The share of this CTA: its first tile as (sequence, tile within the sequence) in *s_seq
// and *s_rem, and [start, end) in tiles of the whole call.
MB_DEV bool find_share(const Work &w, int hh_n, long long *s_warp, int *s_seq, long long *s_rem, long long *start,
                       long long *end, long long *per)
{
    const Args &a = w.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int chunk = (a.seqs + kThreads - 1) / kThreads, b0 = min(tid * chunk, a.seqs), b1 = min(b0 + chunk, a.seqs);
    Walk k;
    long long sum = 0;
    for (k.seq = b0; k.seq < b1; k.seq++) {
        k.load(a);
        sum += (long long)k.t.n * hh_n;
    }
    long long incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; i++) {
        if (i < warp) incl += s_warp[i];
        total += s_warp[i];
    }
    *per = max(div64(total + gridDim.x - 1, gridDim.x), (long long)w.min_tiles);
    *start = *per * blockIdx.x;
    *end = min(*start + *per, total);
    long long at = incl - sum;
    if (*start < total && at <= *start && *start < incl) {
        for (k.seq = b0;; k.seq++) {
            k.load(a);
            const long long n = (long long)k.t.n * hh_n;
            if (*start < at + n) break;
            at += n;
        }
        *s_seq = k.seq;
        *s_rem = *start - at;
    }
    __syncthreads();
    return *start < total;
}

template <typename T, int DP, int NG>
__global__ void __launch_bounds__(kThreads, Ring<T, DP, NG>::kCtas) k_decode(const __grid_constant__ Work w)
{
    constexpr bool F32 = sizeof(T) == 4;
    using R = Ring<T, DP, NG>;
    using S = Smem<T, DP, NG>;
    constexpr int CH = DP * (int)sizeof(T) / 16;  // 16-byte pieces of a row
    constexpr int H = 8 * NG;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char *ring = smem;
    unsigned char *sq = smem + S::kRing;
    float *merge = reinterpret_cast<float *>(sq + 2 * S::kQ);
    float *stat = merge + S::kMerge / 4;
    float *sw = stat + S::kStat / 4;
    __shared__ long long s_warp[kWarps], s_rem;
    __shared__ int s_seq;
    const Args &a = w.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hh_n = a.kv_heads * w.hgroups;
    mb::as::griddep_launch();
    long long start, end, per;
    if (!find_share(w, hh_n, s_warp, &s_seq, &s_rem, &start, &end, &per)) {
        if (tid == 0) a.meta[blockIdx.x].c_end = -1;
        return;
    }
    Walk in;  // the next tile to load
    in.seq = s_seq;
    in.load(a);
    in.hh = (int)div64(s_rem, in.t.n);
    in.i = (int)(s_rem - (long long)in.hh * in.t.n);
    Walk it = in;  // the tile to compute
    const uint32_t wring = mb::as::smem_u32(ring) + warp * R::kStages * R::kStage;

    int pg[2];  // pages of the two halves of this warp's keys of tile `in`
    auto pages = [&]() {
        const int j = in.t.key(in.i) + warp * kKeys;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int jh = j + 8 * h;
            pg[h] = jh < in.len ? __ldg(a.table + in.seq * a.table_stride + div(a.page, jh)) : 0;
        }
    };
    auto issue = [&](int slot) {
        const int j = in.t.key(in.i) + warp * kKeys;
        const int kvh = w.hgroups == 1 ? in.hh : in.hh / w.hgroups;
        const int p = in.len - 1;
        const uint32_t dst = wring + slot * R::kStage;
        long long off[2];
        bool ok[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int jh = j + 8 * h;
            const int row = jh - (int)(div(a.page, jh) * a.page.d);
            ok[h] = jh < in.len && (unsigned)pg[h] < (unsigned)a.pages;
            if (jh < in.len && !ok[h] && a.status &&
                (visible(jh, p, in.len, in.pre, a.window) || visible(min(jh + 7, p), p, in.len, in.pre, a.window)))
                *a.status = 1;
            off[h] = ok[h] ? pg[h] * a.ps + kvh * a.hs + row * a.ts : 0;
        }
#pragma unroll
        for (int x = 0; x < kKeys * CH / 32; x++) {
            const int r = (lane + 32 * x) / CH, c = (lane + 32 * x) % CH;
            const bool use = ok[r / 8] && c * 16 < a.d * (int)sizeof(T) && visible(j + r, p, in.len, in.pre, a.window);
            const long long e = use ? off[r / 8] + (r & 7) * a.ts + c * (16 / (int)sizeof(T)) : 0;
            const uint32_t to = dst + r * DP * (int)sizeof(T) + ((c ^ (r & 7)) * 16);
            cp_async16(to, a.k + e * (long long)sizeof(T), use);
            cp_async16(to + R::kHalf, a.v + e * (long long)sizeof(T), use);
        }
    };

    const int tiles = (int)(end - start);
    pages();
#pragma unroll
    for (int x = 0; x < R::kStages - 1; x++) {
        if (x < tiles) {
            issue(x);
            in.next(a, hh_n);
            pages();
        }
        cp_commit();
    }

    bool began = it.i == 0;  // the unit's first tile lies in this share
    bool fresh = true;
    int buf = 0, head0 = 0, ng = 0, kvh = 0;
    float m[F32 ? 8 : 2 * NG], l[F32 ? 8 : 2 * NG];
    float acc[F32 ? 8 : NG * DP / 16][4];
    for (int x = 0; x < tiles; x++) {
        if (fresh) {
            // the unit's queries, one buffer per other unit: the last unit's may still be read
            kvh = w.hgroups == 1 ? it.hh : it.hh / w.hgroups;
            const int hg = it.hh - kvh * w.hgroups;
            head0 = kvh * a.group + hg * w.unit_heads;
            ng = min(w.unit_heads, a.group - hg * w.unit_heads);
            unsigned char *q = sq + buf * S::kQ;
            for (int e = tid; e < H * CH; e += kThreads) {
                const int h = e / CH, c = e % CH;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (h < ng && c * 16 < a.d * (int)sizeof(T))
                    v = *reinterpret_cast<const uint4 *>(a.q + (it.seq * a.q_row + (head0 + h) * a.q_head) * (long long)sizeof(T) + c * 16);
                *reinterpret_cast<uint4 *>(q + h * DP * sizeof(T) + (F32 ? c : c ^ (h & 7)) * 16) = v;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < (F32 ? 8 : 2 * NG); i++) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
            for (int i = 0; i < (F32 ? 8 : NG * DP / 16); i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][e] = 0.f;
            fresh = false;
        }
        cp_wait<R::kStages - 2>();
        __syncwarp();
        if (x + R::kStages - 1 < tiles) {
            issue((x + R::kStages - 1) % R::kStages);
            in.next(a, hh_n);
            pages();
        }
        cp_commit();
        const int j = it.t.key(it.i) + warp * kKeys, p = it.len - 1;
        const uint32_t kb = wring + (x % R::kStages) * R::kStage, vb = kb + R::kHalf;
        if constexpr (!F32) {
            float s[NG][4];
#pragma unroll
            for (int n = 0; n < NG; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] = 0.f;
            const uint32_t qb = mb::as::smem_u32(sq + buf * S::kQ);
#pragma unroll
            for (int kk = 0; kk < DP / 32; kk++) {
                uint32_t k0[4], k1[4];
                const int r = lane & 15, c = 4 * kk + (lane >> 4);
                ldsm4(kb + r * DP * 2 + ((c ^ (r & 7)) * 16), k0);
                ldsm4(kb + r * DP * 2 + (((c + 2) ^ (r & 7)) * 16), k1);
#pragma unroll
                for (int n = 0; n < NG; n++) {
                    uint32_t q[4];
                    const int h = lane & 7;
                    ldsm4(qb + (n * 8 + h) * DP * 2 + (((4 * kk + (lane >> 3)) ^ h) * 16), q);
                    mma<T>(s[n], k0, q[0], q[1]);
                    mma<T>(s[n], k1, q[2], q[3]);
                }
            }
            const int ja = j + (lane >> 2), jb = ja + 8;
            const bool va = visible(ja, p, it.len, it.pre, a.window), vb_ = visible(jb, p, it.len, it.pre, a.window);
            uint32_t pt[NG][2];
#pragma unroll
            for (int n = 0; n < NG; n++) {
                if (a.cap > 0.f || a.slopes) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int h = n * 8 + 2 * (lane & 3) + (e & 1);
                        const float slope = a.slopes && h < ng ? __ldg(a.slopes + head0 + h) : 0.f;
                        s[n][e] = score2(a, s[n][e], slope, p, e < 2 ? ja : jb);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) s[n][e] *= a.scale * kLog2e;
                }
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (!(e < 2 ? va : vb_)) s[n][e] = -INFINITY;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float mx = fmaxf(s[n][e], s[n][e + 2]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float mn = fmaxf(m[2 * n + e], mx), ms = mn == -INFINITY ? 0.f : mn;
                    const float f = exp2f(m[2 * n + e] - ms);
                    m[2 * n + e] = mn;
                    s[n][e] = exp2f(s[n][e] - ms);
                    s[n][e + 2] = exp2f(s[n][e + 2] - ms);
                    l[2 * n + e] = fmaf(l[2 * n + e], f, s[n][e] + s[n][e + 2]);
#pragma unroll
                    for (int dd = 0; dd < DP / 16; dd++) {
                        acc[n * (DP / 16) + dd][e] *= f;
                        acc[n * (DP / 16) + dd][e + 2] *= f;
                    }
                }
                pt[n][0] = transpose8(pack2<T>(s[n][0], s[n][1]));
                pt[n][1] = transpose8(pack2<T>(s[n][2], s[n][3]));
            }
#pragma unroll
            for (int dd = 0; dd < DP / 16; dd++) {
                uint32_t v[4];
                const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * dd + ((lane >> 3) & 1);
                ldsm4_t(vb + r * DP * 2 + ((c ^ (r & 7)) * 16), v);
#pragma unroll
                for (int n = 0; n < NG; n++) mma<T>(acc[n * (DP / 16) + dd], v, pt[n][0], pt[n][1]);
            }
        } else {
            // scores: lane = key (16) x half of the dims, 8 heads each
            const int r = lane & 15, half = lane >> 4;
            float s[8];
#pragma unroll
            for (int h = 0; h < 8; h++) s[h] = 0.f;
            const float *q = reinterpret_cast<const float *>(sq + buf * S::kQ);
            const float *kr = reinterpret_cast<const float *>(ring + warp * R::kStages * R::kStage + (x % R::kStages) * R::kStage);
#pragma unroll 4
            for (int c = 0; c < CH / 2; c++) {
                const int cc = half * (CH / 2) + c;
                const float4 kx = *reinterpret_cast<const float4 *>(kr + r * DP + ((cc ^ (r & 7)) * 4));
#pragma unroll
                for (int h = 0; h < 8; h++) {
                    const float4 qx = *reinterpret_cast<const float4 *>(q + h * DP + cc * 4);
                    s[h] = fmaf(kx.x, qx.x, s[h]);
                    s[h] = fmaf(kx.y, qx.y, s[h]);
                    s[h] = fmaf(kx.z, qx.z, s[h]);
                    s[h] = fmaf(kx.w, qx.w, s[h]);
                }
            }
            const bool see = visible(j + r, p, it.len, it.pre, a.window);
            float *wt = sw + warp * 8 * kKeys;
#pragma unroll
            for (int h = 0; h < 8; h++) {
                s[h] += __shfl_xor_sync(0xffffffffu, s[h], 16);
                const float slope = a.slopes && h < ng ? __ldg(a.slopes + head0 + h) : 0.f;
                const float z = see ? score2(a, s[h], slope, p, j + r) : -INFINITY;
                const float mn = fmaxf(m[h], mb::warp_max(z)), ms = mn == -INFINITY ? 0.f : mn;
                const float f = exp2f(m[h] - ms), e = exp2f(z - ms);
                m[h] = mn;
                l[h] = fmaf(l[h], f, e);  // every key counts in two lanes
#pragma unroll
                for (int i = 0; i < 4; i++) acc[h][i] *= f;
                if (!half) wt[h * kKeys + r] = e;
            }
            __syncwarp();
            // outputs: a lane holds 4 dims; with 64 dims the half-warps take 8 keys each
            const float *vr = kr + R::kHalf / 4;
            constexpr int KK = DP == 128 ? kKeys : kKeys / 2;
            const int c = DP == 128 ? lane : lane & 15, k0 = DP == 128 ? 0 : half * KK;
#pragma unroll
            for (int g = 0; g < KK / 4; g++) {
                float4 v[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = k0 + 4 * g + i;
                    v[i] = *reinterpret_cast<const float4 *>(vr + row * DP + ((c ^ (row & 7)) * 4));
                }
#pragma unroll
                for (int h = 0; h < 8; h++) {
                    const float4 e = *reinterpret_cast<const float4 *>(wt + h * kKeys + k0 + 4 * g);
                    const float ew[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        acc[h][0] = fmaf(ew[i], v[i].x, acc[h][0]);
                        acc[h][1] = fmaf(ew[i], v[i].y, acc[h][1]);
                        acc[h][2] = fmaf(ew[i], v[i].z, acc[h][2]);
                        acc[h][3] = fmaf(ew[i], v[i].w, acc[h][3]);
                    }
                }
            }
            __syncwarp();
        }

        const bool last = it.i == it.t.n - 1;
        if (last || x == tiles - 1) {
            // the four warps' (m, l, output) into one, in the order of the warps
            float *st = stat + buf * kWarps * H * 2;
            if constexpr (!F32) {
#pragma unroll
                for (int i = 0; i < 2 * NG; i++) {
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
                    if (lane < 4) {
                        const int h = (i / 2) * 8 + 2 * lane + (i & 1);
                        st[(warp * H + h) * 2] = m[i];
                        st[(warp * H + h) * 2 + 1] = l[i];
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < 8; h++) {
                    l[h] = mb::warp_sum(l[h]) * 0.5f;
                    if (DP == 64) {
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[h][i] += __shfl_xor_sync(0xffffffffu, acc[h][i], 16);
                    }
                    if (lane == h) {
                        st[(warp * H + h) * 2] = m[h];
                        st[(warp * H + h) * 2 + 1] = l[h];
                    }
                }
            }
            __syncthreads();
            auto joined = [&](int h, float *M, float *L) {
                *M = -INFINITY;
                *L = 0.f;
#pragma unroll
                for (int i = 0; i < kWarps; i++) *M = fmaxf(*M, st[(i * H + h) * 2]);
#pragma unroll
                for (int i = 0; i < kWarps; i++)
                    *L = fmaf(st[(i * H + h) * 2 + 1], exp2f(st[(i * H + h) * 2] - (*M == -INFINITY ? 0.f : *M)), *L);
            };
            const bool whole = began && last;
            float *part = a.part + ((size_t)blockIdx.x * 2 + (began ? 1 : 0)) * ((size_t)H * (DP + 2));
#pragma unroll
            for (int n = 0; n < NG; n++) {
                float *mine = merge + (warp ? warp - 1 : 0) * 8 * S::kPad;
                if constexpr (!F32) {
                    float f[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float M, L;
                        joined(n * 8 + 2 * (lane & 3) + e, &M, &L);
                        f[e] = exp2f(m[2 * n + e] - (M == -INFINITY ? 0.f : M));
                    }
#pragma unroll
                    for (int dd = 0; dd < DP / 16; dd++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float &y = acc[n * (DP / 16) + dd][e];
                            y *= f[e & 1];
                            if (warp) mine[(2 * (lane & 3) + (e & 1)) * S::kPad + dd * 16 + (lane >> 2) + (e >> 1) * 8] = y;
                        }
                } else {
#pragma unroll
                    for (int h = 0; h < 8; h++) {
                        float M, L;
                        joined(h, &M, &L);
                        const float f = exp2f(m[h] - (M == -INFINITY ? 0.f : M));
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[h][i] *= f;
                        if (warp && lane * 4 < DP)
                            *reinterpret_cast<float4 *>(mine + h * S::kPad + lane * 4) = make_float4(acc[h][0], acc[h][1], acc[h][2], acc[h][3]);
                    }
                }
                __syncthreads();
                if (warp == 0) {
                    if constexpr (!F32) {
#pragma unroll
                        for (int dd = 0; dd < DP / 16; dd++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int at = (2 * (lane & 3) + (e & 1)) * S::kPad + dd * 16 + (lane >> 2) + (e >> 1) * 8;
                                float y = acc[n * (DP / 16) + dd][e];
#pragma unroll
                                for (int i = 0; i < 3; i++) y += merge[i * 8 * S::kPad + at];
                                merge[at] = y;
                            }
                    } else if (lane * 4 < DP) {
#pragma unroll
                        for (int h = 0; h < 8; h++) {
                            float4 y = make_float4(acc[h][0], acc[h][1], acc[h][2], acc[h][3]);
#pragma unroll
                            for (int i = 0; i < 3; i++) {
                                const float4 z = *reinterpret_cast<const float4 *>(merge + (i * 8 + h) * S::kPad + lane * 4);
                                y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
                            }
                            *reinterpret_cast<float4 *>(merge + h * S::kPad + lane * 4) = y;
                        }
                    }
                }
                __syncthreads();
                for (int e = tid; e < 8 * (DP / 4); e += kThreads) {
                    const int hl = e / (DP / 4), c = e % (DP / 4), h = n * 8 + hl;
                    if (h >= ng) break;
                    float4 y = *reinterpret_cast<const float4 *>(merge + hl * S::kPad + c * 4);
                    float M, L;
                    joined(h, &M, &L);
                    if (whole) {
                        const float inv = L == 0.f ? 0.f : 1.f / L;
                        if (c * 4 < a.d)
                            store4(reinterpret_cast<T *>(a.out) + it.seq * a.o_row + (head0 + h) * a.o_head + c * 4,
                                   make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
                        if (a.lse && c == 0)
                            a.lse[(long long)it.seq * a.heads + head0 + h] = L == 0.f ? -INFINITY : ((M == -INFINITY ? 0.f : M) + log2f(L)) * kLn2;
                    } else {
                        *reinterpret_cast<float4 *>(part + (size_t)h * DP + c * 4) = y;
                        if (c == 0) {
                            part[(size_t)H * DP + 2 * h] = M;
                            part[(size_t)H * DP + 2 * h + 1] = L;
                        }
                    }
                }
                if (n + 1 < NG) __syncthreads();  // the merge buffers are written again
            }
            if (x == tiles - 1 && tid == 0) {
                Meta mt{};
                mt.c_end = -1;
                if (began && !last) {
                    mt.c_end = (int)div64(end - 1 + (it.t.n - 1 - it.i), per);
                    mt.row0 = it.seq;
                    mt.ntok = 1;
                    mt.head0 = head0;
                    mt.ng = ng;
                    mt.seq = it.seq;
                    mt.pos0 = p;
                }
                a.meta[blockIdx.x] = mt;
            }
            began = true;
            fresh = true;
            buf ^= 1;
        }
        it.next(a, hh_n);
    }
    cp_wait<0>();
}

template <typename T, int DP, int NG>
int run(Work &w, int ctas, cudaStream_t s)
{
    const char *who = "mocha_kv_decode";
    constexpr int smem = Smem<T, DP, NG>::kTotal;
    if (launch(who, k_decode<T, DP, NG>, dim3(ctas), kThreads, smem, s, false, w)) return 1;
    return launch(who, k_join<T, false>, dim3(2 * mb::kSMs), 32 * kJoinWarps, 0, s, true, w.a, ctas, 8 * NG, DP);
}

template <typename T, int DP>
int run_ng(Work &w, int ng, int ctas, cudaStream_t s)
{
    if constexpr (sizeof(T) == 4) return run<T, DP, 1>(w, ctas, s);
    else return ng == 1 ? run<T, DP, 1>(w, ctas, s) : ng == 2 ? run<T, DP, 2>(w, ctas, s) : run<T, DP, 4>(w, ctas, s);
}

template <typename T>
int run_dp(Work &w, int dp, int ng, int ctas, cudaStream_t s)
{
    return dp == 64 ? run_ng<T, 64>(w, ng, ctas, s) : run_ng<T, 128>(w, ng, ctas, s);
}

// Heads of a unit in eights: all of a group up to 32 (16-bit), 8 (fp32, where a group's
// further heads read the keys again, from L2).
int head_groups(int type, int group)
{
    if (type == MOCHA_KV_F32 || group <= 8) return 1;
    return group <= 16 ? 2 : 4;
}

int cta_count(int type, int ng, int dp)
{
    return mb::kSMs * ((type == MOCHA_KV_F32 && dp == 128) || ng > 1 ? 1 : 2);
}

}  // namespace

namespace kv {
size_t decode_workspace(int type, int group, int d)
{
    const int ng = head_groups(type, group), dp = padded_dim(d), ctas = cta_count(type, ng, dp);
    return meta_bytes(ctas) + part_bytes(ctas, 8 * ng, dp);
}
}  // namespace kv

extern "C" int mocha_kv_decode(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores,
                               const mocha_kv_rows *q, const mocha_kv_rows *out, float *lse, void *workspace,
                               unsigned long long workspace_bytes, void *stream)
{
    const char *who = "mocha_kv_decode";
    if (check_pages(who, pages) || check_seqs(who, seqs) || check_scores(who, pages, scores)) return 1;
    const int b = type_bytes(pages->type), d = pages->head_dim;
    if (check_rows(who, "q", q, b, d, seqs->seqs) || check_rows(who, "out", out, b, d, seqs->seqs)) return 1;
    if (seqs->seqs && !seqs->kv_len) return fail(who, "null kv_len");
    DeviceGuard guard;
    if (guard.enter(who, pages->device)) return 1;
    if (!seqs->seqs) return 0;
    Work w{};
    w.a = make_args(pages, seqs, scores, q, out, lse);
    if (!workspace || !aligned(workspace) || workspace_bytes < decode_workspace(pages->type, w.a.group, d))
        return fail(who, "workspace missing, not 16-byte aligned or smaller than mocha_kv_workspace says");
    const int ng = head_groups(pages->type, w.a.group), dp = padded_dim(d), ctas = cta_count(pages->type, ng, dp);
    w.unit_heads = 8 * ng;
    w.hgroups = (w.a.group + w.unit_heads - 1) / w.unit_heads;
    w.min_tiles = 2;
    w.a.meta = static_cast<Meta *>(workspace);
    w.a.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + meta_bytes(ctas));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return pages->type == MOCHA_KV_F32   ? run_dp<float>(w, dp, ng, ctas, s)
           : pages->type == MOCHA_KV_F16 ? run_dp<__half>(w, dp, ng, ctas, s)
                                         : run_dp<__nv_bfloat16>(w, dp, ng, ctas, s);
}
