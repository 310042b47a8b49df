"""HIP kernel source generators for operators of language models: rotary positions, a key/value cache
held in 8 bits with the attention that reads it, and the adjustment of logits.

Same conventions as hip_kernel.py: every function returns `(source, kernel_name, argfmt)`, kernels are
specialised by layout class and sizes are runtime arguments.
"""
from __future__ import annotations

from functools import cache

from dlgrad_amd.codegen.hip_kernel import PRELUDE, _fmt

# =====================================================================================
# rotary positions
# =====================================================================================

ROTARY_HEADS = 4            # heads a thread turns with one evaluation of the angles

_ANGLES = r"""
// sin and cos of 2 pi t / 2^32 for a 32-bit turn t.  The two top bits (after rounding) are the quadrant; what is left lies
// within an eighth of a turn, where the Taylor series end at x^9 / 9! and x^10 / 10! with less than 2e-9 left over.
static __device__ __forceinline__ void turn_sincos(u32 t, float& s, float& c) {
    const u32 quad = (t + 0x20000000u) >> 30;
    const float x = (float)(int)(t - (quad << 30)) * 1.46291807926715968e-9f;          // 2 pi / 2^32
    const float z = x * x;
    const float ss = x + x * z * (-1.6666667e-1f + z * (8.3333333e-3f + z * (-1.9841270e-4f + z * 2.7557319e-6f)));
    const float cc = 1.0f + z * (-0.5f + z * (4.1666667e-2f + z * (-1.3888889e-3f + z * (2.4801587e-5f + z * -2.7557319e-7f))));
    const float a = (quad & 1u) ? cc : ss, b = (quad & 1u) ? ss : cc;
    s = (quad & 2u) ? -a : a;
    c = ((quad + 1u) & 2u) ? -b : b;
}
// the top 32 bits of p * f mod 2^64: position p (whole, of either sign) times a frequency in turns of 2^-64
static __device__ __forceinline__ u32 turn_of(int p, u64 f) {
    return (u32)(((u64)(long long)p * f) >> 32);
}
"""


@cache
def rotary_kernel(half: bool, vec: bool) -> tuple[str, str, str]:
    """y = x with the first `rot` of the d elements of every head turned pair by pair: (a, b) becomes
    gain * (a cos w - b sin w, a sin w + b cos w) with w = position * frequency of the pair, the other elements
    copied.  half: pair i is elements i and i + rot / 2; otherwise 2 i and 2 i + 1.  back = 1 turns by -w, which
    is the transposed map: it takes the gradient of y to the gradient of x.

    Angles.  A position times a frequency in radians loses everything in 32 bits at far positions (2^17 * 1 rad has
    a step of 2^-7).  Here a frequency is the fraction of a turn per position in 64-bit fixed point, and the product
    modulo 2^64 is the angle modulo one turn, exactly, for whole positions below 2^24 in magnitude; no table of
    cosines is stored or read.

    Rows of H heads lie `pitch` floats apart (x and y may be the same memory: a thread reads what it writes before it
    writes it).  A thread takes one group of pairs (vec: 16-byte accesses; 4 pairs with half, 2 without) of up to
    four heads, H / 4 apart so that neighbouring lanes touch neighbouring heads: the loads are issued first and the
    angles, once for all four heads, are computed while they are in flight.  grid.z = 2 turns a second tensor
    (keys beside queries) in the same launch.  Bound by memory: 8 bytes an element."""
    name = f"rotary_{'half' if half else 'pairs'}_{'v4' if vec else 'v1'}"
    W = (4 if half else 2) if vec else 1                 # pairs of a rotating unit
    if half:
        load = ("const float4 a = *reinterpret_cast<const float4*>(xr + off + j), b = *reinterpret_cast<const float4*>(xr + off + hr + j);"
                if vec else "const float a = xr[off + j], b = xr[off + hr + j];")
        keep = ("va[n][0] = a.x; va[n][1] = a.y; va[n][2] = a.z; va[n][3] = a.w; vb[n][0] = b.x; vb[n][1] = b.y; vb[n][2] = b.z; vb[n][3] = b.w;"
                if vec else "va[n][0] = a; vb[n][0] = b;")
        store = ("*reinterpret_cast<float4*>(yr + off + j) = make_float4(oa[0], oa[1], oa[2], oa[3]); "
                 "*reinterpret_cast<float4*>(yr + off + hr + j) = make_float4(ob[0], ob[1], ob[2], ob[3]);"
                 if vec else "yr[off + j] = oa[0]; yr[off + hr + j] = ob[0];")
    else:
        load = ("const float4 a = *reinterpret_cast<const float4*>(xr + off + 2u * j);" if vec
                else "const float a = xr[off + 2u * j], b = xr[off + 2u * j + 1u];")
        keep = ("va[n][0] = a.x; vb[n][0] = a.y; va[n][1] = a.z; vb[n][1] = a.w;" if vec else "va[n][0] = a; vb[n][0] = b;")
        store = ("*reinterpret_cast<float4*>(yr + off + 2u * j) = make_float4(oa[0], ob[0], oa[1], ob[1]);" if vec
                 else "yr[off + 2u * j] = oa[0]; yr[off + 2u * j + 1u] = ob[0];")
    copy = ("*reinterpret_cast<float4*>(yr + off + c) = *reinterpret_cast<const float4*>(xr + off + c);" if vec else "yr[off + c] = xr[off + c];")
    CW = 4 if vec else 1
    src = f"""{PRELUDE}{_ANGLES}
extern "C" __global__ __launch_bounds__(256) void {name}(const float* x0, float* y0, const float* x1, float* y1,
        const u64* __restrict__ freq, const float* __restrict__ pos, const float* __restrict__ start,
        u32 rows, u32 T, u32 per, u32 H0, u32 H1, u32 d, u32 rot, u32 xp0, u32 xp1, u32 yp0, u32 yp1,
        u32 pos_step, u32 start_step, u32 back, float gain) {{
    const bool second = blockIdx.z != 0u;
    const float* x = second ? x1 : x0;
    float* y = second ? y1 : y0;
    const u32 H = second ? H1 : H0, HG = (H + {ROTARY_HEADS - 1}u) / {ROTARY_HEADS}u;
    const u32 hr = rot >> 1, UR = hr / {W}u, U = UR + (x == y ? 0u : (d - rot) / {CW}u);
    const u64 item = (u64)blockIdx.x * 256u + threadIdx.x;
    if (item >= (u64)rows * HG * U) return;
    const u32 u = (u32)(item % U);
    const u64 rest = item / U;
    const u32 hg = (u32)(rest % HG), row = (u32)(rest / HG);
    const float* xr = x + (u64)row * (second ? xp1 : xp0);
    float* yr = y + (u64)row * (second ? yp1 : yp0);
    if (u >= UR) {{                                                // elements that do not turn
        const u32 c = rot + (u - UR) * {CW}u;
        #pragma unroll
        for (u32 n = 0; n < {ROTARY_HEADS}u; ++n) {{
            const u32 off = (hg + n * HG) * d;
            if (hg + n * HG < H) {{ {copy} }}
        }}
        return;
    }}
    const u32 j = u * {W}u;
    float va[{ROTARY_HEADS}][{W}], vb[{ROTARY_HEADS}][{W}];
    #pragma unroll
    for (u32 n = 0; n < {ROTARY_HEADS}u; ++n) {{
        const u32 off = min(hg + n * HG, H - 1u) * d;
        {load}
        {keep}
    }}
    const u32 t = row % T, b = row / T / per;
    const int p = (pos ? (int)pos[(u64)b * pos_step + t] : (int)t) + (start ? (int)start[(u64)b * start_step] : 0);
    float sn[{W}], cs[{W}];
    #pragma unroll
    for (u32 i = 0; i < {W}u; ++i) {{
        turn_sincos(turn_of(p, freq[j + i]), sn[i], cs[i]);
        cs[i] *= gain;
        sn[i] *= back ? -gain : gain;
    }}
    #pragma unroll
    for (u32 n = 0; n < {ROTARY_HEADS}u; ++n) {{
        if (hg + n * HG >= H) break;
        const u32 off = (hg + n * HG) * d;
        float oa[{W}], ob[{W}];
        #pragma unroll
        for (u32 i = 0; i < {W}u; ++i) {{
            oa[i] = va[n][i] * cs[i] - vb[n][i] * sn[i];
            ob[i] = va[n][i] * sn[i] + vb[n][i] * cs[i];
        }}
        {store}
    }}
}}
"""
    return src, name, _fmt("P" * 7, "I" * 14, "f")


# =====================================================================================
# logits
# =====================================================================================

@cache
def adjust_logits_kernel(items: int, vec: bool) -> tuple[str, str, str]:
    """y = logits (B, V) with what has been said already made less likely, a bias added and forbidden tokens removed:
    for a token that occurs c > 0 times among the first lengths[b] entries of history[b],
      x = x / repetition if x > 0 else x * repetition, then x - (presence + frequency * c);
    then + bias[v]; then -inf where hidden > 0 (whatever stood there, a NaN included).  Entries of the history outside
    [0, V) count for nothing.  Each of the three penalties is a number, or an array with one per row.

    A block owns 256 * items consecutive tokens of one row and counts only those: their counters lie in LDS, every
    block walks the whole history of its row (which stays in L2: 4 bytes an entry) and bumps the counters of its own
    tokens with integer atomics, whose order does not matter.  So there is one launch, no count array in memory and
    no sort.  The logits are loaded before the walk and used after it.  vec: 16-byte accesses (V % 4 == 0)."""
    assert items in (4, 8, 16, 32)
    name = f"adjust_logits_i{items}_{'v4' if vec else 'v1'}"
    W = 4 if vec else 1
    NV = items // W
    if vec:
        load = "const float4 t4 = *reinterpret_cast<const float4*>(lrow + v); x[k][0] = t4.x; x[k][1] = t4.y; x[k][2] = t4.z; x[k][3] = t4.w;"
        bload = "const float4 t4 = *reinterpret_cast<const float4*>(brow + v); x[k][0] += t4.x; x[k][1] += t4.y; x[k][2] += t4.z; x[k][3] += t4.w;"
        hload = ("const float4 t4 = *reinterpret_cast<const float4*>(hrow + v); x[k][0] = t4.x > 0.0f ? NINF : x[k][0]; x[k][1] = t4.y > 0.0f ? NINF : x[k][1]; "
                 "x[k][2] = t4.z > 0.0f ? NINF : x[k][2]; x[k][3] = t4.w > 0.0f ? NINF : x[k][3];")
        store = "*reinterpret_cast<float4*>(yrow + v) = make_float4(x[k][0], x[k][1], x[k][2], x[k][3]);"
    else:
        load, bload = "x[k][0] = lrow[v];", "x[k][0] += brow[v];"
        hload, store = "if (hrow[v] > 0.0f) x[k][0] = NINF;", "yrow[v] = x[k][0];"
    src = f"""{PRELUDE}
#define NINF (-__builtin_inff())
#define SLICE {256 * items}u
extern "C" __global__ __launch_bounds__(256) void {name}(const float* __restrict__ logits, const float* __restrict__ history,
        const float* __restrict__ lengths, const float* __restrict__ bias, const float* __restrict__ hidden, float* __restrict__ y,
        const float* __restrict__ rep_p, const float* __restrict__ pre_p, const float* __restrict__ fre_p,
        u32 V, u32 L, u32 bias_step, u32 hidden_step, float rep, float pre, float fre) {{
    __shared__ u32 count[SLICE];
    const u32 t = threadIdx.x, v0 = blockIdx.x * SLICE;
    const u64 b = blockIdx.y;
    const float* __restrict__ lrow = logits + b * V;
    float* __restrict__ yrow = y + b * V;
    float x[{NV}][{W}];
    #pragma unroll
    for (u32 k = 0; k < {NV}u; ++k) {{
        const u32 v = v0 + (k * 256u + t) * {W}u;
        if (v < V) {{ {load} }}
    }}
    u32 n = 0u;
    if (L) {{
        const float ln = lengths ? lengths[b] : (float)L;
        n = ln >= (float)L ? L : ln > 0.0f ? (u32)ln : 0u;                   // (a NaN counts nothing)
        for (u32 k = t; k < SLICE; k += 256u) count[k] = 0u;
        __syncthreads();
        const float* __restrict__ said = history + b * L;
        #pragma unroll 4
        for (u32 k = t; k < n; k += 256u) {{
            const float id = said[k];
            if (id >= (float)v0 && id < 4294967040.0f) {{
                const u32 at = (u32)id - v0;
                if (at < SLICE) atomicAdd(&count[at], 1u);
            }}
        }}
        __syncthreads();
    }}
    if (n) {{
        const float r = rep_p ? rep_p[b] : rep, p = pre_p ? pre_p[b] : pre, f = fre_p ? fre_p[b] : fre;
        #pragma unroll
        for (u32 k = 0; k < {NV}u; ++k) {{
            #pragma unroll
            for (u32 i = 0; i < {W}u; ++i) {{
                const u32 c = count[(k * 256u + t) * {W}u + i];
                if (c) x[k][i] = (x[k][i] > 0.0f ? x[k][i] / r : x[k][i] * r) - (p + f * (float)c);
            }}
        }}
    }}
    if (bias) {{
        const float* __restrict__ brow = bias + b * bias_step;
        #pragma unroll
        for (u32 k = 0; k < {NV}u; ++k) {{ const u32 v = v0 + (k * 256u + t) * {W}u; if (v < V) {{ {bload} }} }}
    }}
    if (hidden) {{
        const float* __restrict__ hrow = hidden + b * hidden_step;
        #pragma unroll
        for (u32 k = 0; k < {NV}u; ++k) {{ const u32 v = v0 + (k * 256u + t) * {W}u; if (v < V) {{ {hload} }} }}
    }}
    #pragma unroll
    for (u32 k = 0; k < {NV}u; ++k) {{ const u32 v = v0 + (k * 256u + t) * {W}u; if (v < V) {{ {store} }} }}
}}
"""
    return src, name, _fmt("P" * 9, "I" * 4, "fff")


# =====================================================================================
# the 8-bit key/value cache
# =====================================================================================

CACHE8_BLOCK = 64           # tokens of one head that share a scale
CACHE8_MAX_D = 256


def cache8_width(d: int) -> int:
    """Columns a head of d is held in: a multiple of 32, the k extent of one matrix instruction."""
    return (d + 31) // 32 * 32


_CACHE8 = r"""
// Tokens of sequence b before this call, and the rows of it that the call brings; both within what the cache holds.
static __device__ __forceinline__ void cache8_extent(const float* __restrict__ lengths, const float* __restrict__ counts, u32 b, u32 T, u32 cap,
                                                     u32& len, u32& n) {
    const float l = lengths[b], c = counts ? counts[b] : (float)T;
    len = l >= (float)cap ? cap : l > 0.0f ? (u32)l : 0u;
    n = c >= (float)T ? T : c > 0.0f ? (u32)c : 0u;
    n = min(n, cap - len);
}
"""


@cache
def cache8_write_kernel(DP: int, vec: bool) -> tuple[str, str, str]:
    """New key and value rows k, v (B, T, H * d) into the 8-bit cache of one layer, at positions lengths[b] .. of each sequence
    (the first counts[b] rows of each, all T without counts; rows that the cache has no room for are dropped).

    A block of 64 tokens of one head is quantised when its last token arrives, and never again: scale = max |x| / 127
    in 32 bits, code = x / scale to the nearest whole number, ties to even.  Until then its rows stay fp32 in the tail, so what
    the cache holds depends on the tokens alone and not on the calls that brought them.  Key codes lie as [64][DP] bytes, value
    codes transposed, [DP][64], each code + 128; two tails of 64 rows per head, block i's in tail i & 1.

    The quotient is rounded exactly: q = rint(x * (1 / scale)) may be off by one next to a half, and x - q * scale is
    representable (both are multiples of the unit of the smaller one, and it is below two scales), so one fused
    multiply-add gives it without error and the comparison with half a scale decides.

    A row that holds a NaN or an infinity is kept as NaN in the tail, and a block with such a row gets NaN for its scales:
    every output that sees it is NaN, and the codes stay whole numbers.

    One workgroup of 256 threads per (block of 64, head, sequence); a thread holds 4 tokens by 4 columns of keys and values
    at a time.  Workgroup 0 of a head completes the block that the call starts in and then stores the rows of the block it
    ends in, in this order, because both may use the same tail.  Bound by memory: 4 bytes read and 1 written per element."""
    name = f"cache8_write_d{DP}_{'v4' if vec else 'v1'}"
    IT = (DP + 63) // 64                     # items of 4 tokens by 4 columns per thread
    ld = ("const float4 f = *reinterpret_cast<const float4*>(src + c0);" if vec else
          "const float4 f = make_float4(c0 < d ? src[c0] : 0.0f, c0 + 1u < d ? src[c0 + 1u] : 0.0f, c0 + 2u < d ? src[c0 + 2u] : 0.0f, c0 + 3u < d ? src[c0 + 3u] : 0.0f);")
    src = f"""{PRELUDE}{_CACHE8}
#define DP {DP}u
#define C4 {DP // 4}u
static __device__ __forceinline__ u32 code_of(float x, float s, float inv) {{
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), r2 = 2.0f * fabsf(r);
    if (r2 > s || (r2 == s && ((int)q & 1))) q += r < 0.0f ? -1.0f : 1.0f;
    return (u32)((int)fminf(fmaxf(q, -127.0f), 127.0f) + 128);
}}
static __device__ __forceinline__ bool odd_one(float x) {{ return !(fabsf(x) < __builtin_inff()); }}
extern "C" __global__ __launch_bounds__(256) void {name}(const float* __restrict__ k, const float* __restrict__ v,
        const float* __restrict__ lengths, const float* __restrict__ counts,
        unsigned char* __restrict__ kc, unsigned char* __restrict__ vc, float* __restrict__ scales, float* tail_k, float* tail_v,
        u32 T, u32 H, u32 d, u32 NB, u32 kp, u32 vp) {{
    __shared__ __attribute__((aligned(16))) u32 vt[DP * 16u];       // value codes of the block, [DP][64] bytes
    __shared__ float sk[4], sv[4];
    __shared__ u32 bad[64];
    const u32 t = threadIdx.x, lane = t & 63u, h = blockIdx.y, b = blockIdx.z;
    u32 len, n;
    cache8_extent(lengths, counts, b, T, NB * 64u, len, n);
    if (!n) return;
    const u32 total = len + n, first = len >> 6, last = total >> 6;         // last: the block that is not full afterwards
    const u64 bh = (u64)b * H + h, heads = (u64)gridDim.z * H;
    const float* __restrict__ kh = k + (u64)b * T * kp + (u64)h * d;
    const float* __restrict__ vh = v + (u64)b * T * vp + (u64)h * d;
    for (u32 pass = 0; pass < 2u; ++pass) {{
        const u32 blk = pass ? last : first + blockIdx.x;
        if (pass && (blockIdx.x != 0u || last == first)) break;            // (uniform over the workgroup)
        const bool full = blk < last;
        if (!pass && !full && blk != first) break;
        if (blk >= NB) break;
        float* tk = tail_k + (((u64)(blk & 1u) * heads + bh) * 64u) * DP;
        float* tv = tail_v + (((u64)(blk & 1u) * heads + bh) * 64u) * DP;
        const u32 lo = blk == first ? (len & 63u) : 0u, hi = full ? 64u : (total & 63u);       // new rows of this block
        if (t < 64u) bad[t] = 0u;
        __syncthreads();
        float xk[{IT}][4][4], xv[{IT}][4][4];
        float mk = 0.0f, mv = 0.0f;
        #pragma unroll
        for (u32 it = 0; it < {IT}u; ++it) {{
            const u32 item = it * 256u + t, c0 = (item % C4) * 4u, tq = item / C4;
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) {{
                const u32 row = tq * 4u + i;
                float4 fk = make_float4(0.f, 0.f, 0.f, 0.f), fv = fk;
                if (tq < 16u && row < hi) {{
                    if (row < lo) {{                                           // from the tail (only the block the call starts in)
                        if (full) {{
                            fk = *reinterpret_cast<const float4*>(tk + row * DP + c0);
                            fv = *reinterpret_cast<const float4*>(tv + row * DP + c0);
                        }}
                    }} else if (c0 < d) {{
                        const u64 at = (u64)blk * 64u + row - len;
                        {{ const float* __restrict__ src = kh + at * kp; {ld} fk = f; }}
                        {{ const float* __restrict__ src = vh + at * vp; {ld} fv = f; }}
                    }}
                    if (odd_one(fk.x) || odd_one(fk.y) || odd_one(fk.z) || odd_one(fk.w) || odd_one(fv.x) || odd_one(fv.y) || odd_one(fv.z) || odd_one(fv.w))
                        bad[row] = 1u;
                }}
                xk[it][i][0] = fk.x; xk[it][i][1] = fk.y; xk[it][i][2] = fk.z; xk[it][i][3] = fk.w;
                xv[it][i][0] = fv.x; xv[it][i][1] = fv.y; xv[it][i][2] = fv.z; xv[it][i][3] = fv.w;
                mk = fmaxf(mk, fmaxf(fmaxf(fabsf(fk.x), fabsf(fk.y)), fmaxf(fabsf(fk.z), fabsf(fk.w))));
                mv = fmaxf(mv, fmaxf(fmaxf(fabsf(fv.x), fabsf(fv.y)), fmaxf(fabsf(fv.z), fabsf(fv.w))));
            }}
        }}
        mk = wave_max(mk);
        mv = wave_max(mv);
        if (lane == 0u) {{ sk[t >> 6] = mk; sv[t >> 6] = mv; }}
        __syncthreads();
        // the rows as they came: needed while the block is not full (and again if the caller goes back into it)
        if (!full || (blk == first && last == first + 1u)) {{
            #pragma unroll
            for (u32 it = 0; it < {IT}u; ++it) {{
                const u32 item = it * 256u + t, c0 = (item % C4) * 4u, tq = item / C4;
                #pragma unroll
                for (u32 i = 0; i < 4u; ++i) {{
                    const u32 row = tq * 4u + i;
                    if (tq < 16u && row >= lo && row < hi) {{
                        const float z = bad[row] ? __builtin_nanf("") : 0.0f;
                        float4 fk = make_float4(xk[it][i][0], xk[it][i][1], xk[it][i][2], xk[it][i][3]);
                        float4 fv = make_float4(xv[it][i][0], xv[it][i][1], xv[it][i][2], xv[it][i][3]);
                        if (z != z) {{ fk = make_float4(z, z, z, z); fv = fk; }}
                        *reinterpret_cast<float4*>(tk + row * DP + c0) = fk;
                        *reinterpret_cast<float4*>(tv + row * DP + c0) = fv;
                    }}
                }}
            }}
        }}
        if (full) {{
            const bool odd = __any(bad[lane] != 0u);
            const float ak = fmaxf(fmaxf(sk[0], sk[1]), fmaxf(sk[2], sk[3])) / 127.0f, av = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])) / 127.0f;
            const u64 at = bh * NB + blk;
            if (t == 0u) {{
                scales[2u * at] = odd ? __builtin_nanf("") : ak;
                scales[2u * at + 1u] = odd ? __builtin_nanf("") : av;
            }}
            // a scale below 2^-60 has no finite reciprocal or an inexact remainder: both sides times 2^64, exactly
            const float upk = ak < 8.6736174e-19f ? 18446744073709551616.0f : 1.0f, upv = av < 8.6736174e-19f ? 18446744073709551616.0f : 1.0f;
            const float s_k = ak * upk, s_v = av * upv, ik = ak > 0.0f ? 1.0f / s_k : 0.0f, iv = av > 0.0f ? 1.0f / s_v : 0.0f;
            unsigned char* __restrict__ kb = kc + at * (64u * DP);
            #pragma unroll
            for (u32 it = 0; it < {IT}u; ++it) {{
                const u32 item = it * 256u + t, c0 = (item % C4) * 4u, tq = item / C4;
                if (tq < 16u) {{
                    u32 cv[4] = {{0u, 0u, 0u, 0u}};
                    #pragma unroll
                    for (u32 i = 0; i < 4u; ++i) {{
                        u32 ck = 0u;
                        #pragma unroll
                        for (u32 c = 0; c < 4u; ++c) {{
                            ck |= ((ak > 0.0f && !odd) ? code_of(xk[it][i][c] * upk, s_k, ik) : 128u) << (8u * c);
                            cv[c] |= ((av > 0.0f && !odd) ? code_of(xv[it][i][c] * upv, s_v, iv) : 128u) << (8u * i);
                        }}
                        *reinterpret_cast<u32*>(kb + (tq * 4u + i) * DP + c0) = ck;
                    }}
                    #pragma unroll
                    for (u32 c = 0; c < 4u; ++c) vt[(c0 + c) * 16u + tq] = cv[c];
                }}
            }}
            __syncthreads();
            uint4* __restrict__ vb = reinterpret_cast<uint4*>(vc + at * (64u * DP));
            for (u32 i = t; i < DP * 4u; i += 256u) vb[i] = reinterpret_cast<const uint4*>(vt)[i];
        }}
        __syncthreads();
    }}
}}
"""
    return src, name, _fmt("P" * 9, "I" * 6)


@cache
def cache8_read_kernel(DP: int) -> tuple[str, str, str]:
    """The values that the cache of one layer stands for, as fp32 k and v (B, N, H * d): code * scale for the tokens of full
    blocks, the rows themselves for those of the tail, zeros from position lengths[b] + counts[b] on (counts: rows written
    since the lengths were advanced; `extra` for every sequence without them).  One workgroup per (block of 64, head,
    sequence); value codes are transposed through LDS so that rows leave as rows.  Bound by memory."""
    name = f"cache8_read_d{DP}"
    src = f"""{PRELUDE}{_CACHE8}
#define DP {DP}u
extern "C" __global__ __launch_bounds__(256) void {name}(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
        const float* __restrict__ scales, const float* __restrict__ tail_k, const float* __restrict__ tail_v,
        const float* __restrict__ lengths, const float* __restrict__ counts, float* __restrict__ ko, float* __restrict__ vo,
        u32 N, u32 H, u32 d, u32 NB, u32 extra) {{
    __shared__ __attribute__((aligned(16))) u32 vt[DP * 17u];               // rows of 64 bytes, 68 apart
    const u32 t = threadIdx.x, blk = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    u32 len, n;
    cache8_extent(lengths, counts, b, extra, NB * 64u, len, n);
    const u32 total = len + n, last = total >> 6;
    const u64 bh = (u64)b * H + h, heads = (u64)gridDim.z * H, at = bh * NB + blk;
    const float s_k = blk < last ? scales[2u * at] : 0.0f, s_v = blk < last ? scales[2u * at + 1u] : 0.0f;
    const unsigned char* __restrict__ kb = kc + at * (64u * DP);
    if (blk < last) {{
        const u32* __restrict__ vb = reinterpret_cast<const u32*>(vc + at * (64u * DP));
        for (u32 i = t; i < DP * 16u; i += 256u) vt[(i >> 4) * 17u + (i & 15u)] = vb[i];
    }}
    __syncthreads();
    const float* __restrict__ tk = tail_k + (((u64)(blk & 1u) * heads + bh) * 64u) * DP;
    const float* __restrict__ tv = tail_v + (((u64)(blk & 1u) * heads + bh) * 64u) * DP;
    for (u32 i = t; i < 64u * d; i += 256u) {{
        const u32 row = i / d, c = i % d, p = blk * 64u + row;
        if (p >= N) break;
        float x = 0.0f, y = 0.0f;
        if (blk < last) {{
            x = (float)((int)kb[row * DP + c] - 128) * s_k;
            y = (float)((int)reinterpret_cast<const unsigned char*>(vt)[c * 68u + row] - 128) * s_v;
        }} else if (p < total) {{ x = tk[row * DP + c]; y = tv[row * DP + c]; }}
        const u64 o = ((u64)b * N + p) * ((u64)H * d) + (u64)h * d + c;
        ko[o] = x;
        vo[o] = y;
    }}
}}
"""
    return src, name, _fmt("P" * 9, "I" * 5)


@cache
def cache8_attend_kernel(DP: int) -> tuple[str, str, str]:
    """Attention of T new positions per sequence over the 8-bit cache of one layer, after their keys and values were written:
    y = softmax(q K^T * scale) V per query head, query t of sequence b at position lengths[b] + t seeing the positions up to its
    own; `group` query heads share a key head.  q and y are (B, T, H * group * d).  A row beyond counts[b] gives zeros.

    The codes are whole numbers of at most 127 and therefore exact in 16-bit floats, so the matrix units do the work:
    a query row is scaled by a power of two to at most 2^15 and cut into two 16-bit floats, q' = q1 + q2 (22 bits and more of
    it), and S^T = K (q1 + q2)^T has fp32 accuracy from two v_mfma_f32_16x16x32_f16 per 32 columns.  The probabilities go the
    same way: p' = 2^15 exp(s - m) = p1 + p2, the factor cancels in p' V / sum p'.  The scales enter in 32 bits, the keys'
    with the scores, the values' as a block's product joins the running sum.

    A wavefront takes one block of 64 tokens at a time, with (m, l, O) of its own per query.  Its lane r + 16 g (r, g < 16, 4) holds
    query r and, of every product S^T, four tokens; the rows of K are fed in the order that makes those of the four tiles the
    sixteen neighbours 16 g ..: then P is already the B operand of O^T += V^T P^T, and its A operand, sixteen value codes
    of one column, is one 16-byte load from the transposed block.  Nothing passes through LDS.  Bytes become 16-bit floats in one
    operation each: v_perm puts byte c under the exponent of 1024, giving 1024 + c, and a packed addition takes 1152 away.

    The tail, fp32, is shared out 16 tokens to a wavefront and goes through v_mfma_f32_16x16x4_f32.

    A workgroup of four wavefronts per (16 query rows of one key head, split of the blocks); the four are joined through LDS in
    wavefront order.  With one split y is written; else O, m and l go to `part` and cache8_join_kernel adds the splits up
    in their order.  Bound by memory while few query rows share a key head: 2 bytes per token and column."""
    ND, NK, Q4 = DP // 16, DP // 32, DP // 4             # column tiles of V^T, k steps of a score, columns a lane feeds
    name = f"cache8_attend_d{DP}"
    kw = Q4 // 8                                          # 8-byte words of a key row per lane
    src = f"""{PRELUDE}{_CACHE8}
#define DP {DP}u
#define ND {ND}u
#define NK {NK}u
typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
union H8 {{ h8 v; h2 p[4]; _Float16 e[8]; u32 w[4]; }};
#define MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)
#define MFMA32(a, b, c) __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0)
#define NINF (-__builtin_inff())
// eight codes as 16-bit floats
static __device__ __forceinline__ h8 widen(u32 lo, u32 hi) {{
    H8 r;
    const h2 off = {{(_Float16)-1152.0f, (_Float16)-1152.0f}};
    r.w[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
    r.w[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
    r.w[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
    r.w[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
    #pragma unroll
    for (int i = 0; i < 4; ++i) r.p[i] += off;
    return r.v;
}}
extern "C" __global__ __launch_bounds__(256) void {name}(const float* __restrict__ q, const unsigned char* __restrict__ kc,
        const unsigned char* __restrict__ vc, const float* __restrict__ scales, const float* __restrict__ tail_k, const float* __restrict__ tail_v,
        const float* __restrict__ lengths, const float* __restrict__ counts, float* __restrict__ y, float* __restrict__ part,
        u32 B, u32 T, u32 H, u32 group, u32 d, u32 NB, u32 tiles, u32 splits, float scale) {{
    __shared__ float so[4][16][DP + 4u];
    __shared__ float sm[4][16], sl[4][16];
    const u32 t = threadIdx.x, w = t >> 6, lane = t & 63u, r = lane & 15u, g = lane >> 4;
    const u32 split = blockIdx.x % splits, tile = (blockIdx.x / splits) % tiles;
    const u32 bh = blockIdx.x / splits / tiles, b = bh / H, h = bh % H;
    u32 len, n;
    cache8_extent(lengths, counts, b, T, NB * 64u, len, n);
    const u32 rows = T * group, last = (len + n) >> 6;                       // blocks below `last` are codes
    const u32 row = tile * 16u + r, tq = row / group;
    const bool live = row < rows && tq < n;
    const u32 see = live ? len + tq + 1u : 0u;                                 // positions this lane's query sees
    const u32 tile_last = min(min(tile * 16u + 15u, rows - 1u) / group, n ? n - 1u : 0u);
    const u32 most = (n && tile * 16u / group < n) ? len + tile_last + 1u : 0u;               // ... and the last query of the tile
    const u32 least = min(tile * 16u + 15u, rows - 1u) / group < n ? len + tile * 16u / group + 1u : 0u;   // ... and the first (a padded row: none)
    const u64 C = (u64)H * group * d;
    const float* __restrict__ qrow = q + ((u64)b * T + tq) * C + (u64)(h * group + row % group) * d;
    // this lane's quarter of its query row, as two 16-bit floats an element
    H8 q1[NK], q2[NK];
    float back;
    {{
        float f[{Q4}], mx = 0.0f;
        #pragma unroll
        for (u32 i = 0; i < {Q4}u; ++i) {{
            const u32 c = g * {Q4}u + i;
            f[i] = (live && c < d) ? qrow[c] : 0.0f;
            mx = fmaxf(mx, fabsf(f[i]));
        }}
        mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
        mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE));
        const int e = max((int)((__float_as_uint(mx) >> 23) & 255u), 27) - 127;      // 2^e <= mx < 2^(e + 1)
        const float up = __uint_as_float((u32)(14 - e + 127) << 23);
        back = __uint_as_float((u32)(e - 14 + 127) << 23) * (scale * 1.44269504088896340736f);
        #pragma unroll
        for (u32 i = 0; i < {Q4}u; ++i) {{
            const float z = f[i] * up;
            q1[i >> 3].e[i & 7u] = (_Float16)z;
            q2[i >> 3].e[i & 7u] = (_Float16)(z - (float)q1[i >> 3].e[i & 7u]);
        }}
    }}
    f4 o[ND];
    #pragma unroll
    for (u32 dt = 0; dt < ND; ++dt) o[dt] = (f4){{0.f, 0.f, 0.f, 0.f}};
    float m = NINF, l = 0.0f;
    const u32 nb = min(last, (most + 63u) >> 6);                                    // blocks of codes that the tile sees
    const u32 j0 = (u32)((u64)nb * split / splits), j1 = (u32)((u64)nb * (split + 1u) / splits);
    const u64 base = ((u64)bh * NB) * (64u * DP);
    const u32 k_at = (16u * (r >> 2) + (r & 3u)) * DP + g * {Q4}u;              // + 4 u DP for tile u
    const u32 v_at = r * 64u + g * 16u;                                         // + dt 16 * 64
    for (u32 j = j0 + w; j < j1; j += 4u) {{
        const unsigned char* __restrict__ kb = kc + base + (u64)j * (64u * DP) + k_at;
        const unsigned char* __restrict__ vb = vc + base + (u64)j * (64u * DP) + v_at;
        uint2 kr[4][{kw}];
        uint4 vr[ND];
        #pragma unroll
        for (u32 u = 0; u < 4u; ++u)
            #pragma unroll
            for (u32 i = 0; i < {kw}u; ++i) kr[u][i] = *reinterpret_cast<const uint2*>(kb + 4u * u * DP + 8u * i);
        #pragma unroll
        for (u32 dt = 0; dt < ND; ++dt) vr[dt] = *reinterpret_cast<const uint4*>(vb + dt * 1024u);
        const float2 sc = *reinterpret_cast<const float2*>(scales + 2u * ((u64)bh * NB + j));
        float s[16];
        const float f = back * sc.x;
        #pragma unroll
        for (u32 u = 0; u < 4u; ++u) {{
            f4 acc = (f4){{0.f, 0.f, 0.f, 0.f}};
            #pragma unroll
            for (u32 i = 0; i < NK; ++i) {{
                const h8 a = widen(kr[u][i].x, kr[u][i].y);
                acc = MFMA16(a, q2[i].v, acc);
                acc = MFMA16(a, q1[i].v, acc);
            }}
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) s[4u * u + i] = acc[i] * f;
        }}
        if (j * 64u + 64u > least) {{                                               // some query of the tile does not see all of the block
            #pragma unroll
            for (u32 i = 0; i < 16u; ++i) if (j * 64u + 16u * g + i >= see) s[i] = NINF;
        }}
        float mx = s[0];
        #pragma unroll
        for (u32 i = 1; i < 16u; ++i) mx = fmaxf(mx, s[i]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
        mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE));
        const float mn = fmaxf(m, mx), mu = mn == NINF ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m - mu);
        m = mn;
        float sum = 0.0f;
        H8 p1[2], p2[2];
        #pragma unroll
        for (u32 i = 0; i < 16u; ++i) {{
            const float p = __builtin_amdgcn_exp2f(s[i] - mu + 15.0f);
            sum += p;
            p1[i >> 3].e[i & 7u] = (_Float16)p;
            p2[i >> 3].e[i & 7u] = (_Float16)(p - (float)p1[i >> 3].e[i & 7u]);
        }}
        l = l * alpha + sum;
        const float vs = sc.y == sc.y ? sc.y : 0.0f;                               // (a NaN scale has made the scores NaN already)
        #pragma unroll
        for (u32 dt = 0; dt < ND; ++dt) {{
            f4 acc = (f4){{0.f, 0.f, 0.f, 0.f}};
            const h8 a0 = widen(vr[dt].x, vr[dt].y), a1 = widen(vr[dt].z, vr[dt].w);
            acc = MFMA16(a0, p2[0].v, acc);
            acc = MFMA16(a1, p2[1].v, acc);
            acc = MFMA16(a0, p1[0].v, acc);
            acc = MFMA16(a1, p1[1].v, acc);
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) o[dt][i] = o[dt][i] * alpha + vs * acc[i];
        }}
    }}
    if (split == splits - 1u && most > last * 64u + 16u * w) {{                     // sixteen tokens of the tail
        const u64 heads = (u64)B * H;
        const float* __restrict__ tk = tail_k + (((u64)(last & 1u) * heads + bh) * 64u + 16u * w) * DP;
        const float* __restrict__ tv = tail_v + (((u64)(last & 1u) * heads + bh) * 64u + 16u * w) * DP;
        f4 acc = (f4){{0.f, 0.f, 0.f, 0.f}};
        #pragma unroll
        for (u32 i = 0; i < {Q4}u; ++i) {{
            const u32 c = g * {Q4}u + i;
            acc = MFMA32(tk[r * DP + c], (live && c < d) ? qrow[c] : 0.0f, acc);
        }}
        const u32 p0 = last * 64u + 16u * w + 4u * g;                               // this lane's four tokens
        float mx = NINF;
        #pragma unroll
        for (u32 i = 0; i < 4u; ++i) {{
            acc[i] = p0 + i < see ? acc[i] * (scale * 1.44269504088896340736f) : NINF;
            mx = fmaxf(mx, acc[i]);
        }}
        mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
        mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE));
        const float mn = fmaxf(m, mx), mu = mn == NINF ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m - mu);
        m = mn;
        float sum = 0.0f;
        #pragma unroll
        for (u32 i = 0; i < 4u; ++i) {{ acc[i] = __builtin_amdgcn_exp2f(acc[i] - mu + 15.0f); sum += acc[i]; }}
        l = l * alpha + sum;
        #pragma unroll
        for (u32 dt = 0; dt < ND; ++dt) {{
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) o[dt][i] *= alpha;
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) {{
                const float x = tv[(4u * g + i) * DP + dt * 16u + r];
                o[dt] = MFMA32((p0 + i < most && x == x) ? x : 0.0f, acc[i], o[dt]);      // (a NaN row has made the scores NaN already)
            }}
        }}
    }}
    l += __shfl_xor(l, 16, WAVE);
    l += __shfl_xor(l, 32, WAVE);
    if (g == 0u) {{ sm[w][r] = m; sl[w][r] = l; }}
    #pragma unroll
    for (u32 dt = 0; dt < ND; ++dt) *reinterpret_cast<f4*>(&so[w][r][dt * 16u + 4u * g]) = o[dt];
    __syncthreads();
    // sixteen threads a row: the four wavefronts' parts, in their order
    const u32 jr = t >> 4, jc = t & 15u, jrow = tile * 16u + jr;
    if (jrow >= rows) return;
    float M = NINF, L = 0.0f, fac[4];
    #pragma unroll
    for (u32 i = 0; i < 4u; ++i) M = fmaxf(M, sm[i][jr]);
    #pragma unroll
    for (u32 i = 0; i < 4u; ++i) {{ fac[i] = sm[i][jr] == NINF ? 0.0f : __builtin_amdgcn_exp2f(sm[i][jr] - M); L += fac[i] * sl[i][jr]; }}
    if (splits == 1u) {{
        float* __restrict__ yr = y + ((u64)b * T + jrow / group) * C + (u64)(h * group + jrow % group) * d;
        for (u32 c = jc; c < d; c += 16u) {{
            float a = 0.0f;
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) a += fac[i] * so[i][jr][c];
            yr[c] = L == 0.0f ? 0.0f : a / L;
        }}
    }} else {{
        float* __restrict__ pr = part + (((u64)bh * rows + jrow) * splits + split) * (DP + 2u);
        for (u32 c = jc; c < d; c += 16u) {{
            float a = 0.0f;
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) a += fac[i] * so[i][jr][c];
            pr[c] = a;
        }}
        if (jc == 0u) {{ pr[DP] = M; pr[DP + 1u] = L; }}
    }}
}}
"""
    return src, name, _fmt("P" * 10, "I" * 8, "f")


@cache
def cache8_join_kernel(DP: int) -> tuple[str, str, str]:
    """Adds up what cache8_attend_kernel left per split: O = sum exp(m_s - M) O_s over sum exp(m_s - M) l_s, in the order of the
    splits.  One wavefront per query row of a key head."""
    name = f"cache8_join_d{DP}"
    src = f"""{PRELUDE}
#define DP {DP}u
#define NINF (-__builtin_inff())
extern "C" __global__ __launch_bounds__(256) void {name}(const float* __restrict__ part, float* __restrict__ y,
        u32 items, u32 T, u32 H, u32 group, u32 d, u32 splits) {{
    const u32 item = blockIdx.x * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    if (item >= items) return;
    const u32 rows = T * group, bh = item / rows, row = item % rows, b = bh / H, h = bh % H;
    const float* __restrict__ pr = part + (u64)item * splits * (DP + 2u);
    float M = NINF, L = 0.0f;
    for (u32 s = 0; s < splits; ++s) M = fmaxf(M, pr[s * (DP + 2u) + DP]);
    float acc[{(DP + 63) // 64}];
    #pragma unroll
    for (u32 i = 0; i < {(DP + 63) // 64}u; ++i) acc[i] = 0.0f;
    for (u32 s = 0; s < splits; ++s) {{
        const float* __restrict__ ps = pr + s * (DP + 2u);
        const float f = ps[DP] == NINF ? 0.0f : __builtin_amdgcn_exp2f(ps[DP] - M);
        L += f * ps[DP + 1u];
        #pragma unroll
        for (u32 i = 0; i < {(DP + 63) // 64}u; ++i) {{ const u32 c = i * 64u + lane; if (c < d) acc[i] += f * ps[c]; }}
    }}
    float* __restrict__ yr = y + ((u64)b * T + row / group) * ((u64)H * group * d) + (u64)(h * group + row % group) * d;
    #pragma unroll
    for (u32 i = 0; i < {(DP + 63) // 64}u; ++i) {{ const u32 c = i * 64u + lane; if (c < d) yr[c] = L == 0.0f ? 0.0f : acc[i] / L; }}
}}
"""
    return src, name, _fmt("P" * 2, "I" * 6)
