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
def rotary_kernel(half: bool, vec: bool, stream: bool = False) -> tuple[str, str, str]:
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
    (keys beside queries) in the same launch.  stream: loads and stores that bypass the caches, for tensors larger than they
    are.  Bound by memory: 8 bytes an element (30001 rows of 32 + 8 heads of 128: 206 us, 6.0 TB/s; 218 us through the caches)."""
    assert vec or not stream
    name = f"rotary_{'half' if half else 'pairs'}_{'v4' if vec else 'v1'}{'_nt' if stream else ''}"
    get = (lambda at: f"ld4_stream(reinterpret_cast<const float4*>({at}))") if stream else (lambda at: f"*reinterpret_cast<const float4*>({at})")      # noqa: E731
    put = ((lambda at, v: f"{{ const v4f o4 = {{{v}}}; __builtin_nontemporal_store(o4, reinterpret_cast<v4f*>({at})); }}") if stream
           else (lambda at, v: f"*reinterpret_cast<float4*>({at}) = make_float4({v});"))                                            # noqa: E731
    W = (4 if half else 2) if vec else 1                 # pairs of a rotating unit
    if half:
        load = (f"const float4 a = {get('xr + off + j')}, b = {get('xr + off + hr + j')};"
                if vec else "const float a = xr[off + j], b = xr[off + hr + j];")
        keep = ("va[n][0] = a.x; va[n][1] = a.y; va[n][2] = a.z; va[n][3] = a.w; vb[n][0] = b.x; vb[n][1] = b.y; vb[n][2] = b.z; vb[n][3] = b.w;"
                if vec else "va[n][0] = a; vb[n][0] = b;")
        store = (put("yr + off + j", "oa[0], oa[1], oa[2], oa[3]") + " " + put("yr + off + hr + j", "ob[0], ob[1], ob[2], ob[3]")
                 if vec else "yr[off + j] = oa[0]; yr[off + hr + j] = ob[0];")
    else:
        load = (f"const float4 a = {get('xr + off + 2u * j')};" if vec
                else "const float a = xr[off + 2u * j], b = xr[off + 2u * j + 1u];")
        keep = ("va[n][0] = a.x; vb[n][0] = a.y; va[n][1] = a.z; vb[n][1] = a.w;" if vec else "va[n][0] = a; vb[n][0] = b;")
        store = (put("yr + off + 2u * j", "oa[0], ob[0], oa[1], ob[1]") if vec
                 else "yr[off + 2u * j] = oa[0]; yr[off + 2u * j + 1u] = ob[0];")
    copy = (f"const float4 a = {get('xr + off + c')}; " + put("yr + off + c", "a.x, a.y, a.z, a.w") if vec else "yr[off + c] = xr[off + c];")
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

LOGITS_PACKED_L = 65535      # the longest history whose counts fit 16 bits


@cache
def adjust_logits_kernel(items: int, vec: bool, packed: bool) -> tuple[str, str, str]:
    """y = logits (B, V) with what has been said already made less likely, a bias added and forbidden tokens removed:
    for a token that occurs c > 0 times among the first lengths[b] entries of history[b],
      x = x / repetition if x > 0 else x * repetition, then x - (presence + frequency * c);
    then + bias[v]; then -inf where hidden > 0 (whatever stood there, a NaN included).  Entries of the history outside
    [0, V) count for nothing.  Each of the three penalties is a number, or an array with one per row.

    A block owns 256 * items consecutive tokens of one row and counts only those: their counters lie in LDS, every
    block walks the whole history of its row (which stays in L2: 4 bytes an entry) and bumps the counters of its own
    tokens with integer atomics, whose order does not matter.  So there is one launch, no count array in memory and
    no sort.  packed: two 16-bit counters to a word, for histories of at most 65535 -- half the LDS, twice the blocks on a
    compute unit.  The first 16 entries a thread walks and its logits are loaded before the counters are cleared, so all of
    these reads are on their way together.  vec: 16-byte accesses (V % 4 == 0).  Bound by memory: 8 bytes a logit (256 x 128256,
    4000 said: 53.7 us from HBM, 5.0 TB/s; 45 to 47 us partly from the Infinity Cache)."""
    assert items in (4, 8, 16)
    name = f"adjust_logits_i{items}_{'v4' if vec else 'v1'}{'_h' if packed else ''}"
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
    words = 128 * items if packed else 256 * items
    bump = "atomicAdd(&count[at >> 1], 1u << (16u * (at & 1u)))" if packed else "atomicAdd(&count[at], 1u)"
    if vec:
        counts = ("const uint2 c2 = *reinterpret_cast<const uint2*>(&count[at >> 1]); const u32 c[4] = {c2.x & 0xffffu, c2.x >> 16, c2.y & 0xffffu, c2.y >> 16};"
                  if packed else "const uint4 c4 = *reinterpret_cast<const uint4*>(&count[at]); const u32 c[4] = {c4.x, c4.y, c4.z, c4.w};")
    else:
        counts = "const u32 c[1] = {(count[at >> 1] >> (16u * (at & 1u))) & 0xffffu};" if packed else "const u32 c[1] = {count[at]};"
    any_of = " | ".join(f"c[{i}]" for i in range(W))
    src = f"""{PRELUDE}
#define NINF (-__builtin_inff())
#define SLICE {256 * items}u
extern "C" __global__ __launch_bounds__(256) void {name}(const float* __restrict__ logits, const float* __restrict__ history,
        const float* __restrict__ lengths, const float* __restrict__ bias, const float* __restrict__ hidden, float* __restrict__ y,
        const float* __restrict__ rep_p, const float* __restrict__ pre_p, const float* __restrict__ fre_p,
        u32 V, u32 L, u32 bias_step, u32 hidden_step, float rep, float pre, float fre) {{
    __shared__ __attribute__((aligned(16))) u32 count[{words}];
    const u32 t = threadIdx.x, v0 = blockIdx.x * SLICE;
    const u64 b = blockIdx.y;
    const float* __restrict__ lrow = logits + b * V;
    float* __restrict__ yrow = y + b * V;
    const float* __restrict__ said = history + b * L;
    float first[16];
    #pragma unroll
    for (u32 k = 0; k < 16u; ++k) {{ const u32 i = k * 256u + t; first[k] = i < L ? said[i] : -1.0f; }}
    const float ln = (L && lengths) ? lengths[b] : (float)L;
    const u32 n = ln >= (float)L ? L : ln > 0.0f ? (u32)ln : 0u;             // (a NaN counts nothing)
    float x[{NV}][{W}];
    #pragma unroll
    for (u32 k = 0; k < {NV}u; ++k) {{
        const u32 v = v0 + (k * 256u + t) * {W}u;
        if (v < V) {{ {load} }}
    }}
    if (L) {{
        for (u32 k = t; k < {words}u; k += 256u) count[k] = 0u;
        __syncthreads();
        auto bump = [&](float id) {{
            if (id >= (float)v0 && id < 4294967040.0f) {{
                const u32 at = (u32)id - v0;
                if (at < SLICE) {bump};
            }}
        }};
        #pragma unroll
        for (u32 k = 0; k < 16u; ++k) if (k * 256u + t < n) bump(first[k]);
        #pragma unroll 8
        for (u32 k = 4096u + t; k < n; k += 256u) bump(said[k]);
        __syncthreads();
    }}
    if (n) {{
        const float r = rep_p ? rep_p[b] : rep, p = pre_p ? pre_p[b] : pre, f = fre_p ? fre_p[b] : fre;
        #pragma unroll
        for (u32 k = 0; k < {NV}u; ++k) {{
            const u32 at = (k * 256u + t) * {W}u;
            {counts}
            if ({any_of}) {{
                #pragma unroll
                for (u32 i = 0; i < {W}u; ++i)
                    if (c[i]) x[k][i] = (x[k][i] > 0.0f ? x[k][i] / r : x[k][i] * r) - (p + f * (float)c[i]);
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
#define CACHE8_MARKS 32u                                                    // words from one head's marks to the next's
// Whether a tail that says `mark` keeps the first `rows` (1 .. 63) rows of block blk: a mark is 64 * block + the rows that lie there.
static __device__ __forceinline__ bool cache8_kept(u32 mark, u32 blk, u32 rows) {
    return mark >= blk * 64u + rows && mark <= blk * 64u + 64u;
}
"""


def _cache8_layout(DP: int) -> str:
    """Where a block of 64 tokens by DP columns keeps its bytes: in the order in which the wavefront of cache8_attend_kernel reads
    them, so that each of its loads is one run of memory.  Lane r + 16 g (r < 16, g < 4) takes of the keys, for token tile u, the quarter
    g .. of the columns of token 16 (r / 4) + 4 u + r % 4, 16 bytes at a time (8 where a quarter is no multiple of 16); of the
    values, for columns 16 dt + r, the tokens 16 g .. 16 g + 15."""
    Q4 = DP // 4
    w = 16 if Q4 % 16 == 0 else 8
    return f"""
#define DP {DP}u
static __device__ __forceinline__ u32 key_at(u32 row, u32 c) {{
    const u32 g = c / {Q4}u, i = c % {Q4}u;
    return ((row >> 2) & 3u) * {64 * Q4}u + (i / {w}u) * {64 * w}u + (g * 16u + ((row >> 4) << 2) + (row & 3u)) * {w}u + i % {w}u;
}}
static __device__ __forceinline__ u32 value_at(u32 row, u32 c) {{ return (c >> 4) * 1024u + ((row >> 4) * 16u + (c & 15u)) * 16u + (row & 15u); }}
"""


CACHE8_WRITE_THREADS = 512


@cache
def cache8_write_kernel(DP: int, vec: bool) -> tuple[str, str, str]:
    """New key and value rows k, v (B, T, H * d) into the 8-bit cache of one layer, at positions lengths[b] .. of each sequence
    (the first counts[b] rows of each, all T without counts; rows that the cache has no room for are dropped).

    A block of 64 tokens of one head is quantised when its last token arrives, and never again: scale = max |x| / 127
    in 32 bits, code = x / scale to the nearest whole number, ties to even.  Until then its rows stay fp32 in the tail, so what
    the cache holds depends on the tokens alone and not on the calls that brought them.  A code is a byte, code + 128, where
    _cache8_layout says; there are two tails of 64 rows per head, block i's is tail i & 1.

    The quotient is rounded exactly: q = rint(x * (1 / scale)) may be off by one next to a half.  There x - q * scale, which is
    representable (both are multiples of the unit of the smaller one, and it is below two scales), comes without error from
    one fused multiply-add, and the comparison with half a scale decides.

    A row that holds a NaN or an infinity is kept as NaN in the tail, and a block with such a row gets NaN for its scales:
    every output that sees it is NaN, and the codes stay whole numbers.

    A call may be followed by one that starts at a smaller length than it ended at, or at its own again.  Both tails together hold what
    that takes while the call touches two blocks; one that completes more leaves the rows of the blocks between nowhere in fp32, and
    where it ends in the tail that it started in, those of its first block neither.  Each tail's mark says what lies there
    (cache8_kept), and rows that are not there are NaN to whoever needs them.  The marks of a head have a line of memory to
    themselves, because workgroups of different dies write them, and are waited for after the rows (8 x 12 heads of 64, a token: 3.8 us; with
    neighbours in a line 4.1, waited for with the lengths 4.2; without marks 3.4).

    One workgroup of 512 threads per (block of 64, head, sequence), a thread per four columns of a row (DP / 32 times).  With 256 a
    launch of few workgroups, which is one pass over the code, takes longer (2 x 12 heads of 64, 512 tokens: 6.7 us against 5.4),
    with 1024 many wait for each other's barriers (4 x 12 heads of 64, 4096 tokens: 37 us against 29, 4.4 TB/s).  Workgroup 0
    of a head completes the block that the call starts in and then stores the rows of the block it ends in, in this order,
    because both may use the same tail.  Bound by memory for long calls, 4 bytes read and 1 written per element; by its chain of
    reads, reduction and stores for short ones (the token that completes 96 blocks: 5.4 us; one that completes none: 3.0)."""
    name = f"cache8_write_d{DP}_{'v4' if vec else 'v1'}"
    NT = CACHE8_WRITE_THREADS
    IT = -(-16 * DP // NT)                     # four columns of a row per thread, so many times
    if vec:
        # one load whatever the row is: a choice between two loads would wait for one before the other
        load = """const float* pk = row < lo || c0 >= d ? tk + row * DP + c0 : kh + at * kp + c0;
            const float* pv = row < lo || c0 >= d ? tv + row * DP + c0 : vh + at * vp + c0;
            fk = *reinterpret_cast<const float4*>(there ? pk : tk);
            fv = *reinterpret_cast<const float4*>(there ? pv : tv);
            if (!there || (row >= lo && c0 >= d)) { fk = make_float4(0.f, 0.f, 0.f, 0.f); fv = fk; }"""
    else:
        load = """if (there && row < lo) { fk = *reinterpret_cast<const float4*>(tk + row * DP + c0); fv = *reinterpret_cast<const float4*>(tv + row * DP + c0); }
            else if (there) {
                const float* pk = kh + at * kp;
                const float* pv = vh + at * vp;
                if (c0 < d) { fk.x = pk[c0]; fv.x = pv[c0]; }
                if (c0 + 1u < d) { fk.y = pk[c0 + 1u]; fv.y = pv[c0 + 1u]; }
                if (c0 + 2u < d) { fk.z = pk[c0 + 2u]; fv.z = pv[c0 + 2u]; }
                if (c0 + 3u < d) { fk.w = pk[c0 + 3u]; fv.w = pv[c0 + 3u]; }
            }"""
    src = f"""{PRELUDE}{_CACHE8}{_cache8_layout(DP)}#define C4 {DP // 4}u
// four codes + 128 in the bytes of a word
static __device__ __forceinline__ u32 codes_of(float4 f, float s, float inv, float up) {{
    const float x[4] = {{f.x * up, f.y * up, f.z * up, f.w * up}};
    float q[4], far = 0.0f;
    #pragma unroll
    for (u32 i = 0; i < 4u; ++i) {{
        const float z = x[i] * inv;                                     // off by 127 * 2^-23 at most
        q[i] = rintf(z);
        far = fmaxf(far, fabsf(z - q[i]));
    }}
    if (far > 0.49998f) {{                                              // next to a half: the remainder decides
        #pragma unroll
        for (u32 i = 0; i < 4u; ++i) {{
            const float r = fmaf(-q[i], s, x[i]), r2 = 2.0f * fabsf(r);
            if (r2 > s || (r2 == s && ((int)q[i] & 1))) q[i] += r < 0.0f ? -1.0f : 1.0f;
        }}
    }}
    u32 w = 0u;
    #pragma unroll
    for (u32 i = 0; i < 4u; ++i) w |= (u32)(fminf(fmaxf(q[i], -127.0f), 127.0f) + 128.0f) << (8u * i);
    return w;
}}
static __device__ __forceinline__ float most4(float4 f) {{ return fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))); }}
static __device__ __forceinline__ bool odd_one(float x) {{ return !(fabsf(x) < __builtin_inff()); }}
static __device__ __forceinline__ bool odd4(float4 f) {{ return odd_one(f.x) || odd_one(f.y) || odd_one(f.z) || odd_one(f.w); }}
extern "C" __global__ __launch_bounds__({NT}) void {name}(const float* __restrict__ k, const float* __restrict__ v,
        const float* __restrict__ lengths, const float* __restrict__ counts,
        unsigned char* __restrict__ kc, unsigned char* __restrict__ vc, float* __restrict__ scales, float* tail_k, float* tail_v, u32* marks,
        u32* __restrict__ wrote, u32 T, u32 H, u32 d, u32 NB, u32 kp, u32 vp) {{
    __shared__ __attribute__((aligned(16))) u32 kt[DP * 16u], vt[DP * 16u];       // the block's bytes
    __shared__ float sk[{NT // 64}], sv[{NT // 64}];
    __shared__ u32 bad[64];
    const u32 t = threadIdx.x, lane = t & 63u, h = blockIdx.y, b = blockIdx.z;
    u32 len, n;
    const u64 bh = (u64)b * H + h, heads = (u64)gridDim.z * H;
    const u32 was = marks[CACHE8_MARKS * bh + (lane & 1u)];                  // (written by workgroup 0 alone, which alone goes by them; a lane's load, since a scalar one would be waited for with the lengths)
    cache8_extent(lengths, counts, b, T, NB * 64u, len, n);
    const u32 total = len + n, first = len >> 6, last = total >> 6;         // last: the block that is not full afterwards
    bool lost = false;                                                        // the rows before this call are not in their tail
    u32 other = 0u;
    auto look = [&]() {{
        u32 m = was;
        asm volatile("" : "+v"(m));                                             // (the marks are waited for here, not before the rows are loaded)
        lost = (len & 63u) && !cache8_kept(__builtin_amdgcn_readlane(m, first & 1u), first, len & 63u);
        other = __builtin_amdgcn_readlane(m, (first & 1u) ^ 1u);
    }};
    auto leave = [&]() {{                                                      // what the call leaves
        if (h == 0u) wrote[b] = n;
        const u32 f64 = first * 64u, l64 = last * 64u + (total & 63u);
        // the first block's tail: what lay there, and the new rows where they are stored
        u32 a = lost ? 0u : last == first ? l64 : last == first + 1u ? f64 + 64u : f64 + (len & 63u);
        u32 o = other <= f64 ? other : 0u;                                  // the other one: not what a call before this one put there in its place
        if (last > first) {{
            if ((last - first) & 1u) o = l64;
            else if (total & 63u) a = l64;
        }}
        *reinterpret_cast<uint2*>(marks + CACHE8_MARKS * bh) = first & 1u ? make_uint2(o, a) : make_uint2(a, o);
    }};
    if (!n) {{
        if (blockIdx.x == 0u) {{ look(); if (t == 0u) leave(); }}
        return;
    }}
    const float* __restrict__ kh = k + (u64)b * T * kp + (u64)h * d;
    const float* __restrict__ vh = v + (u64)b * T * vp + (u64)h * d;
    for (u32 pass = 0; pass < 2u; ++pass) {{
        const u32 blk = pass ? last : first + blockIdx.x;
        if (pass && (blockIdx.x != 0u || last == first || !(total & 63u))) break;       // (uniform over the workgroup)
        const bool full = blk < last;
        if (!pass && !full && blk != first) break;
        if (blk >= NB) break;
        float* tk = tail_k + (((u64)(blk & 1u) * heads + bh) * 64u) * DP;
        float* tv = tail_v + (((u64)(blk & 1u) * heads + bh) * 64u) * DP;
        const u32 lo = blk == first ? (len & 63u) : 0u, hi = full ? 64u : (total & 63u);       // new rows of this block
        if (t < 64u) bad[t] = 0u;
        __syncthreads();
        float4 xk[{IT}], xv[{IT}];
        float mk = 0.0f, mv = 0.0f;
        #pragma unroll
        for (u32 it = 0; it < {IT}u; ++it) {{
            const u32 row = (it * {NT}u + t) / C4, c0 = (it * {NT}u + t) % C4 * 4u;
            // a row of the block: new, or from the tail (only the block the call starts in, and only if it is quantised now)
            const bool there = row < hi && (row >= lo || full);
            const u64 at = (u64)blk * 64u + row - len;
            float4 fk = make_float4(0.f, 0.f, 0.f, 0.f), fv = fk;
            {load}
            if (odd4(fk) || odd4(fv)) bad[row] = 1u;
            xk[it] = fk;
            xv[it] = fv;
            mk = fmaxf(mk, most4(fk));
            mv = fmaxf(mv, most4(fv));
        }}
        mk = wave_max(mk);
        mv = wave_max(mv);
        if (lane == 0u) {{ sk[t >> 6] = mk; sv[t >> 6] = mv; }}
        if (!pass && blockIdx.x == 0u) look();
        __syncthreads();
        if (!pass && blockIdx.x == 0u && t == 0u) leave();                      // (every thread has read the marks)
        // the rows as they came: needed while the block is not full (and again if the caller goes back into it)
        if (!full || (blk == first && last == first + 1u)) {{
            #pragma unroll
            for (u32 it = 0; it < {IT}u; ++it) {{
                const u32 row = (it * {NT}u + t) / C4, c0 = (it * {NT}u + t) % C4 * 4u;
                if (row >= lo && row < hi) {{
                    const float z = __builtin_nanf("");
                    const bool odd = bad[row] != 0u;
                    *reinterpret_cast<float4*>(tk + row * DP + c0) = odd ? make_float4(z, z, z, z) : xk[it];
                    *reinterpret_cast<float4*>(tv + row * DP + c0) = odd ? make_float4(z, z, z, z) : xv[it];
                }}
            }}
        }}
        if (full) {{
            const bool odd = __any(bad[lane] != 0u) || (lost && blk == first);
            float ak = 0.0f, av = 0.0f;
            #pragma unroll
            for (u32 i = 0; i < {NT // 64}u; ++i) {{ ak = fmaxf(ak, sk[i]); av = fmaxf(av, sv[i]); }}
            ak /= 127.0f;
            av /= 127.0f;
            const u64 at = bh * NB + blk;
            if (t == 0u) *reinterpret_cast<float2*>(scales + 2u * at) = odd ? make_float2(__builtin_nanf(""), __builtin_nanf("")) : make_float2(ak, av);
            // a scale below 2^-60 has no finite reciprocal or an inexact remainder: both sides times 2^64, exactly
            const float upk = ak < 8.6736174e-19f ? 18446744073709551616.0f : 1.0f, upv = av < 8.6736174e-19f ? 18446744073709551616.0f : 1.0f;
            const float s_k = ak * upk, s_v = av * upv, ik = ak > 0.0f ? 1.0f / s_k : 0.0f, iv = av > 0.0f ? 1.0f / s_v : 0.0f;
            unsigned char* vt8 = reinterpret_cast<unsigned char*>(vt);
            #pragma unroll
            for (u32 it = 0; it < {IT}u; ++it) {{
                const u32 row = (it * {NT}u + t) / C4, c0 = (it * {NT}u + t) % C4 * 4u;
                if (row < 64u) {{
                    kt[key_at(row, c0) >> 2] = codes_of(xk[it], s_k, ik, upk);
                    const u32 cv = codes_of(xv[it], s_v, iv, upv);
                    #pragma unroll
                    for (u32 c = 0; c < 4u; ++c) vt8[value_at(row, c0 + c)] = (unsigned char)(cv >> (8u * c));
                }}
            }}
            __syncthreads();
            uint4* __restrict__ kb = reinterpret_cast<uint4*>(kc + at * (64u * DP));
            uint4* __restrict__ vb = reinterpret_cast<uint4*>(vc + at * (64u * DP));
            for (u32 i = t; i < DP * 8u; i += {NT}u) {{
                if (i < DP * 4u) kb[i] = reinterpret_cast<const uint4*>(kt)[i];
                else vb[i - DP * 4u] = reinterpret_cast<const uint4*>(vt)[i - DP * 4u];
            }}
        }}
        __syncthreads();
    }}
}}
"""
    return src, name, _fmt("P" * 11, "I" * 6)


@cache
def cache8_advance_kernel() -> tuple[str, str, str]:
    """lengths[b] += by[b], or `all` for every sequence, as the whole number of rows it stands for and no more than the last write
    brought and an earlier advance left of them (wrote[b]); reset: everything to 0.  A launch and nothing else: three numbers a sequence."""
    src = f"""{PRELUDE}{_CACHE8}
extern "C" __global__ __launch_bounds__(256) void cache8_advance(float* __restrict__ lengths, const float* __restrict__ by, u32* __restrict__ wrote,
        u32 B, u32 cap, u32 all, u32 reset) {{
    const u32 b = blockIdx.x * 256u + threadIdx.x;
    if (b >= B) return;
    u32 len, n;
    const u32 w = wrote[b];
    cache8_extent(lengths, by, b, by ? w : min(w, all), cap, len, n);
    lengths[b] = reset ? 0.0f : (float)(len + n);
    wrote[b] = reset ? 0u : w - n;
}}
"""
    return src, "cache8_advance", _fmt("P" * 3, "I" * 4)


@cache
def cache8_read_kernel(DP: int) -> tuple[str, str, str]:
    """The values that the cache of one layer stands for, as fp32 k and v (B, N, H * d): code * scale for the tokens of full
    blocks, the rows themselves for those of the tail, zeros from position lengths[b] + counts[b] on (counts: rows written
    since the lengths were advanced, of those there are; `extra` for every sequence without them).  One workgroup per (block of 64, head,
    sequence); the codes pass through LDS so that rows leave as rows.  Bound by memory (8 x 1024 tokens of 12 heads of 64: 11.3 us,
    5.6 TB/s)."""
    name = f"cache8_read_d{DP}"
    src = f"""{PRELUDE}{_CACHE8}{_cache8_layout(DP)}extern "C" __global__ __launch_bounds__(256) void {name}(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
        const float* __restrict__ scales, const float* __restrict__ tail_k, const float* __restrict__ tail_v, const u32* __restrict__ marks,
        const u32* __restrict__ wrote, const float* __restrict__ lengths, const float* __restrict__ counts, float* __restrict__ ko, float* __restrict__ vo,
        u32 N, u32 H, u32 d, u32 NB, u32 extra) {{
    __shared__ __attribute__((aligned(16))) u32 kt[DP * 16u], vt[DP * 16u];       // the block's bytes
    const u32 t = threadIdx.x, blk = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    u32 len, n;
    cache8_extent(lengths, counts, b, extra, NB * 64u, len, n);
    n = min(n, wrote[b]);
    const u32 total = len + n, last = total >> 6;
    const u64 bh = (u64)b * H + h, heads = (u64)gridDim.z * H, at = bh * NB + blk;
    const float s_k = blk < last ? scales[2u * at] : 0.0f, s_v = blk < last ? scales[2u * at + 1u] : 0.0f;
    if (blk < last) {{
        const uint4* __restrict__ kb = reinterpret_cast<const uint4*>(kc + at * (64u * DP));
        const uint4* __restrict__ vb = reinterpret_cast<const uint4*>(vc + at * (64u * DP));
        for (u32 i = t; i < DP * 8u; i += 256u) {{
            if (i < DP * 4u) reinterpret_cast<uint4*>(kt)[i] = kb[i];
            else reinterpret_cast<uint4*>(vt)[i - DP * 4u] = vb[i - DP * 4u];
        }}
    }}
    __syncthreads();
    const float* __restrict__ tk = tail_k + (((u64)(blk & 1u) * heads + bh) * 64u) * DP;
    const float* __restrict__ tv = tail_v + (((u64)(blk & 1u) * heads + bh) * 64u) * DP;
    const bool lost = blk == last && (total & 63u) && !cache8_kept(marks[CACHE8_MARKS * bh + (blk & 1u)], blk, total & 63u);
    const u64 C = (u64)H * d;
    // four columns a thread (as many of them as there are)
    for (u32 i = t; i < 64u * {DP // 4}u; i += 256u) {{
        const u32 row = i / {DP // 4}u, c = i % {DP // 4}u * 4u, p = blk * 64u + row;
        if (p >= N || c >= d) continue;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f), z = x;
        if (blk < last) {{
            const u32 w = kt[key_at(row, c) >> 2];
            const unsigned char* vt8 = reinterpret_cast<const unsigned char*>(vt) + value_at(row, c);             // (four columns of one tile: 16 apart)
            x = make_float4((float)((int)(w & 255u) - 128) * s_k, (float)((int)((w >> 8) & 255u) - 128) * s_k,
                            (float)((int)((w >> 16) & 255u) - 128) * s_k, (float)((int)(w >> 24) - 128) * s_k);
            z = make_float4((float)((int)vt8[0] - 128) * s_v, (float)((int)vt8[16] - 128) * s_v, (float)((int)vt8[32] - 128) * s_v, (float)((int)vt8[48] - 128) * s_v);
        }} else if (p < total) {{
            x = *reinterpret_cast<const float4*>(tk + row * DP + c);
            z = *reinterpret_cast<const float4*>(tv + row * DP + c);
            if (lost) {{ const float no = __builtin_nanf(""); x = make_float4(no, no, no, no); z = x; }}
        }}
        const u64 o = ((u64)b * N + p) * C + (u64)h * d + c;
        if ((d & 3u) == 0u) {{                                              // (fresh results are aligned)
            *reinterpret_cast<float4*>(ko + o) = x;
            *reinterpret_cast<float4*>(vo + o) = z;
        }} else {{
            ko[o] = x.x; vo[o] = z.x;
            if (c + 1u < d) {{ ko[o + 1u] = x.y; vo[o + 1u] = z.y; }}
            if (c + 2u < d) {{ ko[o + 2u] = x.z; vo[o + 2u] = z.z; }}
            if (c + 3u < d) {{ ko[o + 3u] = x.w; vo[o + 3u] = z.w; }}
        }}
    }}
}}
"""
    return src, name, _fmt("P" * 11, "I" * 5)


@cache
def cache8_attend_kernel(DP: int, NQ: int = 1, W: int = 4, stream: bool = False) -> tuple[str, str, str]:
    """Attention of T new positions per sequence over the 8-bit cache of one layer, after their keys and values were written:
    y = softmax(q K^T * scale) V per query head, query t of sequence b at position lengths[b] + t seeing the positions up to its
    own; `group` query heads share a key head.  q and y are (B, T, H * group * d).  A row beyond counts[b], or beyond what the last write
    brought, gives zeros.

    The codes are whole numbers of at most 127 and therefore exact in 16-bit floats, so the matrix units do the work:
    a query row is scaled by a power of two to at most 2^15 and held as two 16-bit floats an element, q' = q1 + q2 / 2^11: q1 the
    nearest to q', q2 the nearest to what is left, 2^11 times.  That is q' to 2^-22 of itself or, where q2 runs into the smallest
    steps of a 16-bit float, to 2^-36: 2^-50 of the row's largest element.  (Without the 2^11 they would begin at 2^-17 of the
    largest, not 2^-28.)  S^T = K q1^T + K q2^T / 2^11 is two v_mfma_f32_16x16x32_f16 per 32 columns, added in 32 bits.  The probabilities go
    the same way: p' = 2^15 exp(s - m) = p1 + p2 / 2^11, to 2^-22 of itself or 2^-51 of the largest one, which makes less than 2^-26 of it in the sum of
    2^24 tokens; the factor 2^15 cancels in p' V / sum p'.  The scales enter in 32 bits, the keys' with the scores, the values' as a
    block's product joins the running sum.

    A wavefront takes one block of 64 tokens at a time, for NQ tiles of 16 query rows, with (m, l, O) of its own.  Its lane
    r + 16 g (r < 16, g < 4) holds query r of each tile and, of every product S^T, four tokens; the rows of K are fed in the order
    that makes those of the four token tiles the sixteen neighbours 16 g ..: then P is already the B operand of O^T += V^T P^T,
    and its A operand, sixteen value codes of one column, one 16-byte load.  Nothing passes through LDS, and each load is one
    run of memory (_cache8_layout).  Bytes become 16-bit floats in one operation each: v_perm puts byte c under the exponent
    of 1024, giving 1024 + c, and a packed addition takes 1152 away.  The keys of the next block are loaded when those of this
    one have been used, while its softmax runs, and its values likewise during the next scores.  stream: loads that leave no
    trace in the caches, for codes that are read once and would only displace others.

    The tail, fp32, is shared out 16 tokens to a wavefront and goes through v_mfma_f32_16x16x4_f32, with q1 + q2 / 2^11 as the query.

    A workgroup of W wavefronts per (NQ tiles of one key head, split of the blocks); they are joined through LDS in
    wavefront order.  With one split y is written; else O, m and l go to `part` and cache8_join_kernel adds the splits up
    in their order.  Bound by memory while few query rows share a key head, 2 bytes per token and column (16 sequences up to 32768
    tokens, 32 heads on 8 of 128: 132 us, 6.2 TB/s); with many by the issue of instructions, some 345 vector and 32 matrix ones a block of 64 and
    tile of 16 rows (4 x 12 heads of 64, 256 rows after 4096 tokens: 47 us, 280 TFLOP/s of the formula's operations; the SIMDs issue vector
    instructions in 66 % of the cycles, the matrix units are busy in 21 %); with few blocks by chains of dependent reads (one block and a
    tail: 3.8 us)."""
    ND, NK, Q4 = DP // 16, DP // 32, DP // 4             # column tiles of V^T, k steps of a score, columns a lane feeds
    name = f"cache8_attend_d{DP}" + (f"_q{NQ}" if NQ > 1 else "") + (f"_w{W}" if W != 4 else "") + ("_nt" if stream else "")
    wide = Q4 % 16 == 0                                   # a lane's quarter of a key in 16-byte words, else in words of 8
    kw, kn = (Q4 // 16, 4) if wide else (Q4 // 8, 2)
    fetch = "__builtin_nontemporal_load({})" if stream else "*{}"
    fetch_k = fetch.format(f"reinterpret_cast<const u{kn}*>(p + u * {64 * Q4}u + i * {256 * kn}u)")
    fetch_v = fetch.format("reinterpret_cast<const u4*>(p + dt * 1024u)")
    half = ("i & 1u ? kr[u][i >> 1].z : kr[u][i >> 1].x, i & 1u ? kr[u][i >> 1].w : kr[u][i >> 1].y" if wide else "kr[u][i].x, kr[u][i].y")
    # "256, 2" holds the kernel to 256 registers, with which the matrix instructions write ordinary ones; wider heads need more.  "512, 4": 128, so that
    # two workgroups of eight share a compute unit (48 x 12 heads of 64 over 600 tokens: 16.6 us against 20.4 with 158 registers); that takes the low
    # products of the scores in the same accumulators, ahead of the high ones, where they have accumulators of their own otherwise (4 x 12
    # heads of 64, 512 rows after 4096: 75.8 us, 80.1 in the same)
    tight = W == 8 and NQ == 1 and DP <= 64
    bounds = "256, 2" if W == 4 and DP * NQ <= 128 else "512, 4" if tight else f"{64 * W}"
    if tight:
        scores = f"""h8 k8[NK];
            #pragma unroll
            for (u32 i = 0; i < NK; ++i) k8[i] = widen({half});
            s[0][u] = (f4){{0.f, 0.f, 0.f, 0.f}};
            #pragma unroll
            for (u32 i = 0; i < NK; ++i) s[0][u] = MFMA16(k8[i], q2[0][i].v, s[0][u]);
            s[0][u] *= LOW;
            #pragma unroll
            for (u32 i = 0; i < NK; ++i) s[0][u] = MFMA16(k8[i], q1[0][i].v, s[0][u]);"""
    else:
        scores = f"""f4 low[NQ];
            #pragma unroll
            for (u32 a = 0; a < NQ; ++a) s[a][u] = low[a] = (f4){{0.f, 0.f, 0.f, 0.f}};
            #pragma unroll
            for (u32 i = 0; i < NK; ++i) {{
                const h8 k8 = widen({half});
                #pragma unroll
                for (u32 a = 0; a < NQ; ++a) {{
                    low[a] = MFMA16(k8, q2[a][i].v, low[a]);
                    s[a][u] = MFMA16(k8, q1[a][i].v, s[a][u]);
                }}
            }}
            #pragma unroll
            for (u32 a = 0; a < NQ; ++a)
                #pragma unroll
                for (u32 i = 0; i < 4u; ++i) s[a][u][i] = fmaf(low[a][i], LOW, s[a][u][i]);"""
    src = f"""{PRELUDE}{_CACHE8}{_cache8_layout(DP)}#define ND {ND}u
#define NK {NK}u
#define NQ {NQ}u
#define W {W}u
typedef u32 u2 __attribute__((ext_vector_type(2)));
typedef u32 u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
union H8 {{ h8 v; h2 p[4]; _Float16 e[8]; u32 w[4]; }};
#define MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)
#define MFMA32(a, b, c) __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0)
#define NINF (-__builtin_inff())
#define LOW 4.8828125e-4f                                                        // 2^-11
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
// two numbers as hi + lo / 2^11 in 16-bit floats.  minus is -1 where the compiler does not see it: the subtraction, which is exact, then
// takes the 16-bit float as it is, in one mixed multiply-add
static __device__ __forceinline__ void halves(float a, float b, float minus, h2& hi, h2& lo) {{
    const f2 x = {{a, b}};
    hi = __builtin_convertvector(x, h2);
    const f2 z = {{fmaf((float)hi.x, minus, a) * 2048.0f, fmaf((float)hi.y, minus, b) * 2048.0f}};
    lo = __builtin_convertvector(z, h2);
}}
// the largest of the four lanes r, r + 16, r + 32, r + 48: the swaps leave one half of a pair in each operand
static __device__ __forceinline__ float four_max(float x) {{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}}
struct Inside {{ static constexpr bool edge = false; }};
struct Edge {{ static constexpr bool edge = true; }};
extern "C" __global__ __launch_bounds__({bounds}) void {name}(const float* __restrict__ q, const unsigned char* __restrict__ kc,
        const unsigned char* __restrict__ vc, const float* __restrict__ scales, const float* __restrict__ tail_k, const float* __restrict__ tail_v,
        const u32* __restrict__ marks, const u32* __restrict__ wrote, const float* __restrict__ lengths, const float* __restrict__ counts, float* __restrict__ y,
        float* __restrict__ part,
        u32 B, u32 T, u32 H, u32 group, u32 d, u32 NB, u32 tiles, u32 splits, u32 q_wide, float scale) {{
    __shared__ float so[W][16][DP + 4u];
    __shared__ float sm[W][16], sl[W][16];
    const u32 t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63u, r = lane & 15u, g = lane >> 4;
    // workgroups go round the eight dies: all of a key head's on one, whose L2 then holds its codes once
    const u32 per = tiles * splits, spread = (B * H) % 8u == 0u ? 8u : 1u, at0 = blockIdx.x / spread;
    const u32 bh = (at0 / per) * spread + blockIdx.x % spread, b = bh / H, h = bh % H;
    const u32 split = at0 % splits, tile = (at0 / splits) % tiles;
    const u32 rows = T * group, row0 = tile * (16u * NQ), row1 = min(row0 + 16u * NQ, rows) - 1u, t0 = row0 / group, t1 = row1 / group;
    const u64 C = (u64)H * group * d;
    // this lane's quarter of its query rows: on its way while the lengths are
    float raw[NQ][{Q4}];
    #pragma unroll
    for (u32 a = 0; a < NQ; ++a) {{
        const u32 row = min(row0 + 16u * a + r, rows - 1u);
        const float* __restrict__ qrow = q + ((u64)b * T + row / group) * C + (u64)(h * group + row % group) * d;
        if (q_wide) {{                                                        // rows of whole 16-byte items
            #pragma unroll
            for (u32 i = 0; i < {Q4 // 4}u; ++i) *reinterpret_cast<f4*>(&raw[a][4u * i]) = *reinterpret_cast<const f4*>(qrow + min(g * {Q4}u + 4u * i, d - 4u));
        }} else {{
            #pragma unroll
            for (u32 i = 0; i < {Q4}u; ++i) raw[a][i] = qrow[min(g * {Q4}u + i, d - 1u)];
        }}
    }}
    u32 len, n;
    cache8_extent(lengths, counts, b, T, NB * 64u, len, n);
    n = min(n, wrote[b]);                                                       // (a query whose key was not written is a padded row)
    #pragma unroll
    for (u32 a = 0; a < NQ; ++a)
        #pragma unroll
        for (u32 i = 0; i < {Q4}u; ++i) asm volatile("" : "+v"(raw[a][i]));           // (or each would be loaded where it is chosen, one after the other)
    const u32 last = (len + n) >> 6;                                           // blocks below it are codes
    const u32 most = t0 < n ? len + min(t1, n - 1u) + 1u : 0u;                   // positions that the last query of the tiles sees
    const u32 least = t1 < n ? len + t0 + 1u : 0u;                              // ... and the first (a padded row: none)
    const float l2 = fabsf(scale) * 1.44269504088896340736f;
    float minus = -1.0f;
    asm volatile("" : "+v"(minus));
    // the rows as two 16-bit floats an element; the sign of the scale goes with them
    H8 q1[NQ][NK], q2[NQ][NK];
    float back[NQ];
    u32 see[NQ];                                                              // positions this lane's queries see
    #pragma unroll
    for (u32 a = 0; a < NQ; ++a) {{
        const u32 row = row0 + 16u * a + r, tq = row / group;
        const bool live = row < rows && tq < n;
        see[a] = live ? len + tq + 1u : 0u;
        float f[{Q4}], mx = 0.0f;
        #pragma unroll
        for (u32 i = 0; i < {Q4}u; ++i) {{
            f[i] = live && g * {Q4}u + i < d ? raw[a][i] : 0.0f;
            mx = fmaxf(mx, fabsf(f[i]));
        }}
        mx = four_max(mx);
        const int e = max((int)((__float_as_uint(mx) >> 23) & 255u), 27) - 127;      // 2^e <= mx < 2^(e + 1)
        const float up = copysignf(__uint_as_float((u32)(14 - e + 127) << 23), scale);
        back[a] = __uint_as_float((u32)(e - 14 + 127) << 23) * l2;
        #pragma unroll
        for (u32 i = 0; i < {Q4 // 2}u; ++i) halves(f[2u * i] * up, f[2u * i + 1u] * up, minus, q1[a][i >> 2].p[i & 3u], q2[a][i >> 2].p[i & 3u]);
    }}
    f4 o[NQ][ND];
    float m[NQ], l[NQ];
    #pragma unroll
    for (u32 a = 0; a < NQ; ++a) {{
        m[a] = NINF; l[a] = 0.0f;
        #pragma unroll
        for (u32 dt = 0; dt < ND; ++dt) o[a][dt] = (f4){{0.f, 0.f, 0.f, 0.f}};
    }}
    const u32 nb = min(last, (most + 63u) >> 6);                                    // blocks of codes that the tiles see
    const u32 j0 = (u32)((u64)nb * split / splits) + w, j1 = (u32)((u64)nb * (split + 1u) / splits);
    const u64 base = ((u64)bh * NB) * (64u * DP);
    const unsigned char* __restrict__ kh = kc + base + lane * {4 * kn}u;
    const unsigned char* __restrict__ vh = vc + base + lane * 16u;
    const float2* __restrict__ sh = reinterpret_cast<const float2*>(scales) + (u64)bh * NB;
    u{kn} kr[4][{kw}];
    u4 vr[ND];
    // lane i keeps the scales of this wavefront's i-th block, 64 blocks at a time: none is waited for inside a block
    float2 sc = make_float2(0.0f, 0.0f);
    auto load_k = [&](u32 j) {{
        const unsigned char* __restrict__ p = kh + (u64)j * (64u * DP);
        #pragma unroll
        for (u32 u = 0; u < 4u; ++u)
            #pragma unroll
            for (u32 i = 0; i < {kw}u; ++i) kr[u][i] = {fetch_k};
    }};
    auto load_v = [&](u32 j) {{
        const unsigned char* __restrict__ p = vh + (u64)j * (64u * DP);
        #pragma unroll
        for (u32 dt = 0; dt < ND; ++dt) vr[dt] = {fetch_v};
    }};
    if (j0 < j1) {{ load_k(j0); load_v(j0); }}
    auto block = [&](u32 j, auto kind) {{
        constexpr bool edge = decltype(kind)::edge;                                 // some query does not see all of the block
        const u32 jn = j + W < j1 ? j + W : j, nth = ((j - j0) / W) & 63u;             // (the last one is loaded again)
        if (nth == 0u) {{
            sc = sh[min(j + W * lane, j1 - 1u)];
            asm volatile("" : "+v"(sc.x), "+v"(sc.y));                              // (waited for here, not by every block)
        }}
        const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc.x), nth));
        const float vs0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc.y), nth));
        f4 s[NQ][4];
        #pragma unroll
        for (u32 u = 0; u < 4u; ++u) {{
            {scores}
        }}
        load_k(jn);
        const u32 at = j * 64u + 16u * g;
        const float vs = vs0 == vs0 ? vs0 : 0.0f;                           // (a NaN scale makes the scores NaN as well)
        H8 p1[NQ][2], p2[NQ][2];
        #pragma unroll
        for (u32 a = 0; a < NQ; ++a) {{
            if constexpr (edge) {{
                #pragma unroll
                for (u32 i = 0; i < 16u; ++i) if (at + i >= see[a]) s[a][i >> 2][i & 3u] = NEG_FLT_MAX;
            }}
            float mx = s[a][0][0];
            #pragma unroll
            for (u32 i = 1; i < 16u; ++i) mx = fmaxf(mx, s[a][i >> 2][i & 3u]);
            mx = four_max(mx);
            const float f = back[a] * ks;                                        // not negative: the maximum stays one
            float top = mx * f;
            if constexpr (edge) top = j * 64u < see[a] ? top : NINF;                  // (a query that sees none of the block: f may be 0)
            const float mn = fmaxf(m[a], top), mu = mn == NINF ? 0.0f : mn;
            if (__any(mn != m[a])) {{                                               // (a maximum that stays is the rule after the first blocks)
                const float alpha = __builtin_amdgcn_exp2f(m[a] - mu);
                m[a] = mn;
                l[a] *= alpha;
                #pragma unroll
                for (u32 dt = 0; dt < ND; ++dt) o[a][dt] *= alpha;
            }}
            float sum = 0.0f, up = 15.0f - mu;
            if (__any(fabsf(mu) >= 65536.0f)) {{                                     // (roundings of mu could carry p beyond 16-bit floats: first s - mx, exact near 0)
                up = (top - mu) + 15.0f;
                #pragma unroll
                for (u32 i = 0; i < 16u; ++i) s[a][i >> 2][i & 3u] -= mx;
            }}
            #pragma unroll
            for (u32 i = 0; i < 16u; i += 2u) {{
                float p = __builtin_amdgcn_exp2f(fmaf(s[a][i >> 2][i & 3u], f, up));
                float z = __builtin_amdgcn_exp2f(fmaf(s[a][i >> 2][(i & 3u) + 1u], f, up));
                if constexpr (edge) {{ p = at + i < see[a] ? p : 0.0f; z = at + i + 1u < see[a] ? z : 0.0f; }}
                sum += p + z;
                halves(p, z, minus, p1[a][i >> 3].p[(i & 7u) >> 1], p2[a][i >> 3].p[(i & 7u) >> 1]);
            }}
            l[a] += sum;
        }}
        #pragma unroll
        for (u32 dt = 0; dt < ND; ++dt) {{
            const h8 v0 = widen(vr[dt].x, vr[dt].y), v1 = widen(vr[dt].z, vr[dt].w);
            #pragma unroll
            for (u32 a = 0; a < NQ; ++a) {{
                f4 acc = (f4){{0.f, 0.f, 0.f, 0.f}}, low = acc;
                low = MFMA16(v0, p2[a][0].v, low);
                acc = MFMA16(v0, p1[a][0].v, acc);
                low = MFMA16(v1, p2[a][1].v, low);
                acc = MFMA16(v1, p1[a][1].v, acc);
                #pragma unroll
                for (u32 i = 0; i < 4u; ++i) o[a][dt][i] = fmaf(vs, fmaf(low[i], LOW, acc[i]), o[a][dt][i]);
            }}
        }}
        load_v(jn);
    }};
    u32 j = j0;
    for (; j < j1 && j * 64u + 64u <= least; j += W) block(j, Inside());
    for (; j < j1; j += W) block(j, Edge());
    const u32 tt = W - 1u - w;                                                      // sixteen tokens of the tail: the wavefronts with the fewest blocks
    if (split == splits - 1u && tt < 4u && most > last * 64u + 16u * tt) {{
        const u64 heads = (u64)B * H;
        const float* __restrict__ tk = tail_k + (((u64)(last & 1u) * heads + bh) * 64u + 16u * tt) * DP;
        const float* __restrict__ tv = tail_v + (((u64)(last & 1u) * heads + bh) * 64u + 16u * tt) * DP;
        const u32 p0 = last * 64u + 16u * tt + 4u * g;                              // this lane's four tokens
        const u32 mark = marks[CACHE8_MARKS * bh + (last & 1u)];
        float kt[{Q4}], vt[ND][4];                                                  // (both on their way before the first is used)
        #pragma unroll
        for (u32 i = 0; i < {Q4}u; ++i) kt[i] = tk[r * DP + g * {Q4}u + i];
        #pragma unroll
        for (u32 dt = 0; dt < ND; ++dt)
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) vt[dt][i] = tv[(4u * g + i) * DP + dt * 16u + r];
        const bool kept = cache8_kept(mark, last, (len + n) & 63u);                     // (else: NaN to every query that sees some of it)
        #pragma unroll
        for (u32 a = 0; a < NQ; ++a) {{
            const float turn = kept ? back[a] : __builtin_nanf("");
            f4 acc = (f4){{0.f, 0.f, 0.f, 0.f}};
            #pragma unroll
            for (u32 i = 0; i < {Q4}u; ++i) acc = MFMA32(kt[i], fmaf((float)q2[a][i >> 3].e[i & 7u], LOW, (float)q1[a][i >> 3].e[i & 7u]), acc);
            float mx = NINF;
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) {{
                acc[i] = p0 + i < see[a] ? acc[i] * turn : NINF;
                mx = fmaxf(mx, acc[i]);
            }}
            mx = four_max(mx);
            const float mn = fmaxf(m[a], mx), mu = mn == NINF ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m[a] - mu);
            m[a] = mn;
            float sum = 0.0f;
            #pragma unroll
            for (u32 i = 0; i < 4u; ++i) {{ acc[i] = __builtin_amdgcn_exp2f(acc[i] - mu + 15.0f); sum += acc[i]; }}
            l[a] = l[a] * alpha + sum;
            #pragma unroll
            for (u32 dt = 0; dt < ND; ++dt) {{
                #pragma unroll
                for (u32 i = 0; i < 4u; ++i) o[a][dt][i] *= alpha;
                #pragma unroll
                for (u32 i = 0; i < 4u; ++i) {{
                    const float x = vt[dt][i];
                    o[a][dt] = MFMA32((p0 + i < most && x == x) ? x : 0.0f, acc[i], o[a][dt]);  // (a NaN row makes the scores NaN as well)
                }}
            }}
        }}
    }}
    #pragma unroll
    for (u32 a = 0; a < NQ; ++a) {{
        l[a] += __shfl_xor(l[a], 16, WAVE);
        l[a] += __shfl_xor(l[a], 32, WAVE);
        if (a) __syncthreads();                                                     // (the tile before has been read)
        if (g == 0u) {{ sm[w][r] = m[a]; sl[w][r] = l[a]; }}
        #pragma unroll
        for (u32 dt = 0; dt < ND; ++dt) *reinterpret_cast<f4*>(&so[w][r][dt * 16u + 4u * g]) = o[a][dt];
        __syncthreads();
        // 4 W threads a row: the wavefronts' parts, in their order
        const u32 jr = t / (4u * W), jc = t % (4u * W), jrow = row0 + 16u * a + jr;
        if (jrow < rows) {{
            float M = NINF, L = 0.0f, fac[W];
            #pragma unroll
            for (u32 i = 0; i < W; ++i) M = fmaxf(M, sm[i][jr]);
            #pragma unroll
            for (u32 i = 0; i < W; ++i) {{ fac[i] = sm[i][jr] == NINF ? 0.0f : __builtin_amdgcn_exp2f(sm[i][jr] - M); L += fac[i] * sl[i][jr]; }}
            float* __restrict__ yr = splits == 1u ? y + ((u64)b * T + jrow / group) * C + (u64)(h * group + jrow % group) * d
                                                  : part + (((u64)bh * rows + jrow) * splits + split) * (DP + 2u);
            const float inv = splits > 1u ? 1.0f : L == 0.0f ? 0.0f : 1.0f / L;
            for (u32 c = jc; c < d; c += 4u * W) {{
                float x = 0.0f;
                #pragma unroll
                for (u32 i = 0; i < W; ++i) x += fac[i] * so[i][jr][c];
                yr[c] = x * inv;
            }}
            if (splits > 1u && jc == 0u) {{ yr[DP] = M; yr[DP + 1u] = L; }}
        }}
    }}
}}
"""
    return src, name, _fmt("P" * 12, "I" * 9, "f")


CACHE8_MAX_SPLITS = 64      # what one wavefront joins: a lane per split


@cache
def cache8_join_kernel(DP: int) -> tuple[str, str, str]:
    """Adds up what cache8_attend_kernel left per split: O = sum exp(m_s - M) O_s over sum exp(m_s - M) l_s.  One wavefront per query
    row of a key head: lane s takes m and l of split s (at most 64), the factors go round, and the columns are added in the order of
    the splits with eight loads in flight.  Bound by latency: two dependent reads (512 rows of 4 splits: 4.7 us)."""
    name = f"cache8_join_d{DP}"
    N = (DP + 63) // 64
    src = f"""{PRELUDE}
#define DP {DP}u
#define NINF (-__builtin_inff())
extern "C" __global__ __launch_bounds__(256) void {name}(const float* __restrict__ part, float* __restrict__ y,
        u32 items, u32 T, u32 H, u32 group, u32 d, u32 splits) {{
    const u32 item = blockIdx.x * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    if (item >= items) return;
    const u32 rows = T * group, bh = item / rows, row = item % rows, b = bh / H, h = bh % H;
    const float* __restrict__ pr = part + (u64)item * splits * (DP + 2u);
    const float2 ml = lane < splits ? *reinterpret_cast<const float2*>(pr + lane * (DP + 2u) + DP) : make_float2(NINF, 0.0f);
    const float M = wave_max(ml.x), f = ml.x == NINF ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M), L = wave_sum(f * ml.y);
    float acc[{N}];
    #pragma unroll
    for (u32 i = 0; i < {N}u; ++i) acc[i] = 0.0f;
    #pragma unroll 8
    for (u32 s = 0; s < splits; ++s) {{
        const float fs = __shfl(f, (int)s, WAVE);
        #pragma unroll
        for (u32 i = 0; i < {N}u; ++i) {{ const u32 c = i * 64u + lane; if (c < d) acc[i] += fs * pr[s * (DP + 2u) + c]; }}
    }}
    float* __restrict__ yr = y + ((u64)b * T + row / group) * ((u64)H * group * d) + (u64)(h * group + row % group) * d;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    #pragma unroll
    for (u32 i = 0; i < {N}u; ++i) {{ const u32 c = i * 64u + lane; if (c < d) yr[c] = acc[i] * inv; }}
}}
"""
    return src, name, _fmt("P" * 2, "I" * 6)
