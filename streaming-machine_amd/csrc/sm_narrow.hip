// Operators in few bits: plates of 8-bit digits (sm_plate8_*), a cache of 4 or 8-bit digits and the attention over it
// (sm_narrow_*).  Kernels first, then their entry points.
//
// A row's digits of b bits (the machine's to16, base2.py:24-27, at b bits):
//     sh = max(bitlen(OR |x|) - (b - 1), 0),   digit = clamp(rsh(x, sh), -2^(b-1), 2^(b-1) - 1)
// worth digit 2^sh each at the row's own scale; sh is the row's level, kept in one byte (0 .. 60).
//
// Digits that the matrix units contract stand in the operands' order of v_mfma_i32_16x16x64_i8 (lane l: row or column
// l % 16, bytes k = 16 (l / 16) + b), so an operand is one 16-byte load a lane, no lane's bytes are moved between lanes
// and a wave's loads are 1 KB in a row.
#define NTHREADS 256
// Results of NARROW_STREAM bytes and more are stored past the caches (nontemporal): left in the 256 MB behind them, a large
// result is written out while the next kernel reads, which then takes half as long again (three prompts of 2,048 rows
// written and read back 37 against 50 us, 4,096 rows 4,096 -> 11,008 249 against 270 us).  Smaller ones stay cached for
// whoever reads them (64 rows 768 -> 50,257 18.2 us stored past the caches, 17.2 not), and so do rows that share their lines
// of 128 bytes: past the caches such a line is written in parts (193 rows 364 -> 46,797 65 us, 33 cached).
#define NARROW_STREAM (64 << 20)
typedef i64 i64x2 __attribute__((ext_vector_type(2), aligned(8)));       // (rows stand at 8 bytes' alignment only)
template <bool NT> SMD void put(i64* p, i64 v) {
    if constexpr (NT) __builtin_nontemporal_store(v, p);
    else *p = v;
}
template <bool NT> SMD void put2(i64* p, i64 v, i64 w) {
    if constexpr (NT) __builtin_nontemporal_store(i64x2{v, w}, reinterpret_cast<i64x2*>(p));
    else *reinterpret_cast<i64x2*>(p) = i64x2{v, w};
}

// x 2^-s rounded half up without the sum that wraps near 2^63 (s in 0 .. 63)
SMD i64 rsh_round(i64 x, int s) { return s > 0 ? (x >> s) + ((x >> (s - 1)) & 1) : x; }
SMD int digit_level(u64 orr, int bits) {
    const int top = bitlen_u(orr);
    return top > bits - 1 ? top - (bits - 1) : 0;
}
SMD int digit_of(i64 x, int sh, int bits) {
    const i64 v = rsh_round(x, sh), hi = (1 << (bits - 1)) - 1;
    return (int)(v > hi ? hi : v < -hi - 1 ? -hi - 1 : v);
}
// the same digits of a row whose level shows that its values fit 32 bits (sh < 32 - bits; the low words then hold them): four
// steps a value in place of some twenty of 64 bits.  Only the upper end is ever clamped.
SMD int digit_short(int x, int sh, int bits) {
    const int v = (x >> sh) + (int)(sh ? __builtin_amdgcn_ubfe((unsigned)x, (unsigned)sh - 1, 1) : 0);
    return min(v, (1 << (bits - 1)) - 1);
}
SMD bool digits_short(int sh, int bits) { return sh < 32 - bits; }
SMD u64 mag64(i64 x) { return x < 0 ? (u64)0 - (u64)x : (u64)x; }
// the OR over a wave of 64-bit values, in every lane
SMD u64 wave_or_u64(u64 v) { return (u64)wave_or64((i64)v); }

// ---------------------------------------------------------------------------------------------------------
// the product with 8-bit digits
struct Narrow8Args {
    const signed char* W;        // [column tiles of 16][K / 64][lane][16]
    const int* we; const i64* wb;
    int nin, K, N;               // inputs, inputs up to a multiple of 64, columns
    const i64* X; i64 ldx; int rows;
    signed char* lights;         // [row tiles of 16][K / 64][lane][16]
    int* level;                  // [rows] the rows' sh (ex = sh - 16)
    i64* out; i64 ldo;
};

// four digits of a row as bytes
SMD unsigned digit_quad(const i64 v[4], int sh) {
    unsigned w = 0;
    if (digits_short(sh, 8)) {
#pragma unroll
        for (int i = 0; i < 4; i++) w |= (unsigned)(digit_short((int)v[i], sh, 8) & 255) << (8 * i);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) w |= (unsigned)(digit_of(v[i], sh, 8) & 255) << (8 * i);
    }
    return w;
}
// four values of a row from place 4 q, zeros past its end
SMD void row_quad(const i64* x, int q, int nin, i64 v[4]) {
    if (4 * q + 3 < nin) {
        const i64x2 lo = *reinterpret_cast<const i64x2*>(x + 4 * q), hi = *reinterpret_cast<const i64x2*>(x + 4 * q + 2);
        v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = 4 * q + i < nin ? x[4 * q + i] : 0;
    }
}
// two values of a row from place i, zeros past its end
SMD i64x2 row_pair(const i64* x, int i, int nin) {
    if (i + 1 < nin) return *reinterpret_cast<const i64x2*>(x + i);
    return i64x2{i < nin ? x[i] : 0, 0};
}
// One block a row: the row's level, then its digits in the operand's order.  A thread loads two values in a row, so that a
// wave's load is 1 KB in a row (16 bytes every 32, four values a thread, touch each line twice: 53 us at 4096 rows of 4096),
// and pairs of threads swap halves to store four digits each.  Rows of up to 8,192 values are held in registers between the
// two passes, longer ones are read again.  The 16 rows of a tile share their 128-byte lines of digits: with many rows,
// blocks of one die (every eighth) take one tile, so that the lines fill in that die's L2.  Bound by the rows' read: 4096
// rows of 4096 in 31 us, 4.9 TB/s.
__global__ __launch_bounds__(NTHREADS) void k_narrow_lights(Narrow8Args a) {
    constexpr int HOLD = 8, STEP = 4 * NTHREADS;
    __shared__ u64 wor[NTHREADS / 64];
    const int b = blockIdx.x, r = gridDim.x >= 128 ? ((b >> 7) * 8 + (b & 7)) * 16 + ((b >> 3) & 15) : b;
    const int tid = threadIdx.x;
    if (r >= a.rows) return;
    const i64* x = a.X + (i64)r * a.ldx;
    struct Four { i64x2 lo, hi; };                                   // places i + 2 tid and i + STEP / 2 + 2 tid
    auto load = [&](int i) { return Four{row_pair(x, i + 2 * tid, a.nin), row_pair(x, i + STEP / 2 + 2 * tid, a.nin)}; };
    auto mags = [](const Four& f) { return mag64(f.lo[0]) | mag64(f.lo[1]) | mag64(f.hi[0]) | mag64(f.hi[1]); };
    Four held[HOLD];
    u64 orr = 0;
#pragma unroll
    for (int s = 0; s < HOLD; s++)
        if (s * STEP < a.K) {
            held[s] = load(s * STEP);
            orr |= mags(held[s]);
        }
    for (int i = HOLD * STEP; i < a.K; i += STEP) orr |= mags(load(i));
    orr = wave_or_u64(orr);
    if ((tid & 63) == 0) wor[tid >> 6] = orr;
    __syncthreads();
    orr = 0;
#pragma unroll
    for (int i = 0; i < NTHREADS / 64; i++) orr |= wor[i];
    const int sh = digit_level(orr, 8);
    if (tid == 0) a.level[r] = sh;
    signed char* o = a.lights + (i64)(r >> 4) * a.K * 16 + (r & 15) * 16;
    const bool odd = tid & 1;
    auto store = [&](int i, const Four& f) {
        const i64 v[4] = {f.lo[0], f.lo[1], f.hi[0], f.hi[1]};
        const unsigned d = digit_quad(v, sh);                        // low half: the first place's two
        const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)d, 0xB1, 0xf, 0xf, false);      // the thread beside
        const unsigned w = odd ? (other >> 16) | (d & 0xFFFF0000u) : (d & 0xFFFFu) | (other << 16);
        const int k = i + (odd ? STEP / 2 + 2 * tid - 2 : 2 * tid);
        if (k < a.K) *reinterpret_cast<unsigned*>(o + (i64)(k >> 6) * 1024 + ((k >> 4) & 3) * 256 + (k & 15)) = w;
    };
#pragma unroll
    for (int s = 0; s < HOLD; s++)
        if (s * STEP < a.K) store(s * STEP, held[s]);
    for (int i = HOLD * STEP; i < a.K; i += STEP) store(i, load(i));
}

SMD v4i mfma8(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
// rsh(pile, -(e + ex + 16)) + b; a pile shifted right by 32 places or more rounds to 0
SMD i64 narrow_out(int pile, int we, int sh, i64 wb) {
    const int s = -(we + sh);
    if (s <= 0) return wadd(shl(pile, -s), wb);
    return wadd(s > 31 ? 0 : (pile >> s) + ((pile >> (s - 1)) & 1), wb);
}

// Few values (rows ceil(K / 1024) <= 8): a block a column tile forms the rows' digits itself, in LDS, while its first weights
// are on their way, and its four waves take a quarter of the inputs each.  One launch in place of two: a call is then
// bound by its launch.
constexpr int FEW_QUADS = 8;
__global__ __launch_bounds__(NTHREADS) void k_narrow_one(Narrow8Args a) {
    constexpr int AHEAD = 4;
    __shared__ __attribute__((aligned(16))) signed char x8[FEW_QUADS * 1024];      // [K / 16][rows][16]
    __shared__ u64 wor[FEW_QUADS][4];
    __shared__ int lev[FEW_QUADS];
    __shared__ v4i part[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int kbs = a.K / 64, per = (kbs + 3) / 4, k0 = wave * per, k1 = min(kbs, k0 + per), quads = a.K / 4;
    const v4i* wp = reinterpret_cast<const v4i*>(a.W + (i64)blockIdx.x * a.K * 16) + lane;
    v4i w[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
        if (k0 + i < k1) w[i] = wp[(k0 + i) * 64];
    const int S = (quads + NTHREADS - 1) / NTHREADS, used = a.rows * S;
    i64 v[FEW_QUADS][4];
#pragma unroll
    for (int i = 0; i < FEW_QUADS; i++) {
        const int q = tid + i % S * NTHREADS;
        if (i < used && q < quads) row_quad(a.X + (i64)(i / S) * a.ldx, q, a.nin, v[i]);
        else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0;
    }
#pragma unroll
    for (int i = 0; i < FEW_QUADS; i++)
        if (i < used) {
            const u64 o = wave_or_u64(mag64(v[i][0]) | mag64(v[i][1]) | mag64(v[i][2]) | mag64(v[i][3]));
            if (lane == 0) wor[i][wave] = o;
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FEW_QUADS; i++) {
        const int r = i / S, q = tid + i % S * NTHREADS;
        if (i >= used) continue;
        u64 o = 0;
        for (int j = r * S; j < (r + 1) * S; j++) o |= wor[j][0] | wor[j][1] | wor[j][2] | wor[j][3];
        const int sh = digit_level(o, 8);
        if (tid == 0) lev[r] = sh;
        if (q >= quads) continue;
        *reinterpret_cast<unsigned*>(x8 + ((q >> 2) * a.rows + r) * 16 + 4 * (q & 3)) = digit_quad(v[i], sh);
    }
    __syncthreads();
    v4i acc = {};
    const signed char* xr = x8 + min(n, a.rows - 1) * 16;
    for (int k = k0; k < k1; k += AHEAD)
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (k + i < k1) {
                acc = mfma8(*reinterpret_cast<const v4i*>(xr + (4 * (k + i) + g) * a.rows * 16), w[i], acc);
                if (k + i + AHEAD < k1) w[i] = wp[(k + i + AHEAD) * 64];
            }
    part[wave][lane] = acc;
    __syncthreads();
    const int col = blockIdx.x * 16 + n, row = 4 * g + wave;               // wave w finishes every fourth row
    if (col >= a.N || row >= a.rows) return;
    const int pile = part[0][lane][wave] + part[1][lane][wave] + part[2][lane][wave] + part[3][lane][wave];
    a.out[(i64)row * a.ldo + col] = narrow_out(pile, a.we[col], lev[row], a.wb[col]);
}

// RT row tiles by CT column tiles a wave, the inputs split over KW of a block's four waves and their piles added: weights and
// lights straight from memory into operands, four steps' loads in flight.  Bound by the weights' read and the results' write:
// 64 rows 768 -> 50257 in 17.5 us, 3.7 TB/s; a column tile a wave without the split took 52 us against 25 at 8192 -> 8192.
template <int RT, int CT, int KW>
__global__ __launch_bounds__(NTHREADS) void k_narrow_rows(Narrow8Args a) {
    constexpr int CG = 4 / KW, TILES = RT * CT;
    __shared__ v4i part[4][TILES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ks = wave % KW, cg = wave / KW;
    const int kbs = a.K / 64, per = (kbs + KW - 1) / KW, k0 = ks * per, k1 = min(kbs, k0 + per);
    const int nt = (a.N + 15) / 16, ct0 = (blockIdx.x * CG + cg) * CT, rt0 = blockIdx.y * RT, rts = (a.rows + 15) / 16;
    const v4i *wp[CT], *lp[RT];
#pragma unroll
    for (int c = 0; c < CT; c++) wp[c] = reinterpret_cast<const v4i*>(a.W + (i64)min(ct0 + c, nt - 1) * a.K * 16) + lane;
#pragma unroll
    for (int r = 0; r < RT; r++) lp[r] = reinterpret_cast<const v4i*>(a.lights + (i64)min(rt0 + r, rts - 1) * a.K * 16) + lane;
    v4i acc[RT][CT] = {};
    auto steps = [&](int k, auto many) {
        constexpr int U = decltype(many)::value;
        v4i w[U][CT], x[U][RT];
#pragma unroll
        for (int i = 0; i < U; i++) {
#pragma unroll
            for (int c = 0; c < CT; c++) w[i][c] = wp[c][(k + i) * 64];
#pragma unroll
            for (int r = 0; r < RT; r++) x[i][r] = lp[r][(k + i) * 64];
        }
#pragma unroll
        for (int i = 0; i < U; i++)
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int c = 0; c < CT; c++) acc[r][c] = mfma8(x[i][r], w[i][c], acc[r][c]);
    };
    int k = k0;
    for (; k + 4 <= k1; k += 4) steps(k, std::integral_constant<int, 4>());
    for (; k < k1; k++) steps(k, std::integral_constant<int, 1>());
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int c = 0; c < CT; c++) part[wave][r * CT + c][lane] = acc[r][c];
    __syncthreads();
    for (int t = ks; t < TILES; t += KW) {       // the tiles' piles, shared out over the inputs' waves
        v4i p = part[cg * KW][t][lane];
#pragma unroll
        for (int i = 1; i < KW; i++) p += part[cg * KW + i][t][lane];
        const int col = (ct0 + t % CT) * 16 + (lane & 15);
        if (col >= a.N) continue;
        const int we = a.we[col];
        const i64 wb = a.wb[col];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = (rt0 + t / CT) * 16 + 4 * (lane >> 4) + i;
            if (row < a.rows) a.out[(i64)row * a.ldo + col] = narrow_out(p[i], we, a.level[row], wb);
        }
    }
}

// The product of many rows: WR x WC waves of RT x CT tiles each.  Every step of 64 inputs is a stage of (WR RT + WC CT)
// fragments of 1 KB, loaded from memory straight into LDS in the operands' order (so neither the loads nor the operand
// reads rearrange anything and no two lanes meet in a bank), three stages ahead; a stage's operands are read into registers
// while the stage before is multiplied (255 us at 4096 rows 4096 -> 11008 with the reads in the same step, 200 so).  Bound by
// the matrix units: 1,850 TOP/s there with the results' 360 MB written (a large library product of bytes reaches 2,285).
typedef const __attribute__((address_space(1))) void* gas_p;
typedef __attribute__((address_space(3))) void* las_p;
template <int WR, int WC, int RT, int CT, bool NT>
__global__ __launch_bounds__(64 * WR * WC, 2) void k_narrow_tiles(Narrow8Args a, int tr, int tc) {
    constexpr int W = WR * WC, AF = WR * RT, F = AF + WC * CT, LPW = F / W;
    static_assert(F % W == 0, "every wave loads the same number of fragments");
    __shared__ v4i s0[F * 64], s1[F * 64], s2[F * 64], s3[F * 64];
    // consecutive blocks go to the eight dies in turn: each takes a run of tiles, eight row tiles by turns, so that the
    // blocks that share a die's L2 share their rows and columns
    const int per = (tr * tc + 7) / 8, l = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || l >= tr * tc) return;
    const int grp = l / (8 * tc), gr = min(8, tr - grp * 8), in = l - grp * 8 * tc, br = grp * 8 + in % gr, bc = in / gr;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave / WC, wc = wave % WC;
    const int kbs = a.K / 64, rts = (a.rows + 15) / 16, nt = (a.N + 15) / 16;
    const v4i* src[LPW];
#pragma unroll
    for (int i = 0; i < LPW; i++) {
        const int f = wave * LPW + i;
        const signed char* base = f < AF ? a.lights + (i64)min(br * AF + f, rts - 1) * a.K * 16
                                         : a.W + (i64)min(bc * WC * CT + f - AF, nt - 1) * a.K * 16;
        src[i] = reinterpret_cast<const v4i*>(base) + lane;
    }
    auto fetch = [&](v4i* buf, int k) {
        k = min(k, kbs - 1);             // (past the end: the last stage again, never read)
#pragma unroll
        for (int i = 0; i < LPW; i++)
            __builtin_amdgcn_global_load_lds((gas_p)(src[i] + k * 64), (las_p)(buf + (wave * LPW + i) * 64), 16, 0, 0);
    };
    v4i acc[RT][CT] = {};
    struct Operands { v4i x[RT], w[CT]; } even, odd;
    auto read = [&](const v4i* buf, Operands& o) {
#pragma unroll
        for (int r = 0; r < RT; r++) o.x[r] = buf[(wr * RT + r) * 64 + lane];
#pragma unroll
        for (int c = 0; c < CT; c++) o.w[c] = buf[(AF + wc * CT + c) * 64 + lane];
    };
    // Step k's operands are in registers (read from stage k the step before); stage k + 1 is whole once every wave's loads
    // of it have landed (all but the two stages' after it) and the waves have met, and then nobody reads stage k any more:
    // its place takes stage k + 4.
    auto step = [&](v4i* now, const v4i* next, const Operands& o, Operands& on, int k) {
        __builtin_amdgcn_s_waitcnt(0x0070 | ((2 * LPW) & 15) | ((2 * LPW) >> 4) << 14);      // vmcnt(2 LPW) lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        fetch(now, k + 4);
        read(next, on);
        if (k < kbs) {
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int c = 0; c < CT; c++) acc[r][c] = mfma8(o.x[r], o.w[c], acc[r][c]);
        }
    };
    fetch(s0, 0);
    fetch(s1, 1);
    fetch(s2, 2);
    fetch(s3, 3);
    __builtin_amdgcn_s_waitcnt(0x0F70 | ((3 * LPW) & 15) | ((3 * LPW) >> 4) << 14);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(s0, even);
    for (int k = 0; k < kbs; k += 4) {
        step(s0, s1, even, odd, k);
        step(s1, s2, odd, even, k + 1);
        step(s2, s3, even, odd, k + 2);
        step(s3, s0, odd, even, k + 3);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);              // no load into LDS outlives its wave
    const int n = lane & 15, g = lane >> 4;
    int lev[RT][4];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) lev[r][i] = a.level[min((br * AF + wr * RT + r) * 16 + 4 * g + i, a.rows - 1)];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int col = (bc * WC * CT + wc * CT + c) * 16 + n;
        if (col >= a.N) continue;
        const int we = a.we[col];
        const i64 wb = a.wb[col];
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = (br * AF + wr * RT + r) * 16 + 4 * g + i;
                if (row < a.rows) put<NT>(&a.out[(i64)row * a.ldo + col], narrow_out(acc[r][c][i], we, lev[r][i], wb));
            }
    }
}

// an input-major int8 [nin][nout] array into the operand's order (zeros past nin and past nout)
__global__ __launch_bounds__(NTHREADS) void k_narrow_plate(const signed char* w, int nin, int nout, int K, signed char* W, i64 quads) {
    for (i64 q = (i64)blockIdx.x * NTHREADS + threadIdx.x; q < quads; q += (i64)gridDim.x * NTHREADS) {
        const i64 o = q * 4;                                     // [tile][K / 64][lane][16]
        const int b = (int)(o & 15), lane = (int)(o >> 4) & 63;
        const i64 t = o >> 10;
        const int kbs = K / 64, k = (int)(t % kbs) * 64 + (lane >> 4) * 16 + b, col = (int)(t / kbs) * 16 + (lane & 15);
        unsigned v = 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (k + i < nin && col < nout) v |= (unsigned)(unsigned char)w[(i64)(k + i) * nout + col] << (8 * i);
        *reinterpret_cast<unsigned*>(W + o) = v;
    }
}

// ---------------------------------------------------------------------------------------------------------
// the cache.  Each (stream, head) holds tiles of 64 positions: the key digits, the value digits, 64 key levels, 64 value
// levels (wide: the head's row up to 64, 128 or 256 digits, zeros past its dimension).
//   keys    [wide / 16 or 32][64 positions][16 bytes]: byte j is dimension 16 c + j; of 4 bits dimension 32 c + j in its low
//           half and 32 c + 16 + j in its high one
//   values  [wide / 16][4 g][16 m][16 bytes]: dimension 16 c + m, byte 4 t + r position 16 t + 4 g + r; of 4 bits
//           [wide / 32][4 g][16 m][2 h][8 bytes]: dimension 32 c + 16 h + m, byte 4 t + r position 16 t + 4 g + r (t 0, 1) in
//           its low half and the position 32 further in its high one
// A key operand (64 dimensions of 16 positions) and a value operand (64 positions of 16 dimensions) are then loads of 8 or
// 16 bytes a lane in the operand's order; the positions' order within a value operand is the order in which a score
// accumulator holds them (register r of lane group g of tile t), so weights need no exchange where scores stand
// position-major.  A position's key bytes are its own; its value bytes are shared with the position 32 further at 4 bits.
struct NarrowShape { int streams, heads, dim, wide, ctx, bits, tiles; };
SMD i64 narrow_half(const NarrowShape& s) { return (i64)s.wide * 8 * s.bits; }                   // bytes of a tile's keys
SMD i64 narrow_tile(const NarrowShape& s) { return 2 * narrow_half(s) + 128; }
SMD char* narrow_at(char* buf, const NarrowShape& s, int stream, int head, int tile) {
    return buf + (((i64)stream * s.heads + head) * s.tiles + tile) * narrow_tile(s);
}

struct NarrowRows {
    NarrowShape s; char* buf;
    const i64* k; const i64* v; i64* k2; i64* v2;
    i64 row_stride, stream_stride; int rows;
    const int* start; const int* count;
};
// the rows of a call that are in the cache's range: [lo, hi) of its `rows`
SMD void narrow_range(const int* start, const int* count, int stream, int rows, int ctx, i64& p0, i64& lo, i64& hi) {
    p0 = start[stream];
    hi = count ? min(max(count[stream], 0), rows) : rows;
    lo = p0 < 0 ? -p0 : 0;
    hi = min(hi, (i64)ctx - p0);
}

// A block a (tile, head, stream): its rows' levels and digits (a wave a row, four rows' loads in flight), through LDS in the
// units' order (a dimension's positions 16 t + 4 g + r at byte 16 g + 4 t + r), then whole 16-byte units; a unit of values is
// read first where it also holds positions that the call does not write.  Bound by the rows' read: three prompts of 2,048
// rows of 8 heads of 128 in 19 us, 4.5 TB/s.
template <int BITS, int WIDE, int NW>
__global__ __launch_bounds__(64 * NW) void k_narrow_write(NarrowRows a) {
    constexpr int PER = WIDE / 64, AT_ONCE = PER == 4 ? 2 : 4;
    __shared__ __attribute__((aligned(16))) signed char kd[64][WIDE + 4], vd[WIDE][68];
    // (the heads first: blocks that run together read whole rows)
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, head = blockIdx.x % a.s.heads, stream = blockIdx.z;
    i64 p0, lo, hi;
    narrow_range(a.start, a.count, stream, a.rows, a.s.ctx, p0, lo, hi);
    if (lo >= hi) return;
    const i64 first = p0 + lo, last = p0 + hi - 1;                // positions written
    const i64 tile = first / 64 + blockIdx.x / a.s.heads;
    if (tile > last / 64) return;
    const int b0 = (int)max(first - tile * 64, (i64)0), b1 = (int)min(last - tile * 64, (i64)63);    // within the tile
    char* base = narrow_at(a.buf, a.s, stream, head, (int)tile);
    char* lev = base + 2 * narrow_half(a.s);
    const i64 row0 = tile * 64 - p0, at0 = stream * a.stream_stride + (i64)head * a.s.dim;
    for (int b = b0 + wave; b <= b1; b += NW * AT_ONCE) {
        i64 x[AT_ONCE][2][PER];
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            const i64 at = at0 + (row0 + min(b + i * NW, b1)) * a.row_stride;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int d = lane + 64 * j;
                x[i][0][j] = d < a.s.dim ? a.k[at + d] : 0;
                x[i][1][j] = d < a.s.dim ? a.v[at + d] : 0;
            }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            const int p = b + i * NW;
            if (p > b1) break;
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                u64 o = 0;
#pragma unroll
                for (int j = 0; j < PER; j++) o |= mag64(x[i][kv][j]);
                const int sh = digit_level(wave_or_u64(o), BITS);
                if (lane == 0) lev[64 * kv + p] = (char)sh;
#pragma unroll
                for (int j = 0; j < PER; j++) {
                    const int v = digits_short(sh, BITS) ? digit_short((int)x[i][kv][j], sh, BITS) : digit_of(x[i][kv][j], sh, BITS);
                    if (kv == 0) kd[p][lane + 64 * j] = (signed char)v;
                    else vd[lane + 64 * j][16 * (p >> 2 & 3) + 4 * (p >> 4) + (p & 3)] = (signed char)v;
                }
            }
        }
    }
    __syncthreads();
    // the 4-bit digits of two dwords of bytes, the second ones in the high halves
    auto halves = [](int x, int y) { return (int)(((unsigned)x & 0x0F0F0F0Fu) | ((unsigned)y & 0x0F0F0F0Fu) << 4); };
    constexpr int UNITS = WIDE * BITS / 128;                     // 16-byte units a position, or a dimension's 64 / 4
    const bool whole = b0 == 0 && b1 == 63;
    for (int i = tid; i < UNITS * 64; i += 64 * NW) {
        const int c = i >> 6, b = i & 63;
        if (b < b0 || b > b1) continue;
        const int* row = reinterpret_cast<const int*>(kd[b]);
        v4i w;
#pragma unroll
        for (int q = 0; q < 4; q++) w[q] = BITS == 8 ? row[4 * c + q] : halves(row[8 * c + q], row[8 * c + 4 + q]);
        *reinterpret_cast<v4i*>(base + (i64)i * 16) = w;
    }
    char* vbase = base + narrow_half(a.s);
    for (int i = tid; i < UNITS * 64; i += 64 * NW) {
        const int c = i >> 6, g = (i >> 4) & 3, m = i & 15;
        v4i w;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int* row = reinterpret_cast<const int*>(vd[BITS == 8 ? 16 * c + m : 32 * c + 16 * (q >> 1) + m]) + 4 * g;
            w[q] = BITS == 8 ? row[q] : halves(row[q & 1], row[(q & 1) + 2]);
        }
        v4i* u = reinterpret_cast<v4i*>(vbase + (i64)i * 16);
        if (!whole) {
            // the unit's positions 16 t + 4 g + r: which of them the call writes
            unsigned in = 0;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int p = 16 * (j >> 2) + 4 * g + (j & 3);
                in |= (p >= b0 && p <= b1 ? 1u : 0u) << j;
            }
            if (!in) continue;
            const v4i old = *u;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                unsigned take = 0;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (BITS == 8) take |= (in >> (4 * q + j) & 1 ? 255u : 0u) << (8 * j);
                    else take |= ((in >> (4 * (q & 1) + j) & 1 ? 15u : 0u) | (in >> (4 * (q & 1) + 8 + j) & 1 ? 240u : 0u)) << (8 * j);
                w[q] = (int)(((unsigned)w[q] & take) | ((unsigned)old[q] & ~take));
            }
        }
        *u = w;
    }
}

// A thread two dimensions of a (row, head), k and v: 16-byte stores (rows stand at 8 bytes' alignment only).  Bound by what it
// writes, eight bytes a digit: the same three prompts in 16 us, 5.1 TB/s.
template <int BITS, bool NT>
__global__ __launch_bounds__(NTHREADS) void k_narrow_read(NarrowRows a) {
    const int stream = blockIdx.z, pairs = (a.s.dim + 1) / 2, hd = a.s.heads * pairs;
    i64 p0, lo, hi;
    narrow_range(a.start, a.count, stream, a.rows, a.s.ctx, p0, lo, hi);
    const i64 n = (hi - lo) * hd, half = narrow_half(a.s);
    for (i64 i = (i64)blockIdx.x * NTHREADS + threadIdx.x; i < n; i += (i64)gridDim.x * NTHREADS) {
        const int r = n <= UINT_MAX ? (int)((unsigned)i / (unsigned)hd) : (int)(i / hd), w = (int)(i - (i64)r * hd), h = w / pairs, d = 2 * (w - h * pairs);
        const i64 row = lo + r, p = p0 + row;
        const int b = (int)(p & 63), j = 4 * (b >> 4) + (b & 3), g = (b >> 2) & 3;
        const char* base = narrow_at(a.buf, a.s, stream, h, (int)(p >> 6));
        const char* vbase = base + half;
        const unsigned char* lev = reinterpret_cast<const unsigned char*>(vbase + half);
        const int lk = lev[b], lv = lev[64 + b];
        int k[2], v[2];
        if (BITS == 8) {
            const unsigned kb = *reinterpret_cast<const unsigned short*>(base + (d >> 4) * 1024 + b * 16 + (d & 15));
            k[0] = (signed char)kb; k[1] = (signed char)(kb >> 8);
#pragma unroll
            for (int x = 0; x < 2; x++) v[x] = (signed char)vbase[(d >> 4) * 1024 + (16 * g + (d & 15) + x) * 16 + j];
        } else {
            const unsigned kb = *reinterpret_cast<const unsigned short*>(base + (d >> 5) * 1024 + b * 16 + (d & 15)) >> (d & 16 ? 4 : 0);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const unsigned vb = (unsigned char)vbase[(d >> 5) * 1024 + (16 * g + (d & 15) + x) * 16 + 8 * (d >> 4 & 1) + (j & 7)] >> (j & 8 ? 4 : 0);
                k[x] = (int)(kb >> (8 * x) << 28) >> 28;
                v[x] = (int)(vb << 28) >> 28;
            }
        }
        const i64 at = stream * a.stream_stride + row * a.row_stride + (i64)h * a.s.dim + d;
        if (d + 1 < a.s.dim) {
            put2<NT>(a.k2 + at, shl(k[0], lk), shl(k[1], lk));
            put2<NT>(a.v2 + at, shl(v[0], lv), shl(v[1], lv));
        } else {
            a.k2[at] = shl(k[0], lk);
            a.v2[at] = shl(v[0], lv);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// attention over the cache.  A row (stream, row t, query head) at position p = start + t sees positions 0 .. p of its key
// head.  With q's 8-bit digits at level eq (q 2^(F / 65536) = q8 2^eq, a score's scale folded in through the power's fine
// part, base2.py:50-53) and ARR the arrivals (base2.py:97):
//   sc_i = clamp(rsh(sum_d q8_d k_id, -(eq + level_i - 16 + 10)), +-2^30)
//   chunk j (positions 256 j ..):  m_j = max sc, E_j = max value level (of the positions seen),
//       u_i = rsh(ARR[m_j - sc_i], 2), A_j = sum u_i, w_i = rsh(u_i, E_j - level_i), N_j = rsh(sum_i w_i v_i, 8)
//   row:  M = max m_j, E = max E_j, f_j = ARR[M - m_j], A = sum rsh(A_j f_j, 24), N = sum rsh(N_j f_j, 24 + E - E_j)
//   out = power(N, (E + 8) 65536 - log2fix(A))
// Sums of whole numbers: no split of the positions over waves or blocks changes them.  Up to 256 positions this is
// base2.py:93-99 on the digits.
#define NCHUNK 256

struct NarrowAtt {
    NarrowShape s; const char* buf;
    int group, rows, R, J;       // query heads a key head, rows a stream, rows x group, chunks
    const i64* q; i64 q_row, q_stream; i64* out; i64 o_row, o_stream;
    const int* start; const int* count; int span; int F;
    signed char* q8;             // [streams][heads][R][wide]
    int* eq; int* pos;           // [streams][heads][R] the digits' level; the row's position, -1 a row that is not there
    int* pm; int* pA; int* pE; int* pN;     // [streams][heads][J][R] each chunk's m_j, A_j, E_j and (x wide) N_j
    const double* WF;            // ARR's factors (sm_tables): [alen / 128 + 1], [128]
    Tables tb;
};

// the position of a stream's row t, -1 a row that is not there
SMD int narrow_pos(const NarrowAtt& a, int stream, int t) {
    const i64 p = (i64)a.start[stream] + t;
    return t < (a.count ? a.count[stream] : a.rows) && p >= 0 && p < a.span ? (int)p : -1;
}
// one wave: one row's q (zeros past its dimension, and for a row that is not there), its 8-bit digits and their level
template <int PER>
SMD void narrow_q_load(const NarrowAtt& a, const i64* q, bool here, int lane, i64 x[PER]) {
#pragma unroll
    for (int j = 0; j < PER; j++) x[j] = here && lane + 64 * j < a.s.dim ? q[lane + 64 * j] : 0;
}
template <int PER>
SMD int narrow_q_row(const NarrowAtt& a, i64 x[PER], int lane, signed char* dst) {
    u64 o = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) o |= mag64(x[j]);
    const int s16 = digit_level(wave_or_u64(o), 16);
    const i64 e = a.tb.EXP2[a.F & 0xFFFF];
    o = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        x[j] = rsh_round(x[j], s16) * e;
        o |= mag64(x[j]);
    }
    const int s8 = digit_level(wave_or_u64(o), 8);
#pragma unroll
    for (int j = 0; j < PER; j++) dst[lane + 64 * j] = (signed char)digit_of(x[j], s8, 8);
    return s16 - 16 + (a.F >> 16) - 16 + s8;
}

// one wave a (row, query head): q's digits
template <int PER>
__global__ __launch_bounds__(NTHREADS) void k_narrow_q(NarrowAtt a) {
    const int lane = threadIdx.x & 63, stream = blockIdx.z, q_heads = a.s.heads * a.group;
    const int i = blockIdx.x * (NTHREADS / 64) + (threadIdx.x >> 6);
    if (i >= a.rows * q_heads) return;
    const int t = i / q_heads, hq = i % q_heads, h = hq / a.group, rho = t * a.group + hq % a.group;
    const i64 slot = ((i64)stream * a.s.heads + h) * a.R + rho;
    const int p = narrow_pos(a, stream, t);
    i64 x[PER];
    narrow_q_load<PER>(a, a.q + stream * a.q_stream + t * a.q_row + (i64)hq * a.s.dim, p >= 0, lane, x);
    const int eq = narrow_q_row<PER>(a, x, lane, a.q8 + slot * a.s.wide);
    if (lane == 0) { a.pos[slot] = p; a.eq[slot] = eq; }
}

// 4-bit digits of a dword as bytes of 16 times the digit (the low halves, the high halves)
SMD int nib_lo(int x) { return (int)((unsigned)x << 4 & 0xF0F0F0F0u); }
SMD int nib_hi(int x) { return (int)((unsigned)x & 0xF0F0F0F0u); }
template <int CTRL> SMD int dpp_rot(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false); }
// a row's total over the lanes that hold it (all 16 columns; with GR rows a tile also the lane groups 16 GR / 4 apart),
// in every one of them
template <int GR, class T, class F>
SMD T row_total(T v, F op) {
    auto rot = [&](auto c) { v = op(v, __builtin_bit_cast(T, dpp_rot<decltype(c)::value>(__builtin_bit_cast(int, v)))); };
    rot(std::integral_constant<int, 0x128>());
    rot(std::integral_constant<int, 0x124>());
    rot(std::integral_constant<int, 0x122>());
    rot(std::integral_constant<int, 0x121>());
    if (GR <= 4) v = op(v, __shfl_xor(v, 16, 64));
    if (GR <= 8) v = op(v, __shfl_xor(v, 32, 64));
    return v;
}
struct IMax { SMD int operator()(int x, int y) const { return max(x, y); } };
struct IAdd { SMD int operator()(int x, int y) const { return x + y; } };

// the key digits of 16 positions from 16 `sub`, as they stand, and as DK operands (64 dimensions each)
template <int BITS, int DK> struct KeyRaw {
    static constexpr int U = BITS == 8 ? DK : DK / 2;
    v4i x[U > 0 ? U : 1];
    int2 y;
    SMD void load(const char* keys, int sub, int n, int g) {
        const int p = 16 * sub + n;
        if constexpr (U > 0) {
#pragma unroll
            for (int u = 0; u < U; u++) x[u] = *reinterpret_cast<const v4i*>(keys + (4 * u + g) * 1024 + p * 16);
        } else y = *reinterpret_cast<const int2*>(keys + (g >> 1) * 1024 + p * 16 + 8 * (g & 1));
    }
    SMD void operands(v4i o[DK]) const {
        if constexpr (BITS == 8) {
#pragma unroll
            for (int u = 0; u < DK; u++) o[u] = x[u];
        } else if constexpr (U == 0) {
            o[0] = v4i{nib_lo(y.x), nib_lo(y.y), nib_hi(y.x), nib_hi(y.y)};
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) {
                o[2 * u] = v4i{nib_lo(x[u][0]), nib_lo(x[u][1]), nib_lo(x[u][2]), nib_lo(x[u][3])};
                o[2 * u + 1] = v4i{nib_hi(x[u][0]), nib_hi(x[u][1]), nib_hi(x[u][2]), nib_hi(x[u][3])};
            }
        }
    }
};
// q's digits in the same order (row: the row's digits)
template <int BITS, int DK>
SMD void q_operands(const signed char* row, int g, v4i out[DK]) {
#pragma unroll
    for (int u = 0; u < DK; u++) {
        if constexpr (BITS == 4 && DK == 1) {
            const int2 x = *reinterpret_cast<const int2*>(row + 32 * (g >> 1) + 8 * (g & 1)),
                       y = *reinterpret_cast<const int2*>(row + 32 * (g >> 1) + 8 * (g & 1) + 16);
            out[u] = v4i{x.x, x.y, y.x, y.y};
        } else {
            out[u] = *reinterpret_cast<const v4i*>(row + (BITS == 8 ? 64 * u + 16 * g : 32 * (4 * (u / 2) + g) + 16 * (u % 2)));
        }
    }
}
// the value operands of one unit of a tile: 16 dimensions (8 bits) or twice 16 (4 bits)
template <int BITS>
SMD void value_operands(v4i x, v4i out[8 / BITS]) {
    if constexpr (BITS == 8) out[0] = x;
    else {
        out[0] = v4i{nib_lo(x[0]), nib_lo(x[1]), nib_hi(x[0]), nib_hi(x[1])};
        out[1] = v4i{nib_lo(x[2]), nib_lo(x[3]), nib_hi(x[2]), nib_hi(x[3])};
    }
}
// A score: dot 2^e rounded half up, held to 32 bits (v_cvt_rpi_i32_f32: floor(x + 1/2), saturating; dot has at most 23
// bits, so dot 2^e is exact in float).  Compared with that function in whole numbers for every dot and every e from -60 to
// 100: equal.
// (The compiler's wait states around the matrix units do not know what an asm block writes, so these write the register
// they read: whatever the matrix units still read or write there was waited for by the instruction before.)
SMD int narrow_round(float x) {
    int s = __builtin_bit_cast(int, x);
    asm("v_cvt_rpi_i32_f32 %0, %0" : "+v"(s));
    return s;
}
SMD int narrow_score(int dot, int e) { return narrow_round(ldexpf((float)dot, e)); }
// the exponent that a key's level is added to (past 40 every dot but 0 is clamped all the same)
template <int BITS> SMD int narrow_exp(int eq) { return min(eq - 6 - (BITS == 4 ? 4 : 0), 40); }      // (4-bit operands are 16 times the digit)
// Scores are clamped to +-2^30 where they are compared: m is clamped, and a score's distance to it is held to 0 .. far with
// far = min(alen, m + 2^30): below 0 the score was clamped to m's 2^30, past m + 2^30 to -2^30; from alen on the arrival is 0
#define NARROW_NONE INT_MIN         // the score of a position that a row does not see
SMD int narrow_clamp(int m) { return min(max(m, -(1 << 30)), 1 << 30); }
SMD int narrow_far(int m, int alen) { return (int)min((unsigned)alen, (unsigned)max(m, -(1 << 30)) + (1u << 30)); }      // (2^31 at m 2^30)
SMD int narrow_distance(int m, int s, int far) {
    int d = __builtin_elementwise_sub_sat(m, s);
    asm("v_med3_i32 %0, %0, 0, %1" : "+v"(d) : "v"(far));
    return d;
}
// A weight w in 0 .. 2^22 (u shifted by the levels' distance) as three signed bytes b0 + 256 b1 + 65536 b2: w + 0x808080
// with each byte's top bit flipped; the flip is left to the packed bytes.  u2 = 2 u, so that the shift's half is the 1 below
SMD unsigned narrow_weight(int u2, int shift) { return (((unsigned)u2 >> shift) + 0x1010101u) >> 1; }
// rsh(n0 + 256 n1 + 65536 n2, 8) of the byte planes' sums, the value digits of 4 bits 16 times their value
template <int BITS> SMD int narrow_sum(int n0, int n1, int n2) {
    const int q = n1 + (n2 << 8);
    return BITS == 8 ? q + ((n0 + 128) >> 8) : (q + ((n0 + 2048) >> 8)) >> 4;
}

// The arrivals as products of two short tables in LDS: ARR[d] = rint(e^(-(d / 128) / 8) 2^24 e^(-(d % 128) / 1024)), which the
// tables' creation has compared with every entry.  2^52 + 2^51 + 2 added in the same step leaves ARR[d] + 2 in the low word,
// and 2 rsh(ARR[d], 2) is that without its last two bits, halved.  (Gathered from the 71 KB table in memory, the weights
// took 33 us of the 106 that 64 streams of up to 8,192 positions spent in this kernel.)
#define NARROW_H 140
#define SWEEP_ARR 17790            // entries of the arrival that the kernels hold (base2_convert.py:50-53 gives 17,745)
struct NarrowFactors {
    double h[NARROW_H], l[128];
    SMD void load(const NarrowAtt& a, int tid, int threads) {
        const int nh = a.tb.alen / 128 + 1;
        for (int i = tid; i < nh + 128; i += threads) (i < nh ? h[i] : l[i - nh]) = a.WF[i];
    }
    SMD int weight(int d) const {
        const double x = __builtin_fma(h[d >> 7], l[d & 127], 6755399441055746.0);
        return (int)((unsigned)__builtin_bit_cast(u64, x) >> 1 & ~1u);
    }
};

// A chunk's N_j f_j rounded by s >= 24 places, added in float64: |N_j| is at most 2^29 and f_j at most 2^24, so the product, its
// half and the sum of up to 2^16 chunks are exact (and a quarter of the steps of 64-bit whole numbers)
SMD double narrow_factor(int f, int s) { return ldexp((double)f, -s); }
SMD double narrow_joined(double N, int Nj, double f) { return N + floor(__builtin_fma((double)Nj, f, 0.5)); }

// Few rows: a wave a chunk, a tile of GR rows (RU of every four wanted).  Scores: A = q, B = keys, so a lane is a position.
// With fewer than 16 rows the rows of position tile t' stand in operand rows GR t' .., zeros elsewhere, and 16 / GR position
// tiles add into one accumulator: every lane then holds a score that is wanted.  Weights: byte planes through the wave's
// LDS, their planes stacked as rows of one operand (3 GR rows in NM operands).  All of a chunk's keys are asked for first, then
// its values (in the registers that AHEAD tiles take).  Bound by the cache's read: 64 streams of up to 8,192 positions, 4 rows
// a key head, 4 bits, in 73 us, 4.7 TB/s; 131,072 positions of 8 bits in 63 us, 4.3 TB/s.
template <int BITS, int DK, int GR, int RU> struct NarrowChunk {
    static constexpr int NA = GR / 4, PT = 16 / GR, NM = (3 * GR + 15) / 16, DT = 4 * DK, VU = 8 / BITS, WBUF = NM * 1024;
    static constexpr int TILE_DW = DK * BITS * 2;                   // registers of a tile's keys (of its values)
    static constexpr int AHEAD = TILE_DW <= 16 ? 4 : TILE_DW <= 32 ? 2 : 1;
    v4i q[DK];
    int er[4], pos[4];
    int m[4], E[4], A[4];
    v4i C[NM][DT];

    // base: the head's tiles; c0: the chunk's first position; last: the last tile that holds a position seen; whole: every
    // row sees all 256
    template <bool WHOLE>
    SMD void run(const NarrowAtt& a, const char* base, int c0, int last, int lane, unsigned char* wb, const NarrowFactors& wf) {
        const int n = lane & 15, g = lane >> 4, t0 = c0 / 64;
        const i64 half = narrow_half(a.s), tile_bytes = narrow_tile(a.s);
        auto tile = [&](int t) { return base + (i64)min(t0 + t, last) * tile_bytes; };
        KeyRaw<BITS, DK> k[4][4];
        v4i v[4][DT / VU];
        int lev[4];
        auto load_k = [&](int t) {
#pragma unroll
            for (int sub = 0; sub < 4; sub++) k[t][sub].load(tile(t), sub, n, g);
        };
        auto load_v = [&](int t) {
#pragma unroll
            for (int c = 0; c < DT / VU; c++) v[t][c] = *reinterpret_cast<const v4i*>(tile(t) + half + c * 1024 + lane * 16);
        };
        // a tile's 128 levels are one line: one load of it
#pragma unroll
        for (int t = 0; t < 4; t++) lev[t] = reinterpret_cast<const int*>(tile(t) + 2 * half)[lane & 31];
        int vl[4][NA];
        auto level = [&](int t, int at) { return (int)((unsigned)__shfl(lev[t], at >> 2, 64) >> 8 * (at & 3) & 255u); };
#pragma unroll
        for (int t = 0; t < AHEAD; t++) load_k(t);
        int sc[4][NA][RU];
#pragma unroll
        for (int r = 0; r < RU; r++) { m[r] = NARROW_NONE; E[r] = 0; A[r] = 0; }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (t + AHEAD < 4) load_k(t + AHEAD);
            else load_v(t + AHEAD - 4);
            v4i acc[NA] = {};
#pragma unroll
            for (int sub = 0; sub < 4; sub++) {
                v4i o[DK];
                k[t][sub].operands(o);
#pragma unroll
                for (int u = 0; u < DK; u++) acc[sub / PT] = mfma8(n / GR == sub % PT ? q[u] : v4i{}, o[u], acc[sub / PT]);
            }
#pragma unroll
            for (int x = 0; x < NA; x++) {
                const int at = 16 * (x * PT + 4 * g / GR) + n, i = c0 + 64 * t + at, kl = level(t, at);
                vl[t][x] = level(t, 64 + at);
#pragma unroll
                for (int r = 0; r < RU; r++) {
                    sc[t][x][r] = narrow_score(acc[x][r], er[r] + kl);
                    m[r] = WHOLE || i <= pos[r] ? max(m[r], sc[t][x][r]) : m[r];
                    if (!WHOLE || r == 0) E[r] = max(E[r], WHOLE || i <= pos[r] ? vl[t][x] : 0);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < RU; r++) {
            m[r] = row_total<GR>(m[r], IMax());
            // (every row sees the same levels where each sees all: the total over all lanes)
            if (WHOLE) E[r] = r == 0 ? row_total<4>(E[0], IMax()) : E[0];
            else E[r] = row_total<GR>(E[r], IMax());
        }
        int far[RU];
#pragma unroll
        for (int r = 0; r < RU; r++) {
            m[r] = WHOLE || c0 <= pos[r] ? narrow_clamp(m[r]) : NARROW_NONE;
            far[r] = narrow_far(m[r], a.tb.alen);
        }
#pragma unroll
        for (int k2 = 0; k2 < NM; k2++)
#pragma unroll
            for (int c = 0; c < DT; c++) C[k2][c] = v4i{};
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (t >= 1 && t + AHEAD - 1 < 4 && AHEAD < 4) load_v(t + AHEAD - 1);
#pragma unroll
            for (int x = 0; x < NA; x++) {
                const int T = x * PT + 4 * g / GR, o = 16 * (n >> 2) + 4 * T + (n & 3);
#pragma unroll
                for (int r = 0; r < RU; r++) {
                    int d = narrow_distance(m[r], sc[t][x][r], far[r]), sh = min(E[r] - vl[t][x], 31);
                    if (!WHOLE) {
                        if (c0 + 64 * t + 16 * T + n > pos[r]) d = a.tb.alen;
                        sh = max(sh, 0);
                    }
                    const int u2 = wf.weight(d);
                    A[r] += u2;
                    const unsigned b = narrow_weight(u2, sh) ^ 0x808080u;
                    const int row0 = (4 * g + r) % GR;
                    wb[row0 * 64 + o] = (unsigned char)b;
                    wb[(GR + row0) * 64 + o] = (unsigned char)(b >> 8);
                    wb[(2 * GR + row0) * 64 + o] = (unsigned char)(b >> 16);
                }
            }
            v4i w[NM];
#pragma unroll
            for (int k2 = 0; k2 < NM; k2++) w[k2] = *reinterpret_cast<const v4i*>(wb + (16 * k2 + n) * 64 + 16 * g);
#pragma unroll
            for (int c = 0; c < DT / VU; c++) {
                v4i o[VU];
                value_operands<BITS>(v[t][c], o);
#pragma unroll
                for (int y = 0; y < VU; y++)
#pragma unroll
                    for (int k2 = 0; k2 < NM; k2++) C[k2][c * VU + y] = mfma8(w[k2], o[y], C[k2][c * VU + y]);
            }
        }
#pragma unroll
        for (int r = 0; r < RU; r++) A[r] = (int)((unsigned)row_total<GR>(A[r], IAdd()) >> 1);     // (2^31 at most)
    }
    // N_j of dimension tile c and the lane's row r (lane groups g < GR / 4 hold the rows)
    SMD int sum(int c, int r) const {
        const int n0 = C[0][c][r];
        if constexpr (GR == 16) return narrow_sum<BITS>(n0, C[1][c][r], C[2][c][r]);
        else if constexpr (GR == 8) return narrow_sum<BITS>(n0, __shfl_xor(n0, 32, 64), C[1][c][r]);
        else return narrow_sum<BITS>(n0, __shfl_xor(n0, 16, 64), __shfl_xor(n0, 32, 64));
    }
};

// What the blocks of few rows begin with: the positions of the tile's first and last row (a row that is not there takes no
// part), and the rows' digits, levels and positions in LDS
template <int DK, int GR> struct NarrowFew {
    NarrowFactors wf;
    signed char qd[GR][64 * DK];
    int qe[GR], qp[GR];
};
SMD bool narrow_reach(const NarrowAtt& a, int stream, int first, int end, int& plo, int& phi) {
    const int ta = first / a.group, tz = min((end - 1) / a.group, (a.count ? a.count[stream] : a.rows) - 1);
    const i64 s0 = a.start[stream];
    plo = (int)min(s0 + ta, (i64)a.span);
    phi = (int)min(s0 + tz, (i64)a.span - 1);
    return tz >= ta && phi >= 0;
}
template <int NW, int DK, int GR>
SMD void narrow_few(const NarrowAtt& a, int stream, int h, int rt, int lane, int wave, NarrowFew<DK, GR>& f) {
    constexpr int PER = (GR + NW - 1) / NW;                          // a wave's rows: loaded together
    const int rows = min(GR, a.R - rt * GR);
    f.wf.load(a, wave * 64 + lane, 64 * NW);
    i64 x[PER][DK];
    int p[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = wave + i * NW, rho = rt * GR + r, t = rho / a.group;
        p[i] = r < rows ? narrow_pos(a, stream, t) : -1;
        narrow_q_load<DK>(a, a.q + stream * a.q_stream + t * a.q_row + ((i64)h * a.group + rho % a.group) * a.s.dim, p[i] >= 0, lane, x[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = wave + i * NW;
        if (r >= rows) break;
        const int e = narrow_q_row<DK>(a, x[i], lane, f.qd[r]);
        if (lane == 0) { f.qe[r] = e; f.qp[r] = p[i]; }
    }
    __syncthreads();
}
template <int BITS, int DK, int GR, int RU>
SMD void narrow_ready(NarrowChunk<BITS, DK, GR, RU>& c, const NarrowFew<DK, GR>& f, int rows, int lane) {
    const int n = lane & 15, g = lane >> 4;
    q_operands<BITS, DK>(f.qd[min(n % GR, rows - 1)], g, c.q);
#pragma unroll
    for (int r = 0; r < RU; r++) {
        const int row = min((4 * g + r) % GR, rows - 1);
        c.er[r] = narrow_exp<BITS>(f.qe[row]);
        c.pos[r] = f.qp[row];
    }
}

// a block: NTHREADS / 64 chunks of one row tile, their partial sums to memory (k_narrow_join)
template <int BITS, int DK, int GR, int RU>
__global__ __launch_bounds__(NTHREADS, DK <= 2 ? 2 : 1) void k_narrow_split(NarrowAtt a, int jblocks) {
    using Chunk = NarrowChunk<BITS, DK, GR, RU>;
    __shared__ __attribute__((aligned(16))) unsigned char wbuf[NTHREADS / 64][Chunk::WBUF];
    __shared__ __attribute__((aligned(16))) NarrowFew<DK, GR> few;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int rt = blockIdx.x / jblocks, h = blockIdx.y, stream = blockIdx.z, rows = a.R - rt * GR;
    // blocks go to the eight dies in turn, and a stream's late chunks may be empty: the chunks rotate with head and stream
    const int jb = (int)((blockIdx.x + blockIdx.y + blockIdx.z) % jblocks), j = jb * (NTHREADS / 64) + wave, c0 = j * NCHUNK;
    const i64 head = (i64)stream * a.s.heads + h;
    int plo, phi;
    if (!narrow_reach(a, stream, rt * GR, min(rt * GR + GR, a.R), plo, phi) || phi < jb * (NTHREADS / 64) * NCHUNK) return;
    narrow_few<NTHREADS / 64, DK, GR>(a, stream, h, rt, lane, wave, few);
    if (j >= a.J || c0 > phi) return;
    Chunk c;
    narrow_ready(c, few, rows, lane);
    const char* base = a.buf + head * a.s.tiles * narrow_tile(a.s);
    if (c0 + NCHUNK - 1 <= plo) c.template run<true>(a, base, c0, phi / 64, lane, wbuf[wave], few.wf);
    else c.template run<false>(a, base, c0, phi / 64, lane, wbuf[wave], few.wf);
    const i64 slot0 = (head * a.J + j) * a.R + rt * GR;
    if (n == 0 && 4 * g < GR)
#pragma unroll
        for (int r = 0; r < RU; r++)
            if (4 * g + r < rows) { a.pm[slot0 + 4 * g + r] = c.m[r]; a.pA[slot0 + 4 * g + r] = c.A[r]; a.pE[slot0 + 4 * g + r] = c.E[r]; }
#pragma unroll
    for (int d = 0; d < Chunk::DT; d++)
#pragma unroll
        for (int r = 0; r < RU; r++) {
            const int N = c.sum(d, r);
            if (4 * g < GR && 4 * g + r < rows) a.pN[(slot0 + 4 * g + r) * a.s.wide + 16 * d + n] = N;
        }
}

// The same where a block takes all the chunks of its row tile (J <= NW): their partial sums stay in LDS and are joined there
template <int BITS, int DK, int GR, int RU, int NW>
__global__ __launch_bounds__(64 * NW, DK <= 2 ? 2 : 1) void k_narrow_near(NarrowAtt a) {
    using Chunk = NarrowChunk<BITS, DK, GR, RU>;
    constexpr int WIDE = 64 * DK;
    __shared__ __attribute__((aligned(16))) unsigned char wbuf[NW][Chunk::WBUF];
    __shared__ __attribute__((aligned(16))) NarrowFew<DK, GR> few;
    __shared__ int pN[NW][GR][WIDE], pm[NW][GR], pA[NW][GR], pE[NW][GR];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int rt = blockIdx.x, h = blockIdx.y, stream = blockIdx.z, rows = a.R - rt * GR;
    const i64 head = (i64)stream * a.s.heads + h;
    int plo, phi;
    if (!narrow_reach(a, stream, rt * GR, min(rt * GR + GR, a.R), plo, phi)) return;
    narrow_few<NW, DK, GR>(a, stream, h, rt, lane, wave, few);
    static_assert((SWEEP_ARR + 1) / 128 + 1 <= NARROW_H, "the arrival's factors fit");
    const int c0 = wave * NCHUNK;
    if (c0 <= phi) {
        Chunk c;
        narrow_ready(c, few, rows, lane);
        const char* base = a.buf + head * a.s.tiles * narrow_tile(a.s);
        if (c0 + NCHUNK - 1 <= plo) c.template run<true>(a, base, c0, phi / 64, lane, wbuf[wave], few.wf);
        else c.template run<false>(a, base, c0, phi / 64, lane, wbuf[wave], few.wf);
        if (n == 0 && 4 * g < GR)
#pragma unroll
            for (int r = 0; r < RU; r++) { pm[wave][4 * g + r] = c.m[r]; pA[wave][4 * g + r] = c.A[r]; pE[wave][4 * g + r] = c.E[r]; }
#pragma unroll
        for (int d = 0; d < Chunk::DT; d++)
#pragma unroll
            for (int r = 0; r < RU; r++) {
                const int N = c.sum(d, r);
                if (4 * g < GR) pN[wave][4 * g + r][16 * d + n] = N;
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(GR, rows) * WIDE; i += 64 * NW) {
        const int r = i / WIDE, d = i % WIDE, p = few.qp[r], J = p / NCHUNK + 1;
        if (p < 0 || d >= a.s.dim) continue;
        int M = pm[0][r], E = pE[0][r];
        for (int j = 1; j < J; j++) { M = max(M, pm[j][r]); E = max(E, pE[j][r]); }
        i64 A = 0, N = 0;
        for (int j = 0; j < J; j++) {
            const unsigned df = (unsigned)M - (unsigned)pm[j][r];
            const i64 f = df < (unsigned)a.tb.alen ? a.tb.ARR[df] : 0;
            A += rsh_round(pA[j][r] * f, 24);
            N += rsh_round(pN[j][r][d] * f, min(24 + E - pE[j][r], 63));
        }
        const int rho = rt * GR + r, t = rho / a.group, hq = h * a.group + rho % a.group;
        a.out[stream * a.o_stream + t * a.o_row + (i64)hq * a.s.dim + d] = power(N, ((i64)E + 8) * 65536 - log2fix(A, a.tb), a.tb);
    }
}

// Many rows: a block 16 rows and all the positions that they see, its four waves every fourth chunk.  Scores: A = keys,
// B = q, so that a lane holds one row's scores of 16 positions a tile, and exactly the ones, in the order, that its bytes of a
// weight operand are (the values' layout): nothing moves between lanes.  A first pass over the keys finds each chunk's m_j
// and E_j (kept in memory) and the row's M and E; the second adds each chunk's N_j f_j in registers, and the waves' sums are
// added at the end.  Bound by the vector arithmetic of a score, 23 steps in the second pass and 5 in the first (the matrix
// products take a fifth of that), at three waves a SIMD: 1,024 rows of two prompts over 4,096 positions, 12 heads of 64, in
// 105 us.  (The weights from the 71 KB table in LDS: two waves, 138 us; sums in registers: 111 us.)
#define SWEEP_WAVES 4
template <int BITS, int DK>
__global__ __launch_bounds__(64 * SWEEP_WAVES, 4 - (DK == 4 ? 3 : DK)) void k_narrow_sweep(NarrowAtt a) {
    constexpr int DT = 4 * DK, VU = 8 / BITS, NW = SWEEP_WAVES;
    __shared__ double sums[NW][DT * 4][64];                             // the waves' N, a lane's own (in registers they spill)
    __shared__ NarrowFactors wf;
    __shared__ int wm[NW][16], we[NW][16];
    __shared__ i64 wA[NW][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const int h = blockIdx.y, stream = blockIdx.z;
    const i64 head = (i64)stream * a.s.heads + h;
    // the last rows, which see most, first
    const int rt = (int)(gridDim.x - 1 - blockIdx.x);
    const int rho = min(rt * 16 + n, a.R - 1), pos = a.pos[head * a.R + rho], er = narrow_exp<BITS>(a.eq[head * a.R + rho]);
    int phi = pos, plo = pos;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) { phi = max(phi, __shfl_xor(phi, o, 64)); plo = min(plo, __shfl_xor(plo, o, 64)); }
    phi = __builtin_amdgcn_readfirstlane(phi);
    plo = __builtin_amdgcn_readfirstlane(plo);
    if (phi < 0) return;                                             // (the same in every wave)
    wf.load(a, threadIdx.x, 64 * NW);
    v4i q[DK];
    q_operands<BITS, DK>(a.q8 + (head * a.R + rho) * a.s.wide, g, q);
    const i64 half = narrow_half(a.s), tile_bytes = narrow_tile(a.s);
    const char* base = a.buf + head * a.s.tiles * tile_bytes;
    const int last = phi / 64;
    int* pm = a.pm + head * a.J * a.R + rho;
    int* pE = a.pE + head * a.J * a.R + rho;
    auto max_g = [](int v) {
        v = max(v, __shfl_xor(v, 16, 64));
        return max(v, __shfl_xor(v, 32, 64));
    };
    // a tile's keys and levels, and its values; each register takes the next tile's as soon as it has been used
    KeyRaw<BITS, DK> k[4];
    int lev;                                                         // (one load of the line: see NarrowChunk)
    v4i v[DT / VU];
    auto load_sub = [&](int T, int sub) {
        const char* tp = base + (i64)T * tile_bytes;
        k[sub].load(tp, sub, n, g);
        if (sub == 3) lev = reinterpret_cast<const int*>(tp + 2 * half)[lane & 31];
    };
    auto key_levels = [&](int sub) { return __shfl(lev, 4 * sub + g, 64); };
    auto value_levels = [&](int sub) { return __shfl(lev, 16 + 4 * sub + g, 64); };
    auto load_v = [&](int T, int c) { v[c] = *reinterpret_cast<const v4i*>(base + (i64)T * tile_bytes + half + c * 1024 + lane * 16); };
    auto after = [](int T) { return (T & 3) == 3 ? T + 4 * NW - 3 : T + 1; };
    // dots of the 16 positions of a sub-tile with the lane's row, positions 4 g .. 4 g + 3 of it
    auto dots = [&](int sub) {
        v4i o[DK], acc = {};
        k[sub].operands(o);
#pragma unroll
        for (int u = 0; u < DK; u++) acc = mfma8(o[u], q[u], acc);
        return acc;
    };
    auto byte = [](int x, int r) { return (int)((unsigned)x >> 8 * r & 255u); };
    int M = NARROW_NONE, E = 0;
    {
        float m = -INFINITY;
        int e = 0;
        int T = 4 * wave;
#pragma unroll
        for (int sub = 0; sub < 4; sub++) load_sub(min(T, last), sub);
        while (T <= last) {
            const int Tn = min(after(T), last);
            // (rounding and clamping keep the order: done once, on the largest)
            auto look = [&](auto whole) {
#pragma unroll
                for (int sub = 0; sub < 4; sub++) {
                    const v4i acc = dots(sub);
                    const int l = key_levels(sub), lv = value_levels(sub);
                    load_sub(Tn, sub);
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (decltype(whole)::value || 64 * T + 16 * sub + 4 * g + r <= pos) {
                            m = fmaxf(m, ldexpf((float)acc[r], er + byte(l, r)));
                            e = max(e, byte(lv, r));
                        }
                }
            };
            if (64 * T + 63 <= plo) look(std::true_type());
            else look(std::false_type());
            if ((T & 3) == 3 || T == last) {
                const int j = T >> 2;
                int mi = narrow_round(m);
                mi = max_g(j * NCHUNK + 4 * g <= pos ? narrow_clamp(mi) : NARROW_NONE);
                e = max_g(e);
                if (g == 0) { pm[(i64)j * a.R] = mi; pE[(i64)j * a.R] = e; }
                M = max(M, mi);
                E = max(E, e);
                m = -INFINITY;
                e = 0;
            }
            T = after(T);
        }
    }
    if (g == 0) { wm[wave][n] = M; we[wave][n] = E; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) { M = max(M, wm[w][n]); E = max(E, we[w][n]); }
    i64 A = 0;
#pragma unroll
    for (int i = 0; i < DT * 4; i++) sums[wave][i][lane] = 0;
    int have = -1;                                                   // the tile that is loaded
    for (int j = wave; 4 * j <= last; j += NW) {
        // (this wave's own stores, read by the lanes that made them)
        const int m = __shfl(pm[(i64)j * a.R], n, 64), e = __shfl(pE[(i64)j * a.R], n, 64);
        const unsigned df = (unsigned)M - (unsigned)m;
        const int f = m != NARROW_NONE && df < (unsigned)a.tb.alen ? a.tb.ARR[df] : 0;
        if (!__any(f)) continue;                                     // its sums would be multiplied by 0
        const int far = narrow_far(m, a.tb.alen), tz = min(4 * j + 3, last);
        v4i C[3][DT] = {};
        unsigned Aj = 0;
        if (have != 4 * j) {
#pragma unroll
            for (int sub = 0; sub < 4; sub++) load_sub(4 * j, sub);
#pragma unroll
            for (int c = 0; c < DT / VU; c++) load_v(4 * j, c);
        }
        for (int T = 4 * j; T <= tz; T++) {
            v4i P[3];
            have = T < tz ? T + 1 : min(4 * (j + NW), last);
            auto weigh = [&](auto whole) {
#pragma unroll
                for (int sub = 0; sub < 4; sub++) {
                    const v4i acc = dots(sub);
                    const int l = key_levels(sub), lv = value_levels(sub);
                    load_sub(have, sub);
                    unsigned x[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        int d = narrow_distance(m, narrow_score(acc[r], er + byte(l, r)), far), sh = min(e - byte(lv, r), 31);
                        if (!decltype(whole)::value) {
                            if (64 * T + 16 * sub + 4 * g + r > pos) d = a.tb.alen;
                            sh = max(sh, 0);
                        }
                        const int u2 = wf.weight(d);
                        Aj += u2;
                        x[r] = narrow_weight(u2, sh);
                    }
                    const unsigned p01 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), p23 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
                    P[0][sub] = (int)(__builtin_amdgcn_perm(p23, p01, 0x05040100u) ^ 0x80808080u);
                    P[1][sub] = (int)(__builtin_amdgcn_perm(p23, p01, 0x07060302u) ^ 0x80808080u);
                    P[2][sub] = (int)((__builtin_amdgcn_perm(x[1], x[0], 0x0c0c0602u) | __builtin_amdgcn_perm(x[3], x[2], 0x06020c0cu)) ^ 0x80808080u);
                }
            };
            if (64 * T + 63 <= plo) weigh(std::true_type());
            else weigh(std::false_type());
#pragma unroll
            for (int c = 0; c < DT / VU; c++) {
                v4i o[VU];
                value_operands<BITS>(v[c], o);
                load_v(have, c);
#pragma unroll
                for (int y = 0; y < VU; y++)
#pragma unroll
                    for (int p = 0; p < 3; p++) C[p][c * VU + y] = mfma8(o[y], P[p], C[p][c * VU + y]);
            }
        }
        Aj += __shfl_xor(Aj, 16, 64);
        Aj += __shfl_xor(Aj, 32, 64);
        A += rsh_round((i64)(Aj >> 1) * f, 24);                      // (Aj 2^31 at most)
        const double fs = narrow_factor(f, 24 + E - e);
#pragma unroll
        for (int c = 0; c < DT; c++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                double& N = sums[wave][4 * c + r][lane];
                N = narrow_joined(N, narrow_sum<BITS>(C[0][c][r], C[1][c][r], C[2][c][r]), fs);
            }
    }
    // the waves' sums added: wave w finishes every fourth dimension tile
    if (g == 0) wA[wave][n] = A;
    __syncthreads();
    if (pos < 0 || rt * 16 + n >= a.R) return;
    A = 0;
    for (int w = 0; w < NW; w++) A += wA[w][n];
    const i64 F = ((i64)E + 8) * 65536 - log2fix(A, a.tb);
    const int tt = rho / a.group, hq = h * a.group + rho % a.group;
    i64* o = a.out + stream * a.o_stream + tt * a.o_row + (i64)hq * a.s.dim;
    for (int c = wave; c < DT; c += NW)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            double s = 0;
#pragma unroll
            for (int w = 0; w < NW; w++) s += sums[w][4 * c + r][lane];
            const int d = 16 * c + 4 * g + r;
            if (d < a.s.dim) o[d] = power((i64)s, F, a.tb);
        }
}

// A block a row's db dimensions: its chunks joined, a thread a dimension of a slice of the chunks (NTHREADS / db slices).  The
// first PRE sums of a thread are loaded with all else, before the row's M and E are known; the chunks' factors are formed
// once, in LDS, a batch of NTHREADS chunks at a time.  Bound by its chain of loads with few chunks (all of a row's dimensions
// in one block then: the factors are formed once), by their number with many (8 dimensions a block: 512 chunks of 32 rows 12.0 us, 15.0 with 16 a block, 25.3 with 32).
__global__ __launch_bounds__(NTHREADS, 8) void k_narrow_join(NarrowAtt a, int db) {
    constexpr int PRE = 8, NW = NTHREADS / 64;
    __shared__ int sm[NW], se[NW];
    __shared__ i64 sa[NW];
    __shared__ double sf[NTHREADS], sn[NTHREADS];
    const int wide = a.s.wide, blocks = wide / db;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rho = blockIdx.x / blocks, h = blockIdx.y, stream = blockIdx.z;
    const i64 head = (i64)stream * a.s.heads + h, slot0 = head * a.J * a.R + rho;
    const int p = narrow_pos(a, stream, rho / a.group);
    if (p < 0) return;
    const int J = p / NCHUNK + 1, d = (int)blockIdx.x % blocks * db + tid % db, slice = tid / db, slices = NTHREADS / db;
    const int* pn = a.pN + slot0 * wide + d;
    const i64 step = (i64)a.R * wide;
    int v[PRE];
    auto load = [&](int j0) {
#pragma unroll
        for (int i = 0; i < PRE; i++)
            if (j0 + i * slices < J) v[i] = pn[(j0 + i * slices) * step];
    };
    load(slice);
    int M = NARROW_NONE, E = 0;
    for (int j = tid; j < J; j += NTHREADS) {
        M = max(M, a.pm[slot0 + (i64)j * a.R]);
        E = max(E, a.pE[slot0 + (i64)j * a.R]);
    }
    for (int o = 1; o < 64; o <<= 1) { M = max(M, __shfl_xor(M, o, 64)); E = max(E, __shfl_xor(E, o, 64)); }
    if (lane == 0) { sm[wave] = M; se[wave] = E; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; i++) { M = max(M, sm[i]); E = max(E, se[i]); }
    i64 A = 0;
    double N = 0;
    for (int j0 = 0; j0 < J; j0 += NTHREADS) {
        const int n = min(NTHREADS, J - j0);
        if (j0) __syncthreads();
        if (tid < n) {
            const i64 s = slot0 + (i64)(j0 + tid) * a.R;
            const unsigned df = (unsigned)M - (unsigned)a.pm[s];
            const int f = df < (unsigned)a.tb.alen ? a.tb.ARR[df] : 0;
            A += rsh_round((i64)a.pA[s] * f, 24);
            sf[tid] = narrow_factor(f, 24 + E - a.pE[s]);
        }
        __syncthreads();
        for (int j = slice; j < n; j += PRE * slices) {
            if (j0 + j != slice) load(j0 + j);
#pragma unroll
            for (int i = 0; i < PRE; i++)
                if (j + i * slices < n) N = narrow_joined(N, v[i], sf[j + i * slices]);
        }
    }
    A = wave_reduce64(A, OpAdd());
    if (lane == 0) sa[wave] = A;
    sn[tid] = N;
    __syncthreads();
    if (tid >= db || d >= a.s.dim) return;
    A = sa[0] + sa[1] + sa[2] + sa[3];
    for (int i = 1; i < slices; i++) N += sn[i * db + tid];
    const int t = rho / a.group, hq = h * a.group + rho % a.group;
    a.out[stream * a.o_stream + t * a.o_row + (i64)hq * a.s.dim + d] = power((i64)N, ((i64)E + 8) * 65536 - log2fix(A, a.tb), a.tb);
}

// ---------------------------------------------------------------------------------------------------------
// entry points

// rows of int64 that begin at lines of 128 bytes
static bool whole_lines(const void* p, i64 stride) { return !((uintptr_t)p & 127) && stride % 16 == 0; }

// The device that holds a call's memory, made current for the call.  Memory that no device holds is refused here, before a
// kernel reads it.
struct OnDevice {
    int was = -1, dev = -1;
    bool ok = false;
    explicit OnDevice(const void* p) {
        hipPointerAttribute_t at{};
        if (hipPointerGetAttributes(&at, p) != hipSuccess) { (void)hipGetLastError(); return; }
        if (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged) return;
        if (hipGetDevice(&was) != hipSuccess) return;
        dev = at.device;
        ok = dev == was || hipSetDevice(dev) == hipSuccess;
    }
    ~OnDevice() { if (ok && dev != was) (void)hipSetDevice(was); }
    OnDevice(const OnDevice&) = delete;
};

struct sm_plate8 {
    signed char* W = nullptr; int* e = nullptr; i64* b = nullptr;
    int nin = 0, nout = 0, K = 0;
    i64 bytes = 0;
};
static void plate8_free(sm_plate8* p) {
    hfree(p->W); hfree(p->e); hfree(p->b);
    delete p;
}

extern "C" int sm_plate8_create(const int8_t* w, const int32_t* e, const int64_t* b, int32_t nin, int32_t nout, sm_plate8** out) {
    if (!w || !e || !b || !out) return fail(SM_E_ARG, "sm_plate8_create: null argument");
    if (nin < 1 || nin > SM_PLATE8_NIN || nout < 1 || nout > (1 << 24)) return fail(SM_E_ARG, "sm_plate8_create: nin or nout out of range");
    for (int32_t i = 0; i < nout; i++)
        if (e[i] < -1024 || e[i] > 1024) return fail(SM_E_ARG, "sm_plate8_create: a column's power is out of range");
    sm_plate8* p = new (std::nothrow) sm_plate8();
    if (!p) return fail(SM_E_OOM, "sm_plate8_create: host memory");
    p->nin = nin; p->nout = nout; p->K = (nin + 63) / 64 * 64;
    p->bytes = (i64)((nout + 15) / 16) * 16 * p->K;
    signed char* raw = nullptr;
    int rc;
    auto make = [&]() -> int {
        if ((rc = dalloc(&p->W, (size_t)p->bytes)) || (rc = dalloc(&p->e, (size_t)nout)) || (rc = dalloc(&p->b, (size_t)nout)) ||
            (rc = dalloc(&raw, (size_t)nin * nout)))
            return rc;
        HIP_TRY(hipMemcpy(raw, w, (size_t)nin * nout, hipMemcpyHostToDevice));
        HIP_TRY(hipMemcpy(p->e, e, (size_t)nout * 4, hipMemcpyHostToDevice));
        HIP_TRY(hipMemcpy(p->b, b, (size_t)nout * 8, hipMemcpyHostToDevice));
        const i64 quads = p->bytes / 4;
        const unsigned blocks = (unsigned)std::min<i64>((quads + NTHREADS - 1) / NTHREADS, 1 << 16);
        launch(false, "plate8.lay", k_narrow_plate, dim3(blocks), dim3(NTHREADS), 0, nullptr, (const signed char*)raw, (int)nin, (int)nout, p->K, p->W, quads);
        HIP_TRY(hipGetLastError());
        HIP_TRY(hipStreamSynchronize(nullptr));
        return SM_OK;
    };
    rc = make();
    hfree(raw);
    if (rc) { plate8_free(p); return rc; }
    *out = p;
    return SM_OK;
}
extern "C" int sm_plate8_destroy(sm_plate8* p) {
    if (p) {
        OnDevice on(p->W);
        (void)hipDeviceSynchronize();
        plate8_free(p);
    }
    return SM_OK;
}
extern "C" int64_t sm_plate8_bytes(const sm_plate8* p) { return p ? p->bytes : 0; }

static i64 up256(i64 n) { return (n + 255) / 256 * 256; }
static i64 plate8_lights(const sm_plate8* p, int rows) { return up256((i64)((rows + 15) / 16) * 16 * p->K); }
extern "C" int64_t sm_plate8_work(const sm_plate8* p, int32_t rows) {
    if (!p || rows < 0) { fail(SM_E_ARG, "sm_plate8_work: arguments"); return SM_E_ARG; }
    return plate8_lights(p, rows) + up256((i64)rows * 4);
}

extern "C" int sm_plate8_product(const sm_plate8* p, const int64_t* X, int64_t x_stride, int32_t rows, int64_t* out,
                                 int64_t out_stride, void* work, int64_t work_bytes, void* stream) {
    if (!p) return fail(SM_E_ARG, "sm_plate8_product: null plate");
    if (rows < 0 || rows > SM_PLATE8_ROWS) return fail(SM_E_ARG, "sm_plate8_product: rows out of range");
    if (!rows) return SM_OK;
    if ((i64)rows * p->nout > ((i64)1 << 35)) return fail(SM_E_ARG, "sm_plate8_product: more than 2^35 results in one call");
    if (!X || !out || !work) return fail(SM_E_ARG, "sm_plate8_product: null argument");
    if (x_stride < p->nin || out_stride < p->nout) return fail(SM_E_ARG, "sm_plate8_product: a row stride is shorter than its row");
    if (((uintptr_t)X | (uintptr_t)out) & 7 || (uintptr_t)work & 15) return fail(SM_E_ARG, "sm_plate8_product: alignment (rows 8 bytes, work 16)");
    if (work_bytes < sm_plate8_work(p, rows)) return fail(SM_E_ARG, "sm_plate8_product: the workspace is smaller than sm_plate8_work");
    OnDevice on(p->W);
    if (!on.ok) return fail(SM_E_HIP, "sm_plate8_product: the plate's device");
    Narrow8Args a{};
    a.W = p->W; a.we = p->e; a.wb = p->b; a.nin = p->nin; a.K = p->K; a.N = p->nout;
    a.X = (const i64*)X; a.ldx = x_stride; a.rows = rows; a.out = (i64*)out; a.ldo = out_stride;
    a.lights = static_cast<signed char*>(work);
    a.level = reinterpret_cast<int*>(static_cast<char*>(work) + plate8_lights(p, rows));
    hipStream_t s = (hipStream_t)stream;
    // (every block forms the rows' digits: 8 rows 143 -> 36336, 2,271 blocks, 19.3 us so and 10.4 in two launches; one row
    // 2761 -> 41192, 2,575 blocks of three, 21 us)
    const i64 quads = (i64)rows * ((p->K + 1023) / 1024);
    if (quads <= FEW_QUADS && quads * ((a.N + 15) / 16) <= 8192) {
        launch(g_kt.stages, "plate8.one", k_narrow_one, dim3((unsigned)((a.N + 15) / 16)), dim3(NTHREADS), 0, s, a);
        HIP_TRY(hipGetLastError());
        return SM_OK;
    }
    launch(g_kt.stages, "plate8.lights", k_narrow_lights, dim3((unsigned)(rows < 128 ? rows : (rows + 127) / 128 * 128)), dim3(NTHREADS), 0, s, a);
    const int nt = (a.N + 15) / 16, rts = (rows + 15) / 16;
    if (rts == 1) launch(g_kt.stages, "plate8.rows", k_narrow_rows<1, 1, 4>, dim3(nt, 1), dim3(NTHREADS), 0, s, a);
    else if (rts == 2) launch(g_kt.stages, "plate8.rows", k_narrow_rows<2, 1, 4>, dim3(nt, 1), dim3(NTHREADS), 0, s, a);
    else {
        // Up to 64 rows a block a column tile, which then reads its weights once (64 rows 768 -> 50257 17.2 us, 21.1 in tiles of
        // 128 x 128).  More rows in such tiles from 128 of them on (512 rows 4096 -> 4096, 128 tiles, 33.7 us against 39.8;
        // 256 rows, 64 tiles, 31.2 against 23.7; 512 rows 1024 -> 11008, 344 tiles, 25.0 against 31.1).  Tiles of 256 x 256, one
        // a CU, where they take fewer rounds of the GPU than those of 128, two a CU and a fifth slower: 1024 rows
        // 1024 -> 11008, 172 of them, 36.8 us and 40.9; 2048 rows, 344, 81.8 and 69.5; 2048 rows 4096 -> 4096, 128, 76 and 58
        const bool past = (i64)rows * a.N * 8 >= NARROW_STREAM && whole_lines(out, out_stride);
        const i64 t128 = (i64)((rts + 7) / 8) * ((nt + 7) / 8), t256 = (i64)((rts + 15) / 16) * ((nt + 15) / 16);
        auto tiles = [&](auto kern, int rt, int ct, int threads) {
            const int tr = (rts + rt - 1) / rt, tc = (nt + ct - 1) / ct;
            launch(g_kt.stages, "plate8.tiles", kern, dim3((unsigned)(((i64)tr * tc + 7) / 8 * 8)), dim3(threads), 0, s, a, tr, tc);
        };
        if (rows <= 64 || t128 < 128) launch(g_kt.stages, "plate8.rows", k_narrow_rows<4, 1, 4>, dim3((unsigned)nt, (unsigned)((rts + 3) / 4)), dim3(NTHREADS), 0, s, a);
        else if (8 * ((t256 + 255) / 256) <= 5 * ((t128 + 511) / 512)) past ? tiles(k_narrow_tiles<2, 4, 8, 4, true>, 16, 16, 512) : tiles(k_narrow_tiles<2, 4, 8, 4, false>, 16, 16, 512);
        else past ? tiles(k_narrow_tiles<2, 2, 4, 4, true>, 8, 8, 256) : tiles(k_narrow_tiles<2, 2, 4, 4, false>, 8, 8, 256);
    }
    HIP_TRY(hipGetLastError());
    return SM_OK;
}

// ---- the cache
static int narrow_shape(const sm_narrow* c, NarrowShape& s, const char* who) {
    const std::string w(who);
    if (!c) return fail(SM_E_ARG, w + ": null shape");
    if (c->streams < 1 || c->streams > 65535 || c->heads < 1 || c->heads > 65535 || (i64)c->streams * c->heads > (1 << 20))
        return fail(SM_E_ARG, w + ": streams and heads are 1 .. 65535, their product at most 2^20");
    if (c->dim < 1 || c->dim > 256) return fail(SM_E_ARG, w + ": a head has 1 .. 256 dimensions");
    if (c->ctx < 1 || c->ctx > (1 << 24)) return fail(SM_E_ARG, w + ": ctx is 1 .. 2^24");
    if (c->bits != 4 && c->bits != 8) return fail(SM_E_ARG, w + ": digits of 4 or 8 bits");
    s.streams = c->streams; s.heads = c->heads; s.dim = c->dim; s.ctx = c->ctx; s.bits = c->bits;
    s.wide = c->dim <= 64 ? 64 : c->dim <= 128 ? 128 : 256;
    s.tiles = (c->ctx + 63) / 64;
    return SM_OK;
}
static i64 narrow_tile_bytes(const NarrowShape& s) { return (i64)s.wide * 16 * s.bits + 128; }
extern "C" int64_t sm_narrow_bytes(const sm_narrow* c) {
    NarrowShape s;
    const int rc = narrow_shape(c, s, "sm_narrow_bytes");
    return rc ? rc : (i64)s.streams * s.heads * s.tiles * narrow_tile_bytes(s);
}

static int narrow_rows(const sm_narrow* c, const void* buf, const void* k, const void* v, int64_t row_stride, int64_t stream_stride,
                       int32_t rows, const int32_t* start, NarrowShape& s, const char* who) {
    const std::string w(who);
    int rc = narrow_shape(c, s, who);
    if (rc) return rc;
    if (rows < 0 || rows > s.ctx) return fail(SM_E_ARG, w + ": rows are 0 .. ctx");
    if (!rows) return SM_OK;
    if (!buf || !k || !v || !start) return fail(SM_E_ARG, w + ": null argument");
    if (row_stride < (int64_t)s.heads * s.dim || stream_stride < 0) return fail(SM_E_ARG, w + ": strides");
    if ((uintptr_t)buf & 15 || ((uintptr_t)k | (uintptr_t)v) & 7 || (uintptr_t)start & 3) return fail(SM_E_ARG, w + ": alignment (cache 16 bytes, rows 8)");
    return SM_OK;
}

// whether rows of `width` values of several streams would lie over one another (results may not)
static bool rows_overlap(int streams, int rows, i64 width, i64 row, i64 stream) {
    return streams > 1 && stream < (rows - 1) * row + width && (stream < width || (rows > 1 && row < (streams - 1) * stream + width));
}

extern "C" int sm_narrow_write(const sm_narrow* c, void* buf, const int64_t* k, const int64_t* v, int64_t row_stride,
                               int64_t stream_stride, int32_t rows, const int32_t* start, const int32_t* count, void* stream) {
    NarrowRows a{};
    int rc = narrow_rows(c, buf, k, v, row_stride, stream_stride, rows, start, a.s, "sm_narrow_write");
    if (rc || !rows) return rc;
    OnDevice on(buf);
    if (!on.ok) return fail(SM_E_ARG, "sm_narrow_write: the cache is not in a device's memory");
    a.buf = static_cast<char*>(buf); a.k = (const i64*)k; a.v = (const i64*)v;
    a.row_stride = row_stride; a.stream_stride = stream_stride; a.rows = rows; a.start = start; a.count = count;
    const i64 blocks = (i64)((rows + 62) / 64 + 1) * a.s.heads;
    if (blocks > (1 << 22)) return fail(SM_E_ARG, "sm_narrow_write: too many rows for one call");
    const dim3 grid((unsigned)blocks, 1, (unsigned)a.s.streams);
    auto write = [&](auto nw) {
        constexpr int NW = decltype(nw)::value;
        auto go = [&](auto kern) { launch(g_kt.stages, "narrow.write", kern, grid, dim3(64 * NW), 0, (hipStream_t)stream, a); };
        if (a.s.bits == 4) a.s.wide == 64 ? go(k_narrow_write<4, 64, NW>) : a.s.wide == 128 ? go(k_narrow_write<4, 128, NW>) : go(k_narrow_write<4, 256, NW>);
        else a.s.wide == 64 ? go(k_narrow_write<8, 64, NW>) : a.s.wide == 128 ? go(k_narrow_write<8, 128, NW>) : go(k_narrow_write<8, 256, NW>);
    };
    // eight waves a block where a tile has rows for them (997 rows of 7 heads of 80, five streams: 14.3 us, 16.9 with four)
    if (rows <= 8) write(std::integral_constant<int, 4>());
    else write(std::integral_constant<int, 8>());
    HIP_TRY(hipGetLastError());
    return SM_OK;
}

extern "C" int sm_narrow_read(const sm_narrow* c, const void* buf, int64_t* k, int64_t* v, int64_t row_stride,
                              int64_t stream_stride, int32_t rows, const int32_t* start, const int32_t* count, void* stream) {
    NarrowRows a{};
    int rc = narrow_rows(c, buf, k, v, row_stride, stream_stride, rows, start, a.s, "sm_narrow_read");
    if (rc || !rows) return rc;
    if (rows_overlap(a.s.streams, rows, (i64)a.s.heads * a.s.dim, row_stride, stream_stride)) return fail(SM_E_ARG, "sm_narrow_read: the strides lay rows over one another");
    OnDevice on(buf);
    if (!on.ok) return fail(SM_E_ARG, "sm_narrow_read: the cache is not in a device's memory");
    a.buf = static_cast<char*>(const_cast<void*>(buf)); a.k2 = (i64*)k; a.v2 = (i64*)v;
    a.row_stride = row_stride; a.stream_stride = stream_stride; a.rows = rows; a.start = start; a.count = count;
    const i64 n = (i64)rows * a.s.heads * ((a.s.dim + 1) / 2);
    const dim3 grid((unsigned)std::min<i64>((n + NTHREADS - 1) / NTHREADS, 4096), 1, (unsigned)a.s.streams);
    auto go = [&](auto kern) { launch(g_kt.stages, "narrow.read", kern, grid, dim3(NTHREADS), 0, (hipStream_t)stream, a); };
    const bool nt = (i64)a.s.streams * rows * a.s.heads * a.s.dim * 16 >= NARROW_STREAM && whole_lines(k, row_stride) &&
                    whole_lines(v, row_stride) && stream_stride % 16 == 0;
    if (a.s.bits == 4) nt ? go(k_narrow_read<4, true>) : go(k_narrow_read<4, false>);
    else nt ? go(k_narrow_read<8, true>) : go(k_narrow_read<8, false>);
    HIP_TRY(hipGetLastError());
    return SM_OK;
}

// ---- the attention's workspace: the chunks' partial sums, and with many rows q's digits, the rows' levels and positions
struct NarrowWork { bool sweep; i64 q8, eq, pos, pm, pA, pE, pN, bytes; };
static NarrowWork narrow_work(const NarrowShape& s, int R, int J) {
    const i64 n = (i64)s.streams * s.heads * R;
    NarrowWork w{};
    // The sweep from 640 row tiles on (one a wave's quarter), below that chunks spread over the GPU: 16 streams of 8 heads at
    // 16,000 positions, 20 rows (256 tiles) 176 us swept and 100 split, 100 rows (896) 251 and 256; 4 streams of 32 heads over
    // 8 at 3,000, 40 rows (320) 47 and 52, 100 rows (800) 80 and 92.  And where the chunks' sums would pass 4 GB.
    // With heads past 128 dimensions, whose chunks leave a wave a SIMD, from 256 tiles on: 2 streams of 8 heads of 256 at 1,000,
    // 300 rows (304) 54 and 80; 200 rows of one at 6,000 (104) 106 and 72.
    w.sweep = R > 16 && ((i64)s.streams * s.heads * ((R + 15) / 16) >= (s.wide == 256 ? 256 : 640) || n * J * s.wide * 4 > ((i64)4 << 30));
    w.pm = 0;
    w.pE = up256(n * J * 4);
    w.pA = w.q8 = w.pE + up256(n * J * 4);
    w.pN = w.pA + up256(n * J * 4);
    w.eq = w.q8 + up256(n * s.wide);
    w.pos = w.eq + up256(n * 4);
    w.bytes = w.sweep ? w.pos + n * 4 : w.pN + n * J * s.wide * 4;
    return w;
}
static int narrow_att_args(const sm_narrow* c, int32_t q_heads, int32_t rows, int32_t span, NarrowShape& s, const char* who) {
    const std::string w(who);
    int rc = narrow_shape(c, s, who);
    if (rc) return rc;
    if (q_heads < 1 || q_heads > 65535 || q_heads % s.heads) return fail(SM_E_ARG, w + ": query heads are a multiple of the cache's heads");
    if (rows < 0 || rows > s.ctx) return fail(SM_E_ARG, w + ": rows are 0 .. ctx");
    if (span < 1 || span > s.ctx) return fail(SM_E_ARG, w + ": span is 1 .. ctx");
    if ((i64)rows * q_heads > (1 << 22) || (i64)s.streams * rows * q_heads > (1 << 26))
        return fail(SM_E_ARG, w + ": rows x query heads are at most 2^22, over all streams 2^26");
    return SM_OK;
}
extern "C" int64_t sm_narrow_work(const sm_narrow* c, int32_t q_heads, int32_t rows, int32_t span) {
    NarrowShape s;
    const int rc = narrow_att_args(c, q_heads, rows, span, s, "sm_narrow_work");
    return rc ? rc : narrow_work(s, rows * (q_heads / s.heads), (span + NCHUNK - 1) / NCHUNK).bytes;
}

template <int BITS, int DK>
static void narrow_attend(const NarrowAtt& a, bool sweep, hipStream_t st) {
    const unsigned heads = (unsigned)a.s.heads, streams = (unsigned)a.s.streams;
    if (sweep) {
        launch(g_kt.stages, "narrow.q", k_narrow_q<DK>, dim3((unsigned)((a.R * a.s.heads + 3) / 4), 1, streams), dim3(NTHREADS), 0, st, a);
        launch(g_kt.stages, "narrow.sweep", k_narrow_sweep<BITS, DK>, dim3((unsigned)((a.R + 15) / 16), heads, streams), dim3(64 * SWEEP_WAVES), 0, st, a);
        return;
    }
    const int gr = a.R <= 4 ? 4 : a.R <= 8 ? 8 : 16, rts = (a.R + gr - 1) / gr, jb = (a.J + NTHREADS / 64 - 1) / (NTHREADS / 64);
    // one launch where a block's waves hold all the chunks (one stream at 500 positions 9.1 us a call, 11.7 in two launches); of
    // eight chunks only with four rows a tile (the wider ones' work then stands in too few blocks: 15 rows of 5 heads, nine
    // streams at 1,733 positions, 26.5 us against 16.2 + 5.1)
    const dim3 tiles((unsigned)rts, heads, streams);
    auto near = [&](auto kern, int waves) { launch(g_kt.stages, "narrow.near", kern, tiles, dim3((unsigned)(64 * waves)), 0, st, a); };
    if (a.J <= 4) {
        if (a.R == 1) near(k_narrow_near<BITS, DK, 4, 1, 4>, 4);
        else if (gr == 4) near(k_narrow_near<BITS, DK, 4, 4, 4>, 4);
        else if (gr == 8) near(k_narrow_near<BITS, DK, 8, 4, 4>, 4);
        else near(k_narrow_near<BITS, DK, 16, 4, 4>, 4);
        return;
    }
    if (a.J <= 8 && gr == 4) {
        if (a.R == 1) near(k_narrow_near<BITS, DK, 4, 1, 8>, 8);
        else near(k_narrow_near<BITS, DK, 4, 4, 8>, 8);
        return;
    }
    const dim3 grid((unsigned)(jb * rts), heads, streams);
    auto split = [&](auto kern) { launch(g_kt.stages, "narrow.split", kern, grid, dim3(NTHREADS), 0, st, a, jb); };
    if (a.R == 1) split(k_narrow_split<BITS, DK, 4, 1>);
    else if (gr == 4) split(k_narrow_split<BITS, DK, 4, 4>);
    else if (gr == 8) split(k_narrow_split<BITS, DK, 8, 4>);
    else split(k_narrow_split<BITS, DK, 16, 4>);
    const int db = a.J > 64 ? 8 : a.s.wide;
    launch(g_kt.stages, "narrow.join", k_narrow_join, dim3((unsigned)(a.R * (a.s.wide / db)), heads, streams), dim3(NTHREADS), 0, st, a, db);
}

extern "C" int sm_narrow_attend(const sm_tables* t, const sm_narrow* c, const void* buf, const int64_t* q, int64_t q_row, int64_t q_stream,
                                int32_t q_heads, int32_t rows, int32_t span, const int32_t* start, const int32_t* count, int32_t scale,
                                int64_t* out, int64_t out_row, int64_t out_stream, void* work, int64_t work_bytes, void* stream) {
    NarrowAtt a{};
    if (!t) return fail(SM_E_ARG, "sm_narrow_attend: null tables");
    int rc = narrow_att_args(c, q_heads, rows, span, a.s, "sm_narrow_attend");
    if (rc || !rows) return rc;
    if (!buf || !q || !start || !out || !work) return fail(SM_E_ARG, "sm_narrow_attend: null argument");
    const i64 width = (i64)q_heads * a.s.dim;
    if (q_row < width || out_row < width || q_stream < 0 || out_stream < 0) return fail(SM_E_ARG, "sm_narrow_attend: strides");
    if (rows_overlap(a.s.streams, rows, width, out_row, out_stream)) return fail(SM_E_ARG, "sm_narrow_attend: the strides lay results over one another");
    if (scale < -(64 << 16) || scale > (64 << 16)) return fail(SM_E_ARG, "sm_narrow_attend: the scale's log2 is out of range");
    if (((uintptr_t)buf | (uintptr_t)work) & 15 || ((uintptr_t)q | (uintptr_t)out) & 7 || (uintptr_t)start & 3)
        return fail(SM_E_ARG, "sm_narrow_attend: alignment (cache and work 16 bytes, rows 8)");
    a.group = q_heads / a.s.heads; a.rows = rows; a.R = rows * a.group; a.J = (span + NCHUNK - 1) / NCHUNK;
    if ((i64)((a.J + 3) / 4) * ((a.R + 3) / 4) > (1 << 23)) return fail(SM_E_ARG, "sm_narrow_attend: too many rows at this span for one call");
    const NarrowWork w = narrow_work(a.s, a.R, a.J);
    if (work_bytes < w.bytes) return fail(SM_E_ARG, "sm_narrow_attend: the workspace is smaller than sm_narrow_work");
    if (!t->ARRF || t->alen > SWEEP_ARR) return fail(SM_E_ARG, "sm_narrow_attend: the tables' arrival is not base2_convert.py's");
    OnDevice on(buf);
    if (!on.ok) return fail(SM_E_ARG, "sm_narrow_attend: the cache is not in a device's memory");
    if (on.dev != t->dev) return fail(SM_E_ARG, "sm_narrow_attend: the tables are another device's");
    char* wk = static_cast<char*>(work);
    a.buf = static_cast<const char*>(buf);
    a.q = (const i64*)q; a.q_row = q_row; a.q_stream = q_stream; a.out = (i64*)out; a.o_row = out_row; a.o_stream = out_stream;
    a.start = start; a.count = count; a.span = span; a.F = scale; a.tb = t->tb();
    a.q8 = reinterpret_cast<signed char*>(wk + w.q8); a.eq = reinterpret_cast<int*>(wk + w.eq); a.pos = reinterpret_cast<int*>(wk + w.pos);
    a.pm = reinterpret_cast<int*>(wk + w.pm); a.WF = t->ARRF; a.pA = reinterpret_cast<int*>(wk + w.pA); a.pE = reinterpret_cast<int*>(wk + w.pE);
    a.pN = reinterpret_cast<int*>(wk + w.pN);
    hipStream_t st = (hipStream_t)stream;
    if (a.s.bits == 4) a.s.wide == 64 ? narrow_attend<4, 1>(a, w.sweep, st) : a.s.wide == 128 ? narrow_attend<4, 2>(a, w.sweep, st) : narrow_attend<4, 4>(a, w.sweep, st);
    else a.s.wide == 64 ? narrow_attend<8, 1>(a, w.sweep, st) : a.s.wide == 128 ? narrow_attend<8, 2>(a, w.sweep, st) : narrow_attend<8, 4>(a, w.sweep, st);
    HIP_TRY(hipGetLastError());
    return SM_OK;
}
