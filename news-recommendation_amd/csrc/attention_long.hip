// Softmax attention of any length: which kernels, how split, and their launch (kernels: attention_long_fwd.h, attention_long_bwd.h)
#include "attention_long_dev.h"
#include <algorithm>

namespace nr {
namespace al {

Args make_args(const AttnProblem& p) {
    Args a{};
    a.q = p.q; a.k = p.k; a.v = p.v; a.mask = p.key_mask;
    a.sq = p.sq; a.sk = p.sk; a.sv = p.sv;
    a.N = p.N; a.Sq = p.Sq; a.Sk = p.Sk; a.H = p.H; a.G = p.G; a.rep = p.H / p.G; a.dh = p.dh; a.dhs = (p.dh + 3) / 4 * 4;
    a.R = a.rep * p.Sq;
    a.causal = p.causal; a.additive = p.additive; a.scale = p.scale; a.fill = p.dc.mask_fill;
    a.keep = p.dc.p > 0.f ? 1.f / (1.f - p.dc.p) : 1.f;
    a.thr = drop_threshold(p.dc.p); a.site = p.dc.site; a.seed = p.dc.seed;
    a.splits = 1;
    return a;
}
static bool all_aligned(const AttnProblem& p) {
    const size_t e = p.bf16 ? 2 : 4;
    return aligned16(p.q, p.sq, p.dh, e, 128) && aligned16(p.k, p.sk, p.dh, e, 128) && aligned16(p.v, p.sv, p.dh, e, 128);
}
// Workgroups that do not reach every CU split `length` further, to about two per CU and down to 256 of it each.  Both sides, us of device
// time, forward / forward and backward: 15 rows over 20011 keys, 4 x 4 key heads of 64, bf16: split 21 / 123, whole 139 / 353; one sequence of 2048,
// 12 heads of 64: bf16 36.5 / 135 and 36 / 155, fp32 104 / 437 and 115 / 478; one of 1000, 8 heads of 128, fp32: 58 / 227 and 112 / 483;
// single queries over 1000 keys, 8 x 12 heads of 64, bf16: 12 / 44 either way.  Other aims: one workgroup per CU 34.7 / 135 (bf16) and 94 /
// 384 (fp32) on the sequence of 2048, but four 40 / 157 and 102 / 416.  Down to 128: fp32 wins where few heads are short (one sequence of 512,
// 12 heads of 64: 35 / 135 whole, 20 / 76 in four), bf16 loses where they are more (4 x 512: 12.7 / 53 whole, 19 / 74).
static Split split_axis(int64_t blocks, int length, int unit) {
    Split s{1, length};
    if (blocks <= 0 || blocks >= 256 || length <= 512) return s;
    const int64_t want = std::min<int64_t>((512 + blocks - 1) / blocks, length / 256);
    s.per = (int)((((int64_t)length + want - 1) / want + unit - 1) / unit * unit);
    s.splits = (length + s.per - 1) / s.per;
    return s;
}
// causal rows go by blocks of one query head, so that the blocks with most keys can come first
static int head_blocks(const AttnProblem& p, int rows) { return p.causal && p.Sq >= rows ? cdiv(p.Sq, rows) : 0; }

struct FwdPlan { int wk, nblk, head_blocks; Split sp; size_t ws; };
static FwdPlan plan_fwd(const AttnProblem& p) {
    FwdPlan f;
    const int64_t R = (int64_t)(p.H / p.G) * p.Sq;
    // Few rows share the waves.  33 to 64 of them could in two blocks: better where they have many keys or few heads (64 x 1000 keys, 32 x 4
    // heads of 64, bf16: 18 us as here, 13 shared; 36 x 200, fp32: 14 and 10), worse where there are blocks enough (50 x 50, 64 x 12 heads of
    // 64, bf16: 7.5 and 17 us; 33 x 300, 32 x 12: 11 and 15).
    f.wk = R <= 32 ? 4 : 1;
    f.head_blocks = f.wk == 1 ? head_blocks(p, 128) : 0;
    f.nblk = f.head_blocks ? p.H / p.G * f.head_blocks : cdiv(R, 32 * (4 / f.wk));
    f.sp = split_axis(p.N * p.G * f.nblk, p.Sk, 128);
    const size_t rows = (size_t)(p.N * p.G * R);
    f.ws = f.sp.splits > 1 ? f.sp.splits * rows * (size_t)((p.dh + 3) / 4 * 4 + 2) * 4 : 0;
    return f;
}
static BwdPlan plan_bwd(const AttnProblem& p) {
    BwdPlan f;
    const int64_t R = (int64_t)(p.H / p.G) * p.Sq;
    f.wk = R <= 32 ? 4 : 1;
    f.head_blocks = f.wk == 1 ? head_blocks(p, 128) : 0;
    f.nblk_q = f.head_blocks ? p.H / p.G * f.head_blocks : cdiv(R, 32 * (4 / f.wk));
    f.nblk_k = cdiv(p.Sk, 128);
    f.q = split_axis(p.N * p.G * f.nblk_q, p.Sk, 128);
    f.kv = split_axis(p.N * p.G * f.nblk_k, (int)R, 64);
    const size_t row = (size_t)((p.dh + 3) / 4 * 4) * 4;
    const size_t wq = f.q.splits > 1 ? f.q.splits * (size_t)(p.N * p.G * R) * row : 0;
    const size_t wk = f.kv.splits > 1 ? 2 * f.kv.splits * (size_t)(p.N * p.G * p.Sk) * row : 0;
    f.ws = std::max(wq, wk);                     // the two passes run one after the other
    return f;
}

extern template int run_fwd<float>(const Args&, bool, bool, int, unsigned, hipStream_t);
extern template int run_fwd<__bf16>(const Args&, bool, bool, int, unsigned, hipStream_t);
extern template int run_bwd<float>(Args, const BwdPlan&, bool, bool, bool, hipStream_t);
extern template int run_bwd<__bf16>(Args, const BwdPlan&, bool, bool, bool, hipStream_t);

}  // namespace al

size_t attn_long_fwd_ws_bytes(const AttnProblem& p) { return al::plan_fwd(p).ws; }

int attn_long_fwd(const AttnProblem& p, const AttnOut& o, void* ws, size_t ws_bytes, hipStream_t s) {
    if (p.N == 0 || p.Sq == 0) return NR_OK;
    const al::FwdPlan f = al::plan_fwd(p);
    al::Args a = al::make_args(p);
    a.out = o.out; a.so = o.so; a.row_max = o.row_max; a.row_sum = o.row_sum;
    a.nblk = f.nblk; a.head_blocks = f.head_blocks; a.splits = f.sp.splits; a.per_split = f.sp.per;
    if (f.ws && (!ws || ws_bytes < f.ws)) {      // without room for the joins the keys stay with one workgroup
        a.splits = 1; a.per_split = p.Sk;
    } else if (f.ws) {
        a.part = static_cast<float*>(ws);
        a.part_ml = a.part + (size_t)a.splits * (p.N * p.G * a.R) * a.dhs;
    }
    const int64_t grid = p.N * p.G * (int64_t)a.nblk * a.splits;
    NR_UNSUPPORTED(grid > 0x7fffffff, "attention_fwd: %lld workgroups", (long long)grid);
    const bool vec = al::all_aligned(p) && al::aligned16(o.out, o.so, p.dh, p.bf16 ? 2 : 4, 128), drop = p.dc.p > 0.f;
    return p.bf16 ? al::run_fwd<__bf16>(a, vec, drop, f.wk, (unsigned)grid, s) : al::run_fwd<float>(a, vec, drop, f.wk, (unsigned)grid, s);
}

size_t attn_long_bwd_ws_bytes(const AttnProblem& p) { return al::plan_bwd(p).ws; }

int attn_long_bwd(const AttnProblem& p, const AttnGrad& g, void* ws, size_t ws_bytes, hipStream_t s) {
    if (p.N == 0 || p.Sq == 0 || p.Sk == 0) return NR_OK;
    const al::BwdPlan f = al::plan_bwd(p);
    const int64_t grid = p.N * p.G * std::max<int64_t>((int64_t)f.nblk_k * f.kv.splits, (int64_t)f.nblk_q * f.q.splits);
    const int64_t rows = p.N * p.Sq * p.H;
    NR_UNSUPPORTED(grid > 0x7fffffff || rows > ((int64_t)1 << 34), "attention_bwd: %lld workgroups, %lld rows", (long long)grid, (long long)rows);
    al::Args a = al::make_args(p);
    a.out = const_cast<void*>(g.out); a.so = g.so; a.dout = g.dout; a.sdo = g.sdo;
    a.row_max = const_cast<float*>(g.row_max); a.row_sum = const_cast<float*>(g.row_sum);
    a.delta = g.delta; a.sd = g.sd; a.keep_delta = static_cast<const void*>(g.delta) != g.dq;
    a.dq = g.dq; a.dk = g.dk; a.dv = g.dv; a.sdq = g.sdq; a.sdk = g.sdk; a.sdv = g.sdv;
    a.part = static_cast<float*>(ws);
    const size_t e = p.bf16 ? 2 : 4;
    const bool vec = al::all_aligned(p) && al::aligned16(g.dout, g.sdo, p.dh, e, 128) && al::aligned16(g.out, g.so, p.dh, e, 128) && al::aligned16(g.dq, g.sdq, p.dh, e, 128);
    const bool room = !f.ws || (ws && ws_bytes >= f.ws), drop = p.dc.p > 0.f;      // without room for the partial sums nothing is split
    return p.bf16 ? al::run_bwd<__bf16>(a, f, vec, drop, room, s) : al::run_bwd<float>(a, f, vec, drop, room, s);
}

}  // namespace nr
