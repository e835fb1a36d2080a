// Argument rules of the feed-forward operators on tensor descriptors, without a GPU: every call that stands and every refusal.
#include <cstdio>

#include "../../reference_model_b200/csrc/ffn_check.cu"

using namespace tb200::ffn;

static int bad = 0;
static char memory[1 << 16];
static size_t used = 0;

static tb200_tensor make(tb200_dtype dt, std::initializer_list<int> shape)
{
    tb200_tensor t = {};
    t.dtype = dt;
    t.bytes = tb200::dtype_size(dt);
    for (int s : shape)
    {
        t.shape[t.rank++] = s;
        t.bytes *= (size_t)s;
    }
    t.data = memory + used;
    used += (t.bytes + 15) & ~(size_t)15;
    t.contiguous = true;
    return t;
}

static void expect(const char* what, const std::string& got, const char* part)
{
    const bool ok = *part ? got.find(part) != std::string::npos : got.empty();
    if (!ok)
    {
        printf("%s: got \"%s\", expected %s\n", what, got.c_str(), *part ? part : "none");
        bad++;
    }
}

template <typename F>
static void w4(const char* what, const char* part, F change)
{
    used = 0;
    tb200_tensor a = make(TB200_FP16, { 2, 3, 70 }), d = make(TB200_INT8, { 5, 48 }), s = make(TB200_BF16, { 3, 5 }), z = make(TB200_INT8, { 3, 5 }),
                 o = make(TB200_FP16, { 2, 3, 5 });
    tb200_w4 m = { &d, &s, &z, 32 }, m2 = m;
    const tb200_w4* mats[2] = { &m, &m2 };
    int n = 1, act = 0;
    change(a, d, s, z, o, m, m2, n, act);
    expect(what, check_w4("op", &a, mats, n, act, &o), part);
}

template <typename F>
static void gated(const char* what, const char* part, F change)
{
    used = 0;
    tb200_tensor a = make(TB200_BF16, { 2, 3, 7 }), g = make(TB200_BF16, { 2, 7, 5 }), u = make(TB200_BF16, { 2, 7, 5 }), o = make(TB200_BF16, { 2, 3, 5 }),
                 da = make(TB200_BF16, { 2, 3, 7 }), dg = make(TB200_FP32, { 2, 7, 5 }), du = make(TB200_BF16, { 2, 7, 5 });
    int act = 1;
    tb200_tensor *pa = &da, *pg = &dg, *pu = &du;
    change(a, g, u, o, act, pa, pg, pu);
    std::string why = check_gated("op", &a, &g, &u, act, &o, "output");
    if (why.empty())
        why = check_gated_output("op", &a, &g, &u, &o);
    if (why.empty())
        why = check_gated_grads("op", &a, &g, &u, &o, pa, pg, pu);
    expect(what, why, part);
}

#define W4(what, part, code) w4(what, part, [](tb200_tensor& a, tb200_tensor& d, tb200_tensor& s, tb200_tensor& z, tb200_tensor& o, tb200_w4& m, tb200_w4& m2, int& n, int& act) { \
    (void)a, (void)d, (void)s, (void)z, (void)o, (void)m, (void)m2, (void)n, (void)act; code; })
#define GATED(what, part, code) gated(what, part, [](tb200_tensor& a, tb200_tensor& g, tb200_tensor& u, tb200_tensor& o, int& act, tb200_tensor*& pa, tb200_tensor*& pg, tb200_tensor*& pu) { \
    (void)a, (void)g, (void)u, (void)o, (void)act, (void)pa, (void)pg, (void)pu; code; })

int main()
{
    W4("plain", "", );
    W4("fp32 out", "", o = make(TB200_FP32, { 2, 3, 5 }));
    W4("one group", "", m.group = 70; s = make(TB200_FP32, { 1, 5 }); z = make(TB200_INT8, { 1, 5 }));
    W4("one group of any size", "", m.group = 1000; s = make(TB200_FP32, { 1, 5 }); m.zero = nullptr);
    W4("uint8 rows, tight", "", d = make(TB200_UINT8, { 5, 35 }));
    W4("two matrices", "", n = 2);
    W4("null data", "null operand", m.data = nullptr);
    W4("null scale", "null operand", n = 2; m2.scale = nullptr);
    W4("rank of a", "rank 3", a = make(TB200_FP16, { 6, 70 }));
    W4("view", "contiguous", a.contiguous = false);
    W4("view of weights", "contiguous", d.contiguous = false);
    W4("type of a", "FP16, BF16 or FP32", a.dtype = TB200_INT8);
    W4("type of out", "output dtype", o.dtype = TB200_BF16);
    W4("rows of out", "first two", o = make(TB200_FP16, { 2, 4, 5 }));
    W4("weights' type", "bytes", d.dtype = TB200_INT16);
    W4("weights' rank", "rank 2", d = make(TB200_INT8, { 1, 5, 48 }));
    W4("weights' rows", "a row for each", d = make(TB200_INT8, { 6, 48 }));
    W4("weights' pitch", "does not hold", d = make(TB200_INT8, { 5, 34 }));
    W4("group 0", "multiple of 32", m.group = 0);
    W4("group -32", "multiple of 32", m.group = -32);
    W4("group 48", "multiple of 32", m.group = 48);
    W4("scale's type", "scales must be FP16", s.dtype = TB200_INT16);
    W4("scale's shape", "scales must be [3,5]", s = make(TB200_BF16, { 5, 3 }));
    W4("zero's type", "zero points must be", z.dtype = TB200_UINT8);
    W4("zero's shape", "zero points must be", z = make(TB200_INT8, { 2, 5 }));
    W4("groups differ", "same group", n = 2; m2.group = 128; static tb200_tensor s2; s2 = make(TB200_BF16, { 1, 5 }); m2.scale = &s2; m2.zero = nullptr);
    W4("activation", "unknown activation", n = 2; act = 5);
    W4("output over a", "overlaps", o.data = a.data);
    W4("output over scales", "overlaps", o.data = s.data);
    W4("output over the weights' last byte", "overlaps", o.data = (char*)d.data + d.bytes - 1);

    GATED("plain", "", );
    GATED("shared weights", "", g = make(TB200_BF16, { 1, 7, 5 }); u = make(TB200_BF16, { 1, 7, 5 }); pg = nullptr; pu = nullptr);
    GATED("one gradient", "", pa = nullptr; pg = nullptr);
    GATED("rank", "rank 3", g = make(TB200_BF16, { 7, 5 }));
    GATED("view", "contiguous", u.contiguous = false);
    GATED("types differ", "dtypes differ", u.dtype = TB200_FP16);
    GATED("int", "FP16, BF16 or FP32", a.dtype = TB200_INT16; g.dtype = TB200_INT16; u.dtype = TB200_INT16);
    GATED("batches", "one for each", g = make(TB200_BF16, { 3, 7, 5 }));
    GATED("depth", "gate.shape[1]", g = make(TB200_BF16, { 2, 6, 5 }));
    GATED("up's shape", "same shape", u = make(TB200_BF16, { 2, 7, 6 }));
    GATED("output's shape", "output must be [2,3,5]", o = make(TB200_BF16, { 2, 5, 3 }));
    GATED("output's type", "output dtype", o.dtype = TB200_FP16);
    GATED("activation", "unknown activation", act = -1);
    GATED("output over a", "overlaps", o.data = a.data);
    GATED("output's gradient in fp32", "output's gradient", o = make(TB200_FP32, { 2, 3, 5 }));
    GATED("no gradient", "no gradient", pa = pg = pu = nullptr);
    GATED("gradient's view", "contiguous", pa->contiguous = false);
    GATED("gradient's type", "grad_a must have", pa->dtype = TB200_FP16);
    GATED("gradient's shape", "grad_up must have its operand's shape", *pu = make(TB200_BF16, { 1, 7, 5 }));
    GATED("gradient over an operand", "grad_gate overlaps", pg->data = u.data);
    GATED("gradients overlap", "two gradients", pu->data = pa->data);
    if (!bad)
        printf("ok\n");
    return bad != 0;
}
