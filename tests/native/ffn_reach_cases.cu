// Which sizes the tiled feed-forward kernels take, without a GPU.
#include <cstdio>

#include "../../reference_model_b200/csrc/ffn_check.cu"

using namespace tb200::ffn;

static int bad = 0;

static void expect(const char* what, bool got, bool want)
{
    if (got != want)
    {
        printf("%s: %d\n", what, got);
        bad++;
    }
}

int main()
{
    expect("a long prompt", tiles_reach(1, 4096, 4096, 8192, true), true);
    expect("many batches", tiles_reach(70000, 1, 8, 8, true), true);
    expect("2^30 batches of one tile", tiles_reach(1 << 30, 1, 1, 1, false), true);
    expect("more", tiles_reach((1 << 30) + 1, 1, 1, 1, false), false);
    expect("the most that a tensor has", tiles_reach(0x7fffffff, 1, 1, 1, false), false);
    expect("2^30 tiles of both weights' gradients", tiles_reach(1 << 29, 1, 1, 1, true), true);
    expect("one batch more", tiles_reach((1 << 29) + 1, 1, 1, 1, true), false);
    expect("2^30 tiles of grad_a", tiles_reach(1 << 22, 256, 128 << 7, 1, true), true);
    expect("more of them", tiles_reach(1 << 22, 256, (128 << 7) + 1, 1, true), false);
    expect("forward only", tiles_reach(1 << 22, 256, (128 << 7) + 1, 1, false), true);
    expect("2^30 tiles of rows and columns", tiles_reach(1, 1 << 30, 64, 128 * 64, false), true);
    expect("one column more", tiles_reach(1, 1 << 30, 64, 128 * 64 + 1, false), false);
    expect("rows", tiles_reach(1, (1LL << 30) + 1, 1, 1, false), false);
    expect("all at once", tiles_reach(0x7fffffff, 1 << 30, 1 << 30, 1 << 29, true), false);
    if (!bad)
        printf("ok\n");
    return bad != 0;
}
