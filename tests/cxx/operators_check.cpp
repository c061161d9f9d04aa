// Host-only check of the drafted-token and page calls of include/reef_hip/attention.hpp:
// every call here fails host validation, so no device is touched.
#include <cstdio>
#include <stdexcept>

#include "reef_hip/attention.hpp"

static int failures = 0;

template <typename E, typename F>
static void expect(const char *name, F f) {
    try {
        f();
        std::printf("FAIL %s: no exception\n", name);
    } catch (const E &e) {
        std::printf("ok   %s: %s\n", name, e.what());
        return;
    } catch (const std::exception &e) {
        std::printf("FAIL %s: wrong exception '%s'\n", name, e.what());
    }
    ++failures;
}

int main() {
    // Non-null, aligned host addresses: validation never dereferences them.
    auto *i8 = reinterpret_cast<int8_t *>(0x10000);
    auto *f32 = reinterpret_cast<float *>(0x20000);
    auto *i32 = reinterpret_cast<int32_t *>(0x30000);
    auto *u64 = reinterpret_cast<uint64_t *>(0x40000);

    reef_tree_params tree{2, 8, 2, 128, 5, 64, 0, 0.1f, REEF_SCALE_PER_TOKEN, 0, 0};
    const size_t bytes = reef_hip::tree_workspace_bytes(tree);
    if (bytes == 0) {
        std::printf("FAIL tree workspace\n");
        ++failures;
    }
    expect<std::invalid_argument>("tree with a short workspace", [&] {
        reef_hip::decode_tree(tree, i8, nullptr, f32, i8, i8, f32, f32, i32, u64, f32, nullptr, i8,
                              bytes - 1, nullptr, nullptr);
    });
    expect<std::invalid_argument>("paged tree with a short table", [&] {
        reef_hip::decode_tree_paged(tree, i8, nullptr, f32, i8, i8, f32, f32, i32, 3, 9, i32, u64,
                                    f32, nullptr, i8, bytes, nullptr, nullptr);
    });
    reef_tree_params wide = tree;
    wide.draft_len = 65;
    expect<reef_hip::unsupported>("65 drafted tokens", [&] {
        reef_hip::decode_tree(wide, i8, nullptr, f32, i8, i8, f32, f32, i32, u64, f32, nullptr, i8,
                              1 << 30, nullptr, nullptr);
    });
    reef_tree_params full = tree;
    full.draft_len = 17;
    full.max_context = 16;
    expect<std::length_error>("more drafted tokens than the cache holds", [&] {
        reef_hip::decode_tree(full, i8, nullptr, f32, i8, i8, f32, f32, i32, u64, f32, nullptr, i8,
                              1 << 30, nullptr, nullptr);
    });
    const reef_kv_append_params rows{2, 2, 128, 5, 64};
    expect<std::invalid_argument>("keep whose lengths overlap", [&] {
        reef_hip::kv_keep(rows, i32, i32, i32, i8, i8, f32, f32, i32 + 1, nullptr, nullptr);
    });
    expect<std::invalid_argument>("paged keep without a table", [&] {
        reef_hip::kv_keep_paged(rows, i32, i32, i32, nullptr, 4, 9, i8, i8, f32, f32, nullptr,
                                nullptr, nullptr);
    });
    expect<reef_hip::unsupported>("copy of pages of head_dim 96", [&] {
        reef_hip::kv_copy_pages(i32, i32, 1, 2, 96, i8, i8, f32, f32, 9, nullptr, nullptr);
    });

    const reef_hip::page_table table{i32, 4, 10, i32, i32, 100};
    expect<std::invalid_argument>("free of no sequences",
                                  [&] { table.free(i32, 0, nullptr, nullptr); });
    expect<std::invalid_argument>("fork without children",
                                  [&] { table.fork(i32, nullptr, 1, nullptr, nullptr); });
    expect<std::length_error>("reserve past the table", [&] {
        table.reserve(161, i32, i32, i8, table.reserve_workspace_bytes(161), nullptr, nullptr);
    });
    expect<std::invalid_argument>("compact with a short workspace", [&] {
        table.compact(i32, i32, nullptr, i8, table.compact_workspace_bytes() - 1, nullptr, nullptr);
    });

    const reef_epilogue unknown{nullptr, 0, 9}, narrow{f32, 7, REEF_ACT_SILU};
    expect<std::invalid_argument>("an unknown activation", [&] {
        reef_hip::gemm_w8a8(i8, f32, 4, 16, i8, f32, nullptr, unknown, 8, f32, 8, nullptr, nullptr);
    });
    expect<std::invalid_argument>("residual rows closer than their width", [&] {
        reef_hip::linear_w8a8(f32, 4, 16, 16, i8, f32, nullptr, narrow, 8, f32, 8, i8, 1 << 20,
                              nullptr, nullptr);
    });
    expect<std::invalid_argument>("norm with a sum and no residual", [&] {
        reef_hip::rmsnorm_quantize(f32, 4, 16, 16, nullptr, 0, nullptr, 1e-6, i8, f32, f32, 16,
                                   nullptr, nullptr);
    });
    std::printf("%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
