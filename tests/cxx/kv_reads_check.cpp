// Host-only check of the 4-bit cache's and the page selection's calls of
// include/reef_hip/attention.hpp: every call here fails host validation, so no device is touched.
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
    auto *u8 = reinterpret_cast<uint8_t *>(0x20000);
    auto *f32 = reinterpret_cast<float *>(0x30000);
    auto *i32 = reinterpret_cast<int32_t *>(0x40000);

    const reef_kv_append_params rows{2, 2, 128, 5, 64}, many{2, 2, 128, 65, 64};
    expect<std::length_error>("more tokens than the cache holds", [&] {
        reef_hip::append_kv_cache_int4(many, f32, nullptr, f32, nullptr, i32, nullptr, 0, 0, u8, u8,
                                       f32, f32, nullptr, nullptr, nullptr);
    });
    expect<reef_hip::unsupported>("pages of head_dim 96", [&] {
        reef_hip::kv_unpack_int4(u8, u8, f32, f32, 1, 96, f32, f32, nullptr);
    });
    expect<reef_hip::unsupported>("copy of pages of head_dim 96", [&] {
        reef_hip::kv_copy_pages(i32, i32, 1, 2, 96, u8, u8, f32, f32, 9, nullptr, nullptr);
    });
    expect<std::length_error>("bounds of more tokens than the cache holds", [&] {
        reef_hip::kv_page_bounds(many, i32, i8, f32, nullptr, 0, 0, i8, f32, nullptr, nullptr);
    });
    expect<std::invalid_argument>("bounds with a short table", [&] {
        reef_hip::kv_page_bounds(rows, i32, u8, f32, i32, 3, 9, i8, f32, nullptr, nullptr);
    });

    const reef_decode_params step{2, 8, 2, 128, 64, 0, 0.1f, REEF_SCALE_PER_TOKEN, 0, 0};
    const size_t bytes = reef_hip::decode_workspace_bytes(step);
    const size_t words = reef_hip::select_workspace_bytes(step);
    if (bytes == 0 || words == 0) {
        std::printf("FAIL workspaces\n");
        ++failures;
    }
    expect<std::invalid_argument>("decode with a short workspace", [&] {
        reef_hip::decode_int4(step, i8, f32, u8, u8, f32, f32, nullptr, 0, 0, i32, nullptr, f32, i8,
                              bytes - 1, nullptr, nullptr);
    });
    const reef_page_selection none{i32, i32, 0};
    expect<std::invalid_argument>("decode over a list without pages", [&] {
        reef_hip::decode_selected(step, i8, f32, i8, i8, f32, f32, nullptr, 0, 0, i32, none, f32, i8,
                                  bytes, nullptr, nullptr);
    });
    expect<std::invalid_argument>("selection of no pages", [&] {
        reef_hip::kv_select_pages(step, i8, f32, i8, f32, nullptr, 0, 0, i32, 0, 0, 1, i32, i32, i8,
                                  words, nullptr, nullptr);
    });
    const reef_attention_params chunk{2, 8, 2, 8, 40, 128, 32, 0, 0.1f, REEF_SCALE_PER_HEAD,
                                      REEF_SCALE_PER_TOKEN, 0};
    expect<std::invalid_argument>("prefill over a cache that is too short", [&] {
        reef_hip::context_cache(chunk, i8, nullptr, f32, u8, u8, f32, f32, 32, nullptr, 0, 0, f32,
                                nullptr, i8, size_t(1) << 30, nullptr, nullptr);
    });
    std::printf("%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
