// Host-only check of the page bounds' C++ face up to each sequence's length: every call here fails
// host validation, so no device is touched.
#include <cstdio>
#include <stdexcept>

#include "reef_hip/attention.hpp"

template <typename E, typename F>
static int fails(const char *name, F f) {
    try {
        f();
    } catch (const E &e) {
        std::printf("ok   %s: %s\n", name, e.what());
        return 0;
    } catch (const std::exception &e) {
        std::printf("FAIL %s: wrong exception '%s'\n", name, e.what());
        return 1;
    }
    std::printf("FAIL %s: no exception\n", name);
    return 1;
}

int main() {
    // Non-null, aligned host addresses: validation never dereferences them.
    auto *i8 = reinterpret_cast<int8_t *>(0x10000);
    auto *u8 = reinterpret_cast<uint8_t *>(0x20000);
    auto *f32 = reinterpret_cast<float *>(0x30000);
    auto *i32 = reinterpret_cast<int32_t *>(0x40000);
    const reef_kv_append_params rows{2, 2, 128, 64, 64}, many{2, 2, 128, 65, 64};
    int failed = 0;
    failed += fails<std::length_error>("more tokens than the int8 cache holds", [&] {
        reef_hip::kv_page_bounds(many, i32, i32, i8, f32, nullptr, 0, 0, i8, f32, nullptr, nullptr);
    });
    failed += fails<std::length_error>("more tokens than the 4-bit cache holds", [&] {
        reef_hip::kv_page_bounds(many, i32, i32, u8, f32, nullptr, 0, 0, i8, f32, nullptr, nullptr);
    });
    failed += fails<std::invalid_argument>("a table of too few blocks", [&] {
        reef_hip::kv_page_bounds(rows, i32, i32, i8, f32, i32, 3, 9, i8, f32, nullptr, nullptr);
    });
    failed += fails<std::invalid_argument>("no lengths", [&] {
        const int32_t *none = nullptr;
        reef_hip::kv_page_bounds(rows, i32, none, u8, f32, nullptr, 0, 0, i8, f32, nullptr, nullptr);
    });
    return failed;
}
