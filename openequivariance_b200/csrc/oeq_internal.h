// What the translation units of liboeq_b200.so share.
#pragma once
#include <string>

// Sets the calling thread's error text (oeq_last_error) and returns `code`.
__attribute__((visibility("hidden"))) int oeq_fail(int code, const std::string& message);
