// mfar_error.h -- the error slot of libmfar_hip.so, shared by its translation units (hidden: no part of the C ABI).
#pragma once
// Stores `msg` as this thread's mfar_last_error() and returns `code`.
__attribute__((visibility("hidden"))) int mfar_report(int code, const char* msg);
