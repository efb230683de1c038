// gl3_create_err.h — what gl3_last_error(NULL) returns: errors of calls without a plan (creating one, operators).  Included once by a library's entry points.
#pragma once
#include <mutex>
#include <string>

static thread_local std::string g_create_err;          // the calling thread's own: operators are called from several at once
static std::mutex g_any_mu;
static std::string g_any_err;                          // the newest of all threads: what a thread without an error of its own reads

static void publish_create_error() {
    try {
        std::lock_guard<std::mutex> lock(g_any_mu);
        g_any_err = g_create_err;
    } catch (...) {}
}
void gl3_set_create_error(const char* msg) {
    try { g_create_err = msg ? msg : ""; } catch (...) { g_create_err.clear(); }
    publish_create_error();
}
static const char* create_error() {
    if (!g_create_err.empty()) return g_create_err.c_str();
    static thread_local std::string seen;
    try {
        std::lock_guard<std::mutex> lock(g_any_mu);
        seen = g_any_err;
    } catch (...) { seen.clear(); }
    return seen.c_str();
}
