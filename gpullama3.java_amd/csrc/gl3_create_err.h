// gl3_create_err.h — what gl3_last_error(NULL) returns: errors of calls without a plan (making one, operators).  Included once by a library's entry points.
//
// Plans are often made in one thread and the message read in another, so a plan that could not be made is told to every thread.  Operators are called from several
// threads at once, so a refused one is told to its own thread, which keeps it until its next call without a plan.
#pragma once
#include <mutex>
#include <string>

static thread_local std::string g_op_err;                  // this thread's operator error
static thread_local bool g_op = false, g_made = false;     // this thread's last call without a plan: an operator that failed; a plan that could not be made
static std::mutex g_any_mu;
static std::string g_create_err, g_any_err;                // the newest of all threads: of making plans, and of either kind

static void gl3_put_error(bool op, const char* msg) {
    g_op = op; g_made = !op;
    try {
        std::lock_guard<std::mutex> lock(g_any_mu);
        g_any_err = msg ? msg : "";
        if (op) g_op_err = g_any_err; else g_create_err = g_any_err;
    } catch (...) { g_op = g_made = false; }
}
void gl3_set_create_error(const char* msg) { gl3_put_error(false, msg); }
void gl3_set_op_error(const char* msg) { gl3_put_error(true, msg); }
void gl3_no_error() { g_op = g_made = false; }             // at the start of a call without a plan
static const char* create_error() {
    if (g_op) return g_op_err.c_str();
    static thread_local std::string seen;
    try {
        std::lock_guard<std::mutex> lock(g_any_mu);
        seen = g_made ? g_create_err : g_any_err;
    } catch (...) { seen.clear(); }
    return seen.c_str();
}
