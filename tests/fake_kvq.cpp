// Calls of the entry points for caches in fewer bits over the pretended HIP
// runtime of fake_hip.cpp: every line of stdin is an entry point's name and
// its arguments in order, pointers as 0 (null), 1 (16-byte aligned) or 2
// (misaligned), a scaling as five numbers and mscale, or "-". Prints
// "<status> <kernels launched ...>" a line, and the message of an error.
#define main fake_hip_main
#include "fake_hip.cpp"
#undef main

#include <iostream>
#include <sstream>

static std::istringstream* in;
static int I() {
    int v;
    if (!(*in >> v)) std::exit(3);
    return v;
}
static double D() {
    double v;
    if (!(*in >> v)) std::exit(3);
    return v;
}
static char* P() {
    static int n;
    const int v = I();
    return v ? (char*)((uintptr_t)++n << 32) + (v == 2 ? 4 : 0) : nullptr;
}
static char* Same(char* other) {  // 3: the pointer given before
    std::streampos at = in->tellg();
    if (I() == 3) return other;
    in->seekg(at);
    return P();
}

int main() {
    std::string line;
    bool init = false;
    while (std::getline(std::cin, line)) {
        std::istringstream s(line);
        in = &s;
        std::string w;
        s >> w;
        launches.clear();
        long long rc = 0;
        if (w == "init") rc = orc_init(0), init = true;
        else if (w == "bytes") { int a = I(), b = I(), c = I(), d = I(), e = I(); rc = (long long)orc_kvq_bytes(a, b, c, d, e); }
        else if (w == "work") { int a = I(), b = I(), c = I(), d = I(), e = I(), f = I(), g = I(); rc = (long long)orc_attn_kvq_workspace(a, b, c, d, e, f, g); }
        else if (w == "table") {
            float* p = (float*)P();
            int a = I(), b = I(), c = I();
            double base = D();
            std::string more;
            orc_rope_scaling sc{}, *scp = nullptr;
            std::streampos at = s.tellg();
            if (s >> more && more != "-") {
                s.clear();
                s.seekg(at);
                sc.kind = I(); sc.factor = (float)D(); sc.low = (float)D(); sc.high = (float)D(); sc.orig_ctx = I(); sc.mscale = (float)D();
                scp = &sc;
            }
            rc = orc_rope_table(p, a, b, c, base, scp, nullptr);
        } else if (w == "store") {
            int type = I();
            char* qkv = P();
            int ld = I(), ns = I(), nt = I(), h = I(), kv = I(), hd = I(), lay = I(), rot = I();
            char* rope = P();
            int ro = I();
            char* pos = P();
            int off = I();
            char* q = Same(qkv);
            int ldq = I();
            char *k = P(), *v = P();
            int ctx = I();
            rc = orc_kvq_store(type, (float*)qkv, ld, ns, nt, h, kv, hd, lay, rot, (float*)rope, ro, (int32_t*)pos, off, (float*)q, ldq, k, v, ctx, nullptr);
        } else if (w == "load") {
            int type = I();
            char *k = P(), *v = P();
            int ns = I(), kv = I(), hd = I(), ctx = I();
            char* pos = P();
            int off = I(), n = I();
            char *ko = P(), *vo = P();
            rc = orc_kvq_load(type, k, v, ns, kv, hd, ctx, (int32_t*)pos, off, n, (float*)ko, (float*)vo, nullptr);
        } else if (w == "attn") {
            int type = I();
            char* q = P();
            int ldq = I(), ns = I(), nt = I(), h = I(), kv = I(), hd = I();
            char *pk = P(), *pv = P();
            int pl = I(), pc = I();
            char *k = P(), *v = P();
            int ctx = I();
            char* pos = P();
            int off = I(), lim = I();
            char* o = P();
            int ldo = I();
            char* work = P();
            rc = orc_attn_kvq(type, (float*)q, ldq, ns, nt, h, kv, hd, pk, pv, pl, pc, k, v, ctx, (int32_t*)pos, off, lim, (float*)o, ldo, work, nullptr);
        } else return 4;
        std::cout << rc;
        if (w != "init")
            for (const std::string& l : launches) std::cout << " " << l.substr(l.rfind(' ') + 1);
        if (rc < 0) std::cout << " | " << orc_last_error();
        std::cout << std::endl;
    }
    return init ? 0 : 0;
}
