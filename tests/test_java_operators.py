"""The JNI natives of the operators, run against a JNIEnv of the test's own: what they refuse themselves leaves a text in opsError()."""
import os
import subprocess

from test_java_glue import JNI_H, ROOT, SHIM

DRIVER = r"""
#include <stdio.h>
#include <string.h>
#include "%(shim)s"
#define N(name) Java_com_omega_engine_nn_layer_llama_OmoeNative_##name
typedef struct { int n; void *p; } array;
static jsize length(JNIEnv *e, jarray a) { (void)e; return ((array *)a)->n; }
static jlong *longs(JNIEnv *e, jlongArray a, jboolean *c) { (void)e; (void)c; return ((array *)a)->p; }
static jint *ints(JNIEnv *e, jintArray a, jboolean *c) { (void)e; (void)c; return ((array *)a)->p; }
static void put_longs(JNIEnv *e, jlongArray a, jlong *p, jint m) { (void)e; (void)a; (void)p; (void)m; }
static void put_ints(JNIEnv *e, jintArray a, jint *p, jint m) { (void)e; (void)a; (void)p; (void)m; }
static jstring text(JNIEnv *e, const char *s) { (void)e; return (jstring)s; }
int main(void) {
    struct JNINativeInterface_ f;
    memset(&f, 0, sizeof f);
    f.GetArrayLength = length; f.GetLongArrayElements = longs; f.GetIntArrayElements = ints;
    f.ReleaseLongArrayElements = put_longs; f.ReleaseIntArrayElements = put_ints; f.NewStringUTF = text;
    JNIEnv table = &f, *env = &table;
    jlong values[9] = {4, 2, 8, 1, 8, 4096, 8192, 12288, 16384}, wide[9] = {(jlong)1 << 40, 2, 8, 1, 8, 4096, 8192, 12288, 16384};
    jint types[2] = {0, 0};
    array none = {0, NULL}, few = {8, values}, big = {9, wide}, two = {2, values}, one = {1, types};
    jlongArray plans[] = {NULL, (jlongArray)&none, (jlongArray)&few, (jlongArray)&big};
#define SHOW(call) do { \
        N(layerNorm)(env, NULL, 0, 8, 0, 0, 0, 0, 0, 8, 0, 0, 0, -1, 8); /* another failure before */ \
        jint rc = call; \
        printf("%%d %%s\n", (int)rc, (const char *)N(opsError)(env, NULL)); \
    } while (0)
    for (int i = 0; i < 4; i++) {
        SHOW(N(sortPlan)(env, NULL, plans[i], 65536));
        SHOW(N(sortRows)(env, NULL, plans[i], 65536, 8, 0, 131072, 8, 0, 8));
        SHOW(N(sortRowsBackward)(env, NULL, plans[i], 65536, 8, 0, 131072, 8, 0, 8));
        SHOW(N(unsortRows)(env, NULL, plans[i], 65536, 8, 0, 0, 131072, 8, 0, 8));
        SHOW(N(unsortRowsBackward)(env, NULL, plans[i], 65536, 8, 0, 131072, 8, 0, 0, 262144, 8, 0, 8));
    }
    jlongArray a = (jlongArray)&two;
    jintArray lists[] = {NULL, (jintArray)&one};
    for (int i = 0; i < 2; i++) {
        SHOW(N(gradNorm)(env, NULL, a, a, lists[i], 65536, 131072, 16384));
        SHOW(N(gradScale)(env, NULL, a, a, lists[i], 65536, 1.f));
        SHOW(N(gradClip)(env, NULL, a, a, lists[i], 1.f, 65536, 131072, 16384));
    }
    return 0;
}
"""


def test_refusals_of_the_shim_have_a_text(tmp_path):
    from omega_ai_b200 import native

    lib = native.build()
    (tmp_path / "jni.h").write_text(JNI_H)
    (tmp_path / "driver.c").write_text(DRIVER % {"shim": SHIM})
    exe = str(tmp_path / "driver")
    subprocess.check_call(["gcc", "-std=gnu11", "-Wall", "-Werror", "-I", str(tmp_path), "-I", os.path.join(ROOT, "include"), "-o", exe,
                           str(tmp_path / "driver.c"), lib, f"-Wl,-rpath,{os.path.dirname(lib)}"])
    lines = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines()
    plans = ["omoe_sort_plan", "omoe_sort_rows", "omoe_sort_rows_backward", "omoe_unsort_rows", "omoe_unsort_rows_backward"]
    want = [f"-1 {fn}: null plan" for _ in range(4) for fn in plans]
    want += [f"-1 {fn}: bad list of tensors" for _ in range(2) for fn in ("omoe_grad_norm", "omoe_grad_scale", "omoe_grad_clip")]
    assert lines == want
