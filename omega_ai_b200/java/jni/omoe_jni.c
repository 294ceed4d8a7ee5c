/*
 * JNI shim for com.omega.engine.nn.layer.llama.OmoeNative: forwards each native
 * method to the C ABI of libomoe.so.  Naming follows the engine's own JNI
 * precedent (jni/com_omega_engine_gpu_JNITest.h: Java_<package>_<Class>_<method>).
 *
 * Build where a JDK exists:
 *   gcc -shared -fPIC -I"$JAVA_HOME/include" -I"$JAVA_HOME/include/linux" -I../../../include \
 *       omoe_jni.c -o libomoe_jni.so -L.. -lomoe -Wl,-rpath,'$ORIGIN'
 */
#if defined(__has_include)
#if __has_include(<jni.h>)
#define OMOE_HAVE_JNI 1
#endif
#endif

#ifdef OMOE_HAVE_JNI
#include <jni.h>
#include <stdlib.h>
#include <string.h>

#include "omoe.h"

#define JFN(ret, name) JNIEXPORT ret JNICALL Java_com_omega_engine_nn_layer_llama_OmoeNative_##name

JFN(jlong, create)(JNIEnv *env, jclass c, jint tMax, jint d, jint dff, jint E, jint k, jint cdt, jint renorm,
                   jint hasBias, jint world, jint rank, jint recvRows) {
    omoe_config cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.t_max = tMax; cfg.d_model = d; cfg.d_ff = dff; cfg.n_experts = E; cfg.top_k = k;
    cfg.compute_dtype = cdt; cfg.renormalize = renorm; cfg.has_router_bias = hasBias;
    cfg.world = world; cfg.rank = rank; cfg.recv_rows_max = recvRows;
    omoe_handle *h = NULL;
    return omoe_create(&cfg, &h) == OMOE_OK ? (jlong)(intptr_t)h : 0;
}

JFN(jint, destroy)(JNIEnv *env, jclass c, jlong h) { return omoe_destroy((omoe_handle *)(intptr_t)h); }

JFN(jstring, lastError)(JNIEnv *env, jclass c, jlong h) {
    return (*env)->NewStringUTF(env, omoe_last_error((omoe_handle *)(intptr_t)h));
}

JFN(jint, setWeights)(JNIEnv *env, jclass c, jlong h, jlong wr, jlong rb, jlong wg, jlong wu, jlong wd, jint dt) {
    return omoe_set_weights((omoe_handle *)(intptr_t)h, (const void *)(intptr_t)wr, (const void *)(intptr_t)rb,
                            (const void *)(intptr_t)wg, (const void *)(intptr_t)wu, (const void *)(intptr_t)wd, dt,
                            NULL /* legacy default stream */);
}

JFN(jint, forward)(JNIEnv *env, jclass c, jlong h, jlong x, jlong y, jint T, jint io) {
    return omoe_forward((omoe_handle *)(intptr_t)h, (const void *)(intptr_t)x, (void *)(intptr_t)y, T, io, NULL);
}

JFN(jint, forwardHost)(JNIEnv *env, jclass c, jlong h, jfloatArray x, jfloatArray y, jint T) {
    jfloat *xp = (*env)->GetFloatArrayElements(env, x, NULL);
    jfloat *yp = (*env)->GetFloatArrayElements(env, y, NULL);
    int rc = omoe_forward_host((omoe_handle *)(intptr_t)h, xp, yp, T, OMOE_F32, NULL);
    (*env)->ReleaseFloatArrayElements(env, x, xp, JNI_ABORT);
    (*env)->ReleaseFloatArrayElements(env, y, yp, 0);
    return rc;
}

/* The arrays of an asynchronous call stay pinned (GetFloatArrayElements) until waitDone releases them. */
static jfloatArray g_async_x, g_async_y;
static jfloat *g_async_xp, *g_async_yp;

static void release_async(JNIEnv *env) {
    if (g_async_x) {
        (*env)->ReleaseFloatArrayElements(env, g_async_x, g_async_xp, JNI_ABORT);
        (*env)->ReleaseFloatArrayElements(env, g_async_y, g_async_yp, 0);
        (*env)->DeleteGlobalRef(env, g_async_x);
        (*env)->DeleteGlobalRef(env, g_async_y);
        g_async_x = g_async_y = NULL;
    }
}

JFN(jint, forwardHostAsync)(JNIEnv *env, jclass c, jlong h, jfloatArray x, jfloatArray y, jint T) {
    if (g_async_x) {  /* one call in flight per process through this shim: finish the previous one first */
        int rc0 = omoe_wait((omoe_handle *)(intptr_t)h);
        release_async(env);
        if (rc0 != OMOE_OK) return rc0;
    }
    g_async_x = (jfloatArray)(*env)->NewGlobalRef(env, x);
    g_async_y = (jfloatArray)(*env)->NewGlobalRef(env, y);
    g_async_xp = (*env)->GetFloatArrayElements(env, g_async_x, NULL);
    g_async_yp = (*env)->GetFloatArrayElements(env, g_async_y, NULL);
    int rc = omoe_forward_host_async((omoe_handle *)(intptr_t)h, g_async_xp, g_async_yp, T, OMOE_F32, NULL);
    if (rc != OMOE_OK) release_async(env);
    return rc;
}

JFN(jint, waitDone)(JNIEnv *env, jclass c, jlong h) {
    int rc = omoe_wait((omoe_handle *)(intptr_t)h);
    release_async(env);
    return rc;
}

JFN(jint, forwardBlock)(JNIEnv *env, jclass c, jlong h, jlong x, jlong gamma, jfloat eps, jlong y, jint T, jint io) {
    return omoe_forward_block((omoe_handle *)(intptr_t)h, (const void *)(intptr_t)x, (const float *)(intptr_t)gamma, eps,
                              (void *)(intptr_t)y, T, io, NULL);
}

JFN(jint, getRouting)(JNIEnv *env, jclass c, jlong h, jintArray idx, jfloatArray w, jintArray counts,
                      jintArray offsets, jintArray perm) {
    jint *pi = idx ? (*env)->GetIntArrayElements(env, idx, NULL) : NULL;
    jfloat *pw = w ? (*env)->GetFloatArrayElements(env, w, NULL) : NULL;
    jint *pc = counts ? (*env)->GetIntArrayElements(env, counts, NULL) : NULL;
    jint *po = offsets ? (*env)->GetIntArrayElements(env, offsets, NULL) : NULL;
    jint *pp = perm ? (*env)->GetIntArrayElements(env, perm, NULL) : NULL;
    int rc = omoe_get_routing((omoe_handle *)(intptr_t)h, (int32_t *)pi, pw, (int32_t *)pc, (int32_t *)po, (int32_t *)pp);
    if (pi) (*env)->ReleaseIntArrayElements(env, idx, pi, 0);
    if (pw) (*env)->ReleaseFloatArrayElements(env, w, pw, 0);
    if (pc) (*env)->ReleaseIntArrayElements(env, counts, pc, 0);
    if (po) (*env)->ReleaseIntArrayElements(env, offsets, po, 0);
    if (pp) (*env)->ReleaseIntArrayElements(env, perm, pp, 0);
    return rc;
}

JFN(jint, setTraining)(JNIEnv *env, jclass c, jlong h, jint on) {
    return omoe_set_training((omoe_handle *)(intptr_t)h, on);
}

JFN(jint, backward)(JNIEnv *env, jclass c, jlong h, jlong x, jlong dy, jlong dx, jint T, jint io) {
    return omoe_backward((omoe_handle *)(intptr_t)h, (const void *)(intptr_t)x, (const void *)(intptr_t)dy,
                         (void *)(intptr_t)dx, T, io, NULL);
}

JFN(jint, getWeightGrads)(JNIEnv *env, jclass c, jlong h, jlong dr, jlong db, jlong dg, jlong du, jlong dd) {
    return omoe_get_weight_grads((omoe_handle *)(intptr_t)h, (float *)(intptr_t)dr, (float *)(intptr_t)db,
                                 (float *)(intptr_t)dg, (float *)(intptr_t)du, (float *)(intptr_t)dd, NULL);
}

JFN(jint, epConnectLocal)(JNIEnv *env, jclass c, jlongArray hs) {
    jsize n = (*env)->GetArrayLength(env, hs);
    jlong *p = (*env)->GetLongArrayElements(env, hs, NULL);
    omoe_handle *arr[8];
    if (n > 8) n = 8;
    for (jsize i = 0; i < n; i++) arr[i] = (omoe_handle *)(intptr_t)p[i];
    int rc = omoe_ep_connect_local(arr, (int32_t)n);
    (*env)->ReleaseLongArrayElements(env, hs, p, JNI_ABORT);
    return rc;
}

JFN(jint, epExport)(JNIEnv *env, jclass c, jlong h, jbyteArray blob) {
    jbyte *p = (*env)->GetByteArrayElements(env, blob, NULL);
    int rc = omoe_ep_export((omoe_handle *)(intptr_t)h, p);
    (*env)->ReleaseByteArrayElements(env, blob, p, 0);
    return rc;
}

JFN(jint, epImport)(JNIEnv *env, jclass c, jlong h, jbyteArray blobs) {
    jbyte *p = (*env)->GetByteArrayElements(env, blobs, NULL);
    int rc = omoe_ep_import((omoe_handle *)(intptr_t)h, p);
    (*env)->ReleaseByteArrayElements(env, blobs, p, JNI_ABORT);
    return rc;
}
/* ---- operators without a handle ---- */
#define P(a) ((void *)(intptr_t)(a))

JFN(jstring, opsError)(JNIEnv *env, jclass c) { return (*env)->NewStringUTF(env, omoe_ops_error()); }

JFN(jlong, sortRowsCap)(JNIEnv *env, jclass c, jint T, jint k, jint E, jint align) {
    return omoe_sort_rows_cap(T, k, E, align);
}

/* The plan's sizes and addresses, 9 longs; NULL, which the library refuses, where there are fewer or a size does not fit. */
static const omoe_sort *read_plan(JNIEnv *env, jlongArray plan, omoe_sort *p) {
    if (!plan || (*env)->GetArrayLength(env, plan) < 9) return NULL;
    jlong *v = (*env)->GetLongArrayElements(env, plan, NULL);
    if (!v) return NULL;
    int ok = 1;
    for (int i = 0; i < 4; i++) ok = ok && v[i] >= INT32_MIN && v[i] <= INT32_MAX;
    p->n_tokens = (int32_t)v[0]; p->top_k = (int32_t)v[1]; p->n_experts = (int32_t)v[2]; p->row_align = (int32_t)v[3];
    p->rows_cap = v[4];
    p->pos = (int32_t *)P(v[5]); p->perm = (int32_t *)P(v[6]); p->counts = (int32_t *)P(v[7]); p->offsets = (int32_t *)P(v[8]);
    (*env)->ReleaseLongArrayElements(env, plan, v, JNI_ABORT);
    return ok ? p : NULL;
}

JFN(jint, sortPlan)(JNIEnv *env, jclass c, jlongArray plan, jlong idx) {
    omoe_sort p;
    return omoe_sort_plan(read_plan(env, plan, &p), (const int32_t *)P(idx), NULL);
}

JFN(jint, sortRows)(JNIEnv *env, jclass c, jlongArray plan, jlong x, jlong ldx, jint xdt, jlong xs, jlong ldxs, jint xsdt, jint d) {
    omoe_sort p;
    return omoe_sort_rows(read_plan(env, plan, &p), P(x), ldx, xdt, P(xs), ldxs, xsdt, d, NULL);
}

JFN(jint, sortRowsBackward)(JNIEnv *env, jclass c, jlongArray plan, jlong dxs, jlong lddxs, jint dxsdt, jlong dx, jlong lddx,
                            jint dxdt, jint d) {
    omoe_sort p;
    return omoe_sort_rows_backward(read_plan(env, plan, &p), P(dxs), lddxs, dxsdt, P(dx), lddx, dxdt, d, NULL);
}

JFN(jint, unsortRows)(JNIEnv *env, jclass c, jlongArray plan, jlong ys, jlong ldys, jint ysdt, jlong w, jlong y, jlong ldy,
                      jint ydt, jint d) {
    omoe_sort p;
    return omoe_unsort_rows(read_plan(env, plan, &p), P(ys), ldys, ysdt, (const float *)P(w), P(y), ldy, ydt, d, NULL);
}

JFN(jint, unsortRowsBackward)(JNIEnv *env, jclass c, jlongArray plan, jlong dy, jlong lddy, jint dydt, jlong ys, jlong ldys,
                              jint ysdt, jlong w, jlong dys, jlong lddys, jlong dw, jint d) {
    omoe_sort p;
    return omoe_unsort_rows_backward(read_plan(env, plan, &p), P(dy), lddy, dydt, P(ys), ldys, ysdt, (const float *)P(w),
                                     P(dys), lddys, (float *)P(dw), d, NULL);
}

JFN(jint, layerNorm)(JNIEnv *env, jclass c, jlong x, jlong ldx, jint xdt, jlong gamma, jlong beta, jfloat eps, jlong y, jlong ldy,
                     jint ydt, jlong mean, jlong rstd, jint T, jint d) {
    return omoe_layer_norm(P(x), ldx, xdt, (const float *)P(gamma), (const float *)P(beta), eps, P(y), ldy, ydt, (float *)P(mean),
                           (float *)P(rstd), T, d, NULL);
}

JFN(jlong, layerNormBackwardWorkspace)(JNIEnv *env, jclass c, jint T, jint d) { return omoe_layer_norm_backward_workspace(T, d); }

JFN(jint, layerNormBackward)(JNIEnv *env, jclass c, jlong dy, jlong lddy, jint dydt, jlong x, jlong ldx, jint xdt, jlong gamma,
                             jlong mean, jlong rstd, jlong dx, jlong lddx, jlong dgamma, jlong dbeta, jint T, jint d, jlong ws,
                             jlong wsBytes) {
    return omoe_layer_norm_backward(P(dy), lddy, dydt, P(x), ldx, xdt, (const float *)P(gamma), (const float *)P(mean),
                                    (const float *)P(rstd), P(dx), lddx, (float *)P(dgamma), (float *)P(dbeta), T, d, P(ws),
                                    wsBytes, NULL);
}

/* Host table of the tensors, to be freed; *n is -1, which the library refuses, where the arrays do not agree or memory is short. */
static omoe_tensor *read_tensors(JNIEnv *env, jlongArray ptrs, jlongArray counts, jintArray dtypes, jint *n) {
    *n = -1;
    if (!ptrs || !counts || !dtypes) return NULL;
    jint m = (*env)->GetArrayLength(env, ptrs);
    if ((*env)->GetArrayLength(env, counts) != m || (*env)->GetArrayLength(env, dtypes) != m) return NULL;
    omoe_tensor *t = (omoe_tensor *)malloc(sizeof(omoe_tensor) * (size_t)(m > 0 ? m : 1));
    if (!t) return NULL;
    jlong *a = (*env)->GetLongArrayElements(env, ptrs, NULL), *b = (*env)->GetLongArrayElements(env, counts, NULL);
    jint *d = (*env)->GetIntArrayElements(env, dtypes, NULL);
    if (a && b && d) {
        for (jint i = 0; i < m; i++) {
            t[i].ptr = P(a[i]); t[i].count = b[i]; t[i].dtype = d[i]; t[i].reserved = 0;
        }
        *n = m;
    }
    if (a) (*env)->ReleaseLongArrayElements(env, ptrs, a, JNI_ABORT);
    if (b) (*env)->ReleaseLongArrayElements(env, counts, b, JNI_ABORT);
    if (d) (*env)->ReleaseIntArrayElements(env, dtypes, d, JNI_ABORT);
    return t;
}

JFN(jint, gradNorm)(JNIEnv *env, jclass c, jlongArray g, jlongArray n, jintArray dt, jlong norm, jlong ws, jlong wsBytes) {
    jint m;
    omoe_tensor *t = read_tensors(env, g, n, dt, &m);
    int rc = omoe_grad_norm(t, m, (float *)P(norm), P(ws), wsBytes, NULL);
    free(t);
    return rc;
}

JFN(jint, gradScale)(JNIEnv *env, jclass c, jlongArray g, jlongArray n, jintArray dt, jlong norm, jfloat maxNorm) {
    jint m;
    omoe_tensor *t = read_tensors(env, g, n, dt, &m);
    int rc = omoe_grad_scale(t, NULL, m, (const float *)P(norm), maxNorm, NULL);
    free(t);
    return rc;
}

JFN(jint, gradClip)(JNIEnv *env, jclass c, jlongArray g, jlongArray n, jintArray dt, jfloat maxNorm, jlong norm, jlong ws,
                    jlong wsBytes) {
    jint m;
    omoe_tensor *t = read_tensors(env, g, n, dt, &m);
    int rc = omoe_grad_clip(t, NULL, m, maxNorm, (float *)P(norm), P(ws), wsBytes, NULL);
    free(t);
    return rc;
}
#else
/* No JDK headers on this machine: nothing to compile. */
typedef int omoe_jni_unavailable;
#endif
